// Attention over selected key blocks, backward, in a fixed order throughout (no floating-point atomics).
//   P = exp(S - lse);  dP = dO V^T;  dS = P (dP - delta),  delta = sum_d dO O (O unrounded)
//   dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO;  dbias[bucket][head] = sum of dS over the bucket's pairs
// Two passes recompute S and dP (7 products of the pairs instead of 5): one per query group for dQ and dbias, one per key block for dK
// and dV, which needs the selection the other way round: a bit for every (key block, query group), then the blocks' query rows cut
// into chunks of equal length, since a first block is chosen by every group and most blocks by few.
//
// Four launches: the selection turned round; dQ, dbias, delta and the chunks; dK and dV; the chunks' sums.  2 x 4096 bf16 tokens, 16
// heads of 64 over 4 key heads, 16 blocks of 64: 5 + 67 + 105 + 10 us behind a forward pass of 59 with 54 % of the pairs
// live, 280 for the four with all of them; 65536 fp32 tokens of 48, one head: 5 + 177 + 288 + 17 behind 122.  (One launch more for each of delta,
// the chunks and dbias: an eighth more for the first.)
#include "block_attn.hpp"

namespace scipnp {

int attn_check(const scipnp_block_attn_args* a);
Attn attn_params(const scipnp_block_attn_args* a);

constexpr int KB = 64;                                    // keys of a dK / dV workgroup

__device__ __forceinline__ unsigned fast_div(unsigned x, unsigned d, unsigned m, unsigned& rem) {   // m = floor(2^32 / d), 2^32 - 1 for 1
    unsigned q = __umulhi(x, m), r = x - q * d;
    if (r >= d) { ++q; r -= d; }
    rem = r;
    return q;
}
static inline unsigned div_magic(int d) { return d <= 1 ? 0xFFFFFFFFu : (unsigned)((1ull << 32) / (unsigned)d); }

// ---- the selection the other way round: a workgroup gathers 32 query groups, a bit each in a word for every key block.  No word is
// written twice, so nothing has to be cleared before; and the zeros that rows that do not exist are read from.  Latency: 5 us, whether
// 1024 groups choose among 64 blocks or among 1024 (atomics on words in memory: 15 us where every group chooses one block)
constexpr int MARK_WAVES = 16, MARK_CAP = 16384;          // (key blocks in LDS at a time)
__global__ void __launch_bounds__(64 * MARK_WAVES) attn_mark_kernel(Attn a, int cap) {
    extern __shared__ unsigned bits[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, word = blockIdx.x, bh = blockIdx.y;
    int* const list = (int*)(bits + cap) + wave * a.n;
    const Seq s = seq_of(a, bh / a.Hk);
    if (word == 0 && bh == 0 && tid < 64) a.zeros[tid] = 0.f;
    for (int base = 0; base < a.nb; base += cap) {
        const int m = min(cap, a.nb - base);
        for (int i = tid; i < m; i += 64 * MARK_WAVES) bits[i] = 0;
        __syncthreads();
        for (int g = 32 * word + wave; g < min(a.ng, 32 * word + 32); g += MARK_WAVES) {
            const int q0 = g * a.qb, nq = min(a.qb, s.qlen - q0);
            if (nq <= 0) break;
            const int far = a.causal ? min(s.klen, s.shift + q0 + nq) : s.klen;
            const int c = live_blocks(a, a.sel + ((size_t)bh * a.ng + g) * a.n, far, list, lane);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int i = lane; i < c; i += 64) {
                const int e = list[i] - base;
                if (e >= 0 && e < m) atomicOr(&bits[e], 1u << (g & 31));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        __syncthreads();
        for (int i = tid; i < m; i += 64 * MARK_WAVES) a.member[((size_t)bh * a.words + word) * a.nb4 + base + i] = bits[i];
        __syncthreads();
    }
}

// ---- chunks of every key block of one (sequence, key head), by one workgroup: chunk_start[j] = chunks of the blocks before j; a block's
// chunks are of one length, chunk_rows[j] <= CH (a multiple of 64; the last may be shorter)
__device__ __forceinline__ void plan_chunks(const Attn& a, int bh, int R, int CH, int* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    int* const wsum = lds;
    int* const cs = a.chunk_start + (size_t)bh * (a.nb + 1);
    int* const cr = a.chunk_rows + (size_t)bh * a.nb;
    int carry = 0;
    for (int base = 0; base < a.nb; base += 4 * blockDim.x) {     // four neighbouring blocks a thread
        const int j = base + 4 * tid;
        int n[4] = {0, 0, 0, 0};
        if (j < a.nb) {
            const uint4* p = (const uint4*)(a.member + (size_t)bh * a.words * a.nb4 + j);
#pragma unroll 16
            for (int w = 0; w < a.words; ++w) {
                const uint4 x = p[(size_t)w * (a.nb4 / 4)];
                n[0] += __popc(x.x), n[1] += __popc(x.y), n[2] += __popc(x.z), n[3] += __popc(x.w);
            }
        }
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const long long rows = (long long)n[e] * R;
            const int c = j + e < a.nb ? (int)((rows + CH - 1) / CH) : 0;
            if (c > 0) cr[j + e] = (int)(((rows + c - 1) / c + 63) / 64 * 64);
            n[e] = sum;
            sum += c;
        }
        int incl = sum;
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) wsum[wave] = incl;
        __syncthreads();
        int at = carry + incl - sum;
        for (int w = 0; w < waves; ++w) {
            if (w < wave) at += wsum[w];
            carry += wsum[w];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < a.nb) cs[j + e] = at + n[e];
        __syncthreads();
    }
    if (tid == 0) cs[a.nb] = carry;
}

// ---- dQ, dbias: the forward's sets of waves and tiles.  The bias sums: one LDS word a bucket and row, the two ends (where
// most tiles lie) in registers.  Three products a tile and vector work of twice their length: 67 us for 131072 bf16 rows of 64, 54 % of
// them live, with about 1000 keys each (three waves a SIMD; two, with the transposed keys read before the vector work, were a quarter slower; 128 wide two
// waves instead of one: 72 us less), 177 us for 65536 x 1024 of 48 wide fp32 (109 TFLOP/s against 133)
template <typename T, int DP>
struct DqCfg {
    static constexpr int TILE = 2 * DmaTile<T, DP>::BYTES;                    // K and V
    static constexpr int MAIN = 2 * TILE;
    static constexpr int KP = 2 * KT * 4;
};
constexpr int HROW = 33;                                  // a bucket's sums of 32 rows, shifted by a bank

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? (DP > 64 ? 2 : 3) : DP > 64 ? 1 : 2) block_attn_dq_kernel(Attn a, int sets, int set_bytes, int plans, int CH) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = DqCfg<T, DP>;
    using Frag = typename Mat<T>::Frag;
    constexpr int NB = (DP + 31) / 32;
    constexpr bool LEAN = sizeof(T) == 2;                 // K read behind the vector work, the ends' bias from LDS: nothing in scratch at three waves
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    if (blockIdx.x < plans) {                             // the first workgroups cut the chunks of the launch behind this one
        plan_chunks(a, blockIdx.x, a.qb * a.G, CH, (int*)smem_all);
        return;
    }
    const long long total = (long long)a.B * a.Hk * a.ng * a.chunks, first = xcd_item(blockIdx.x - plans, (total + sets - 1) / sets);
    if (first < 0) return;
    const int lane = threadIdx.x & 63, li = lane & 31, hi = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int set = wave / RW, rw = wave % RW, tset = rw * 64 + lane;
    const bool there_is = first * sets + set < total;
    const unsigned item = there_is ? (unsigned)(first * sets + set) : 0;
    const int chunk = item % a.chunks, g = item / a.chunks % a.ng, bh = item / a.chunks / a.ng, hk = bh % a.Hk, b = bh / a.Hk;
    const Seq sq = seq_of(a, b);
    const int R = a.qb * a.G, r0 = chunk * 32 * RW;
    const int row = r0 + rw * 32 + li, tok = g * a.qb + row / a.G, gl = row % a.G, head = hk * a.G + gl;
    const bool live = there_is && row < R && tok < sq.qlen;
    const int qkey = sq.shift + tok;
    int lim = !live ? -1 : a.causal ? min(qkey, sq.klen - 1) : sq.klen - 1;
    const bool any = there_is && g * a.qb + r0 / a.G < sq.qlen;             // a live row in this chunk

    unsigned char* const lut = (unsigned char*)smem_all;
    int* const longest = (int*)(smem_all + bias_lut_bytes(a.nbuckets, a.maxd));
    char* const smem = smem_all + bias_lut_bytes(a.nbuckets, a.maxd) + 16 + set * set_bytes;
    int* const kp_lds = (int*)(smem + C::MAIN);
    int* const list = (int*)(smem + C::MAIN + C::KP);
    int* const nlist = list + a.n;
    float* const tbl = (float*)(smem + C::MAIN + C::KP + (a.n + 4) / 4 * 16);
    const Bias bias = load_bias(a, lut, tbl, hk, tset, 64 * RW);
    float* const hist = tbl + (a.nbuckets * a.G + 3) / 4 * 4;
    float* const mine = hist + rw * a.nbuckets * HROW + li;
    if (hi == 0)
        for (int i = 0; i < a.nbuckets; ++i) mine[i * HROW] = 0.f;
    if (threadIdx.x == 0) *longest = 0;
    if (rw == 0) {
        int c = 0;
        if (any) {
            const int rows_end = min(min(R, r0 + 32 * RW), (sq.qlen - g * a.qb) * a.G);
            const int far = a.causal ? min(sq.klen, sq.shift + g * a.qb + (rows_end - 1) / a.G + 1) : sq.klen;
            c = live_tiles(a, a.sel + ((size_t)bh * a.ng + g) * a.n, far, list, lane);
        }
        if (lane == 0) *nlist = c;
    }
    Frag qf[DP / Mat<T>::K], gf[DP / Mat<T>::K];
    load_frags<T, DP>(live ? (const T*)a.q + b * a.sq.b + (long long)tok * a.sq.t + head * a.sq.h : nullptr, a.D, hi, qf);
    load_frags<T, DP>(live ? (const T*)a.dout + b * a.sdo.b + (long long)tok * a.sdo.t + head * a.sdo.h : nullptr, a.D, hi, gf);
    const size_t stat = ((size_t)b * a.Hq + head) * a.Lq + tok;
    // minus the row's log-sum-exp.  A row that does not exist (or saw nothing) has a weight of exp2(-inf) = 0 whatever its bias: the sums of
    // dbias run over all rows of a wave, and its exponential of a large bias would be infinity there, times a zero
    Shift shift = {-INFINITY, 0.f};
    if (live) {
        const float lse = a.lse[stat];
        if (lse == -INFINITY) lim = -1;                   // (a row that saw nothing: of its keys, or because the bias masks them)
        else shift = load_lse(lse, a.lse_rest[stat]);
    }
    // delta of the row, in fp64: each half of a row's lanes has half of it
    double dsum = 0.0;
    if (live) {
        const float* const orow = a.out32 + (((size_t)b * a.Lq + tok) * a.Hq + head) * a.D;
#pragma unroll
        for (int s = 0; s < DP / Mat<T>::K; ++s) {
            const int c = Mat<T>::K * s + Mat<T>::E * hi;
            if (c < a.D)
#pragma unroll
                for (int i = 0; i < Mat<T>::E; ++i) dsum = fma((double)(float)gf[s][i], (double)orow[c + i], dsum);
        }
    }
    const float delta = (float)(dsum + __shfl_xor(dsum, 32, 64));
    if (live && hi == 0) a.delta[stat] = delta;
    const int qp = a.nbuckets && live ? (a.q_pos ? a.q_pos[(size_t)b * a.Lq + tok] : qkey) : 0;
    const RowRange range = {wave_min(live ? qp : INT_MAX), wave_max(live ? qp : INT_MIN)};
    const int min_lim = wave_min(live ? lim : INT_MAX);
    const unsigned ks = (unsigned)(a.sk.t * (long long)sizeof(T)), vs = (unsigned)(a.sv.t * (long long)sizeof(T));
    DmaOffsets<T, DP, RW> ko, vo;
    ko.init(rw, lane, ks, a.D);
    vo.init(rw, lane, vs, a.D);
    __syncthreads();

    const int count = __builtin_amdgcn_readfirstlane(*nlist);
    int trips = count;                                    // sets that share a barrier take the same number of trips
    if constexpr (RW > 1) {
        if (sets > 1) {
            if (tset == 0) atomicMax(longest, count);
            __syncthreads();
            trips = __builtin_amdgcn_readfirstlane(*longest);
        }
    }
    const T* const kb = (const T*)a.k + b * a.sk.b + hk * a.sk.h;
    const T* const vb = (const T*)a.v + b * a.sv.b + hk * a.sv.h;
    int kpr = 0, blk = 0, off = 0;                        // the next tile to ask for
    auto next_key = [&]() -> int {
        const int key = __builtin_amdgcn_readfirstlane(list[blk]) * a.block + off;
        off += KT;
        if (off == a.block) { off = 0; ++blk; }
        return key;
    };
    auto issue = [&](int key0, int buf) {
        const int there = min(KT, sq.klen - key0);
        char* const tile = smem + buf * C::TILE;
        ko.issue(kb + (long long)key0 * a.sk.t, there, ks, a.D, tile, rw);
        vo.issue(vb + (long long)key0 * a.sv.t, there, vs, a.D, tile + DmaTile<T, DP>::BYTES, rw);
        if (a.k_pos && tset < KT) kpr = tset < there ? a.k_pos[(size_t)b * a.Lk + key0 + tset] : 0;
    };
    const int far = 2 * a.maxd;
    const float bias_lo = a.nbuckets ? bias.tbl[bias.lut[0] * a.G + gl] : 0.f, bias_hi = a.nbuckets ? bias.tbl[bias.lut[far] * a.G + gl] : 0.f;
    float sum_lo = 0.f, sum_hi = 0.f;
    auto add_bucket = [&](int n, float v) {
        v += __shfl_xor(v, 32, 64);
        if (hi == 0) mine[n * HROW] += v;
    };
    Acc<T, DP> sums;
    sums.zero();

    int key0 = 0;
    if (count > 0) {
        key0 = next_key();
        issue(key0, 0);
    }
    for (int t = 0; t < count; ++t) {
        const int buf = t & 1, cur = key0;
        int* const kp = kp_lds + buf * KT;
        if (a.k_pos && tset < KT) kp[tset] = kpr;
        dma_wait<RW>();
        if (t + 1 < count) {
            key0 = next_key();
            issue(key0, buf ^ 1);
        }
        const char* const kt = smem + buf * C::TILE;
        __builtin_amdgcn_s_setprio(1);
        f32x16a s = dma_rows<T, DP>(kt, qf, lane);
        const f32x16a dp = dma_rows<T, DP>(kt + DmaTile<T, DP>::BYTES, gf, lane);
        __builtin_amdgcn_s_setprio(0);
        ColTile<T, DP> kc;
        if constexpr (!LEAN) kc.read(kt, lane);
        const int dist = a.nbuckets ? tile_distance(a, range, cur, a.k_pos ? kp : nullptr, lane) : 0;
        // fp32: the large numbers, score and log-sum-exp, meet in one fused operation, and what is small is added behind it; bf16 weights
        // are rounded to 8 bits anyway: one operation
        if (dist >= 0) {
            const float b = !a.nbuckets ? 0.f : !LEAN && dist == 0 ? bias_lo : !LEAN && dist == far ? bias_hi : bias.tbl[bias.lut[dist] * a.G + gl];
            if constexpr (sizeof(T) == 4) {
                const float rest = b + shift.lo;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, shift.hi) + rest);
            } else {
                const float add = b + shift.hi;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, add));
            }
        } else {
            float x[16];
            tile_bias(a, bias, cur, a.k_pos ? kp : nullptr, qp, gl, hi, x);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, shift.hi) + (x[r] + shift.lo));
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
        if (cur + KT - 1 > min_lim) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = cur + tile_key(r, hi) <= lim ? s[r] : 0.f;
        }
        if (a.dbias) {
            if (dist >= 0) {
                const float sum = (((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]))) +
                                  (((s[8] + s[9]) + (s[10] + s[11])) + ((s[12] + s[13]) + (s[14] + s[15])));
                if (dist == 0) sum_lo += sum;
                else if (dist == far) sum_hi += sum;
                else add_bucket(bias.lut[dist], sum);
            } else {
                int d[16];
                tile_buckets(a, bias, cur, a.k_pos ? kp : nullptr, qp, hi, d);
#pragma unroll
                for (int half = 0; half < 2; ++half) {    // (the two lanes of a row share its words: one after the other, the fence keeps them apart)
                    if (hi == half)
#pragma unroll
                        for (int r = 0; r < 16; ++r) mine[d[r] * HROW] += s[r];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
            }
        }
        __builtin_amdgcn_s_setprio(1);
        if constexpr (LEAN) kc.read(kt, lane);
        kc.mma(Weights<T, 2>(s), sums);                   // (dS in 16 bits: its rows sum to zero, so a rounding to 8 weighs more than the result's own)
        __builtin_amdgcn_s_setprio(0);
    }
    for (int t = count; t < trips; ++t) dma_wait<RW>();   // (the other sets' barriers)
    f32x16a o[NB];
    sums.blocks(o);
    if (a.dbias) {                                        // the set's sums: a (bucket, head) adds its lanes in order, in fp64
        add_bucket(bias.lut[0], sum_lo);
        add_bucket(bias.lut[far], sum_hi);
        __syncthreads();
        if (there_is)
            for (int i = tset; i < a.nbuckets * a.G; i += 64 * RW) {
                const int n = i / a.G, h = i - n * a.G;
                double sum = 0.0;
                for (int w = 0; w < RW; ++w) {
                    const int at = (r0 + w * 32) % a.G;
                    for (int y = (h - at + a.G) % a.G; y < 32; y += a.G)
                        sum += (double)hist[(w * a.nbuckets + n) * HROW + y];
                }
                a.pbias[(size_t)item * a.nbuckets * a.G + i] = sum;
            }
    }
    if (!there_is || row >= R || tok >= a.Lq) return;
    T* const dst = (T*)a.dq + (((size_t)b * a.Lq + tok) * a.Hq + head) * a.D;
    each_four<T, DP>(hi, [&](int d, auto at) {
        if (d >= a.D) return;
        f32x4a v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live ? o[at(e) >> 4][at(e) & 15] * a.scale : 0.f;
        store_four(dst + d, v);
    });
#endif
}


// ---- dK, dV of 64 keys over one chunk of the query rows that chose their block.  Waves: two halves of the keys x two of the row tiles;
// a wave keeps its 32 keys and values in registers (the B operands) and streams rows, which the memory system writes to LDS
// (global_load ... lds: the rows of a tile may belong to several query groups): S, dP with the rows as A, then dV += dO^T P and
// dK += Q^T dS with the transposed rows as A and the score registers as B.
// Bound by the vector work between the products: the products of 32 x 32, the second ones in two parts, take 768 cycles a tile at bf16, 64
// wide, the rest about 1000, of which the rows' books are a fifth (they were half while every lane divided for its own requests: 447
// instead of 350 us in fp32, then).  Chunks of a 2048th of all rows: larger ones leave CUs idle at the end (the whole backward pass at 2 x 4096 tokens
// of 64 286 us instead of 280 at a 1024th, 1292 instead of 1200 in fp32 at 56 wide; 555 instead of 580 at 128), smaller ones pay for their
// beginnings (318 at a 4096th).
// What a row brings besides: its last visible key, delta, log-sum-exp, and its bias where all 64 keys share its bucket.
template <typename T, int DP>
struct DkvCfg {
    static constexpr int INFO = KT * 24 + 16;             // - lse (bf16: + bias), delta, last key, position, head, (fp32) bias - rest of lse of each row; flags
    static constexpr int TILE = 2 * DmaTile<T, DP>::BYTES + INFO + KT * 16;   // ... and where the rows of q and dout begin
    static constexpr int MAIN = 4 * TILE;                 // two row tiles, two buffers
    static constexpr int JOIN = 2 * 32 * ((DP + 31) / 32 * 32 + 4) * 4;
    static_assert(JOIN <= MAIN, "the join reuses the tiles");
    static constexpr int LIST = 1032;                     // query groups of a chunk
};
// bf16: the transposed rows are read behind the vector work.  Early, under it, they would leave one wave a SIMD at 96 columns (the whole
// backward pass of 131072 rows: 497 us instead of 376, then) and gain nothing at 64 (283 us both ways)

template <typename T, int DP>
__global__ void __launch_bounds__(256, DP > (sizeof(T) == 2 ? 96 : 64) ? 1 : 2) block_attn_dkv_kernel(Attn a, int subs, unsigned magic_r, unsigned magic_g) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = DkvCfg<T, DP>;
    using Frag = typename Mat<T>::Frag;
    constexpr int NB = (DP + 31) / 32, LC = DmaTile<T, DP>::LC, PIECES = DmaTile<T, DP>::PIECES, MINE = (PIECES + 1) / 2, BYTES = DmaTile<T, DP>::BYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // (chunks in turn over the XCDs: the last of a sequence and key head's slots are empty)
    const int sub = blockIdx.x % subs, c = blockIdx.x / subs % a.max_chunks, bh = blockIdx.x / subs / a.max_chunks, hk = bh % a.Hk, b = bh / a.Hk;
    const int* const cs = a.chunk_start + (size_t)bh * (a.nb + 1);
    if (c >= cs[a.nb]) return;                            // (uniform)
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave & 1, rs = wave >> 1;
    char* const main = smem;
    int* const list = (int*)(smem + C::MAIN);
    int* const misc = list + C::LIST;                     // block, scan
    char* const bias_at = smem + C::MAIN + (C::LIST + 8) * 4;
    const Bias bias = load_bias(a, (unsigned char*)bias_at, (float*)(bias_at + bias_lut_bytes(a.nbuckets, a.maxd)), hk, tid, 256);
    for (int j = tid; j < a.nb; j += 256)
        if (cs[j] <= c && c < cs[j + 1]) misc[0] = j;
    __syncthreads();
    const int j = __builtin_amdgcn_readfirstlane(misc[0]), nchunks = cs[j + 1] - cs[j];
    const int R = a.qb * a.G;
    const Seq sq = seq_of(a, b);
    // the chunk's rows are x0 .. x1 of the block's groups laid end to end; their groups into the list
    const unsigned len = (unsigned)a.chunk_rows[(size_t)bh * a.nb + j], x0 = (unsigned)(c - cs[j]) * len;
    int count = 0;
    {
        const unsigned* w = a.member + (size_t)bh * a.words * a.nb4 + j;
        const int e0 = (int)(x0 / R), e1 = (int)((x0 + len + R - 1) / R);
        for (int base = 0; base < a.words; base += 256) {
            const unsigned bits = base + tid < a.words ? w[(size_t)(base + tid) * a.nb4] : 0;
            const int n = __popc(bits);
            int incl = n;
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(incl, off, 64);
                if (lane >= off) incl += o;
            }
            __syncthreads();
            if (lane == 63) misc[1 + wave] = incl;
            __syncthreads();
            int rank = count + incl - n;
            for (int v = 0; v < wave; ++v) rank += misc[1 + v];
            for (unsigned rest = bits; rest; rest &= rest - 1, ++rank)
                if (rank >= e0 && rank < e1 && rank - e0 < C::LIST) list[rank - e0] = 32 * (base + tid) + __ffs(rest) - 1;
            count += misc[1] + misc[2] + misc[3] + misc[4];
        }
        __syncthreads();
    }
    const unsigned x1 = (unsigned)min((long long)x0 + len, (long long)count * R);
    const int e0 = (int)(x0 / R);

    const int k64 = j * a.block + sub * KB, kbase = k64 + kw * 32, key = kbase + li;
    const bool klive = key < sq.klen;
    Frag kf[DP / Mat<T>::K], vf[DP / Mat<T>::K];
    load_frags<T, DP>(klive ? (const T*)a.k + b * a.sk.b + (long long)key * a.sk.t + hk * a.sk.h : nullptr, a.D, hi, kf);
    load_frags<T, DP>(klive ? (const T*)a.v + b * a.sv.b + (long long)key * a.sv.t + hk * a.sv.h : nullptr, a.D, hi, vf);
    const int kpos = a.k_pos ? (klive ? a.k_pos[(size_t)b * a.Lk + key] : 0) : key;
    int klo = k64, khi = k64 + KB - 1;                    // positions of the 64 keys
    if (a.k_pos) {
        const int mine = k64 + lane < sq.klen ? a.k_pos[(size_t)b * a.Lk + k64 + lane] : INT_MAX;
        klo = wave_min(mine);
        khi = wave_max(k64 + lane < sq.klen ? mine : INT_MIN);
    }

    Acc<T, DP> kacc, vacc;
    kacc.zero();
    vacc.zero();

    // row x of the chunk -> token and head; tokens behind qlen: -1
    auto row_of = [&](unsigned x, int& tok, int& gl) {
        tok = -1;
        gl = 0;
        if (x >= x1) return;
        unsigned r, h;
        const unsigned e = fast_div(x, (unsigned)R, magic_r, r), q = fast_div(r, (unsigned)a.G, magic_g, h);
        const int t = list[(int)e - e0] * a.qb + (int)q;
        if (t < sq.qlen) { tok = t; gl = (int)h; }
    };
    const T* const qb0 = (const T*)a.q + b * a.sq.b + hk * a.G * a.sq.h;
    const T* const gb0 = (const T*)a.dout + b * a.sdo.b + hk * a.G * a.sdo.h;
    // Each row half's first wave keeps where the rows of the next tile begin, its second what they bring besides (32 lanes each)
    float ilse = 0.f, irest = 0.f, idelta = 0.f;
    int ilim = -1, iqp = 0, ig = 0, tok = -1, gl = 0;     // (tok, gl: of the row of the next tile)
    auto tile_at = [&](int it) -> char* { return main + (rs * 2 + (it & 1)) * C::TILE; };
    auto put_rows = [&](int it) {
        long long* const off = (long long*)(tile_at(it) + 2 * BYTES + C::INFO);
        off[lane] = tok < 0 ? -1 : tok * a.sq.t + gl * a.sq.h;
        off[KT + lane] = tok < 0 ? -1 : tok * a.sdo.t + gl * a.sdo.h;
    };
    auto get_info = [&]() {
        ilim = -1;
        ilse = irest = idelta = 0.f;
        iqp = 0;
        ig = gl;
        if (tok >= 0) {
            const size_t stat = ((size_t)b * a.Hq + hk * a.G + gl) * a.Lq + tok;
            ilse = a.lse[stat];
            irest = a.lse_rest[stat];
            idelta = a.delta[stat];
            ilim = a.causal ? min(sq.shift + tok, sq.klen - 1) : sq.klen - 1;
            iqp = a.q_pos ? a.q_pos[(size_t)b * a.Lq + tok] : sq.shift + tok;
        }
    };
    int chunk_at[MINE];                                   // elements into a row of this lane's 16 bytes, -1: past D
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int y = (kw + 2 * i) * 64 + lane, ch = (y % LC) ^ swz<T, LC>(y / LC);
        chunk_at[i] = ch * Mat<T>::E < a.D ? ch * Mat<T>::E : -1;
    }
    auto issue = [&](int it) {
        char* const tile = tile_at(it);
        const long long* const off = (const long long*)(tile + 2 * BYTES + C::INFO);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int piece = kw + 2 * i;
            if (PIECES % 2 == 0 || piece < PIECES) {
                const int at = (piece * 64 + lane) / LC;
                const long long oq = off[at], og = off[KT + at];
                const bool ok = oq >= 0 && chunk_at[i] >= 0;
                const T* const qa = ok ? qb0 + oq + chunk_at[i] : (const T*)a.zeros;
                const T* const ga = ok ? gb0 + og + chunk_at[i] : (const T*)a.zeros;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)qa, (__attribute__((address_space(3))) void*)(tile + 1024 * piece), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)ga, (__attribute__((address_space(3))) void*)(tile + BYTES + 1024 * piece), 16, 0, 0);
            }
        }
    };
    const int iters = (int)((x1 - x0 + 2 * KT - 1) / (2 * KT));
    const unsigned xs = x0 + rs * KT + lane;
    if (lane < KT) {
        row_of(xs, tok, gl);
        if (kw == 0) put_rows(0);
        else get_info();
        row_of(xs + 2 * KT, tok, gl);
    }
    __syncthreads();
    issue(0);
    for (int it = 0; it < iters; ++it) {
        char* const at = tile_at(it);
        float* const info = (float*)(at + 2 * BYTES);
        if (lane < KT) {
            if (kw == 0) {
                put_rows(it + 1);
            } else {
                if (ilse == -INFINITY) {                  // (a row that saw nothing)
                    ilse = 0.f;
                    ilim = -1;
                }
                const Shift shift = load_lse(ilse, irest);
                float own = 0.f;                          // its bias
                bool one = true;                          // every key has the same bucket for this row
                if (a.nbuckets && ilim >= 0) {
                    const int lo = clamp_dist(klo - iqp, a.maxd);
                    one = lo == clamp_dist(khi - iqp, a.maxd);
                    if (one) own = bias.tbl[bias.lut[lo] * a.G + ig];
                }
                const bool all_one = __ballot(!one) == 0, open = __ballot(ilim < k64 + KB - 1) == 0;
                if (!all_one) own = 0.f;
                info[lane] = sizeof(T) == 4 ? shift.hi : shift.hi + own;
                info[5 * KT + lane] = own + shift.lo;
                info[KT + lane] = idelta;
                info[2 * KT + lane] = __int_as_float(ilim);
                info[3 * KT + lane] = __int_as_float(iqp);
                info[4 * KT + lane] = __int_as_float(ig);
                if (lane == 0) info[6 * KT] = __int_as_float((all_one ? 0 : 1) | (open ? 0 : 2));
            }
        }
        dma_wait<4>();
        if (it + 1 < iters) {
            if (lane < KT) {                              // (before the tile is asked for: its wait is no wait for the tile)
                if (kw != 0) get_info();
                row_of(xs + (it + 2) * 2 * KT, tok, gl);
            }
            issue(it + 1);
        }
        const int flags = __builtin_amdgcn_readfirstlane(__float_as_int(info[6 * KT]));
        __builtin_amdgcn_s_setprio(1);
        f32x16a s = dma_rows<T, DP>(at, kf, lane);
        f32x16a dp = dma_rows<T, DP>(at + BYTES, vf, lane);
        __builtin_amdgcn_s_setprio(0);
        ColTile<T, DP> gc, qc;
        const float* const mine = info + 4 * hi;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4a add = *(const f32x4a*)(mine + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q + e] = fmaf(s[4 * q + e], a.scale2, add[e]);
            if constexpr (sizeof(T) == 4) {               // (the small numbers behind the large ones, as in the pass for dQ)
                const f32x4a rest = *(const f32x4a*)(mine + 5 * KT + 8 * q);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * q + e] += rest[e];
            }
        }
        if (flags & 1) {                                  // the bias key by key
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4a qp = *(const f32x4a*)(mine + 3 * KT + 8 * q), gh = *(const f32x4a*)(mine + 4 * KT + 8 * q);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[4 * q + e] += bias.tbl[bias.lut[clamp_dist(kpos - __float_as_int(qp[e]), a.maxd)] * a.G + __float_as_int(gh[e])];
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4a delta = *(const f32x4a*)(mine + KT + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * q + e;
                s[r] = __builtin_amdgcn_exp2f(s[r]);
                dp[r] = s[r] * (dp[r] - delta[e]);
            }
        }
        if (flags & 2) {                                  // some row does not see some key
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4a lim = *(const f32x4a*)(mine + 2 * KT + 8 * q);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool see = key <= __float_as_int(lim[e]);
                    s[4 * q + e] = see ? s[4 * q + e] : 0.f;
                    dp[4 * q + e] = see ? dp[4 * q + e] : 0.f;
                }
            }
        }
        __builtin_amdgcn_s_setprio(1);
        gc.read(at + BYTES, lane);
        gc.mma(Weights<T, 2>(s), vacc);                   // (bf16: P and dS in 16 bits, as in the pass for dQ; with 8 the gradients were 1.4 x as far off)
        qc.read(at, lane);
        qc.mma(Weights<T, 2>(dp), kacc);
        __builtin_amdgcn_s_setprio(0);
    }
    f32x16a dk[NB], dv[NB];
    kacc.blocks(dk);
    vacc.blocks(dv);
    // the two row halves: 1 into LDS, 0 adds
    float* const obuf = (float*)main + kw * 32 * (NB * 32 + 4);
    auto join = [&](f32x16a (&x)[NB]) {
        __syncthreads();
        float* const p = obuf + li * (NB * 32 + 4) + 4 * hi;
        if (rs == 1) {
#pragma unroll
            for (int db = 0; db < NB; ++db)
#pragma unroll
                for (int q = 0; q < 4; ++q) *(f32x4a*)(p + 32 * db + 8 * q) = f32x4a{x[db][4 * q], x[db][4 * q + 1], x[db][4 * q + 2], x[db][4 * q + 3]};
        }
        __syncthreads();
        if (rs == 0) {
#pragma unroll
            for (int db = 0; db < NB; ++db)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4a v = *(const f32x4a*)(p + 32 * db + 8 * q);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[db][4 * q + e] += v[e];
                }
        }
    };
    join(dv);
    join(dk);
    if (rs == 1) return;
    const size_t slot = ((size_t)bh * a.max_chunks + c) * subs + sub;
    auto put = [&](const f32x16a (&x)[NB], int which, T* dst, float scale) {
        each_four<T, DP>(hi, [&](int d, auto at) {
            if (d >= a.D) return;
            f32x4a v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[at(e) >> 4][at(e) & 15] * scale;
            if (nchunks > 1) *(f32x4a*)(a.pkv + ((slot * 2 + which) * KB + kw * 32 + li) * a.D + d) = v;
            else if (key < a.Lk) store_four(dst + (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D + d, v);
        });
    };
    put(dk, 0, (T*)a.dk, a.scale);
    put(dv, 1, (T*)a.dv, 1.f);
#endif
}

// dbias[n][head]: one wave sums the workgroups' partials, every 64th a lane
__device__ __forceinline__ void dbias_pair(const Attn& a, int pair) {
    const int n = pair / a.Hq, head = pair % a.Hq, hk = head / a.G, h = head % a.G, lane = threadIdx.x & 63;
    const size_t per = (size_t)a.ng * a.chunks, row = (size_t)a.nbuckets * a.G;
    double s = 0.0;
    for (int b = 0; b < a.B; ++b) {
        const double* p = a.pbias + ((size_t)(b * a.Hk + hk) * per) * row + (size_t)n * a.G + h;
        for (size_t i = lane; i < per; i += 64) s += p[i * row];
    }
    s = wave_sum_f64(s);
    if (lane == 0) a.dbias[(size_t)n * a.Hq + head] = (float)s;
}

// blocks that more than one chunk worked on (their partials in order), and blocks that nobody chose (zeros)
template <typename T>
__global__ void __launch_bounds__(256) attn_end_kernel(Attn a, int subs, unsigned joins) {
    if (blockIdx.x >= joins) {
        if (blockIdx.y) return;
        const int pair = (blockIdx.x - joins) * 4 + (threadIdx.x >> 6);
        if (pair < a.nbuckets * a.Hq) dbias_pair(a, pair);
        return;
    }
    const unsigned x = blockIdx.x;
    const int sub = x % subs, j = x / subs % a.nb, bh = x / subs / a.nb, hk = bh % a.Hk, b = bh / a.Hk;
    const int* const cs = a.chunk_start + (size_t)bh * (a.nb + 1);
    const int c0 = cs[j], n = cs[j + 1] - c0;
    if (n == 1) return;
    const int per = a.D / 4, i = blockIdx.y * 256 + threadIdx.x, which = i / (KB * per), k = i / per % KB, d = 4 * (i % per);
    const int key = j * a.block + sub * KB + k;
    if (which > 1 || key >= a.Lk) return;
    f32x4a s = {0.f, 0.f, 0.f, 0.f};
    const float* p = a.pkv + ((((size_t)bh * a.max_chunks + c0) * subs + sub) * 2 + which) * KB * a.D + (size_t)k * a.D + d;
    const size_t step = (size_t)subs * 2 * KB * a.D;
    int c = 0;
    for (; c + 8 <= n; c += 8) {
        f32x4a v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = *(const f32x4a*)(p + (c + u) * step);
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; c < n; ++c) s += *(const f32x4a*)(p + c * step);
    store_four((T*)(which ? a.dv : a.dk) + (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D + d, s);
}

struct BwdPlan {
    int R, rw, chunks, subs, CH, max_chunks, words, ng, nb;
    size_t o_member, o_chunk, o_pkv, o_pbias, total;      // offsets in the workspace (delta first)
};
static BwdPlan bwd_plan(const scipnp_block_attn_args* a) {
    BwdPlan p = {};
    p.R = a->query_block * (a->Hq / a->Hk);
    p.rw = p.R <= 32 ? 1 : p.R <= 64 ? 2 : 4;
    p.chunks = (p.R + 32 * p.rw - 1) / (32 * p.rw);
    p.subs = a->block / KB;
    p.ng = (a->Lq + a->query_block - 1) / a->query_block;
    p.nb = (a->Lk + a->block - 1) / a->block;
    p.words = (p.ng + 31) / 32;
    // rows a chunk takes: about 2048 workgroups over the whole call, 256 to 8192 rows each, at most 1024 groups in its list
    const long long entries = (long long)p.ng * (a->n_sel < p.nb ? a->n_sel : p.nb);
    long long ch = (entries * p.R * a->B * a->Hk * p.subs / 2048 + 63) / 64 * 64;
    if (ch < 256) ch = 256;
    if (ch > 8192) ch = 8192;
    if (ch > 1024ll * p.R) ch = 1024ll * p.R;
    p.CH = (int)ch;
    const long long mc = p.nb + entries * p.R / p.CH + 1;
    p.max_chunks = (int)(mc < (1ll << 30) ? mc : (1ll << 30));
    const size_t bh = (size_t)a->B * a->Hk;
    auto up = [](size_t v) { return (v + 255) / 256 * 256; };
    size_t at = up((size_t)a->B * a->Hq * a->Lq * 4) + 256;                  // delta, zeros
    p.o_member = at; at += up(bh * ((p.nb + 3) / 4 * 4) * p.words * 4);
    p.o_chunk = at; at += up(bh * (2 * p.nb + 1) * 4);
    p.o_pkv = at; at += up(bh * p.max_chunks * p.subs * 2 * KB * a->D * 4);
    p.o_pbias = at; at += a->num_buckets ? up(bh * p.ng * p.chunks * a->num_buckets * (a->Hq / a->Hk) * 8) : 0;
    p.total = at;
    return p;
}
size_t attn_backward_workspace(const scipnp_block_attn_args* a) { return bwd_plan(a).total; }

template <typename T, int DP, int RW>
static int dq_launch(const Attn& p, int CH, hipStream_t st) {
    using C = DqCfg<T, DP>;
    const size_t set = ((size_t)C::MAIN + C::KP + (size_t)(p.n + 4) / 4 * 16 + (size_t)(p.nbuckets * p.G + 3) / 4 * 16 + (size_t)RW * p.nbuckets * HROW * 4 + 15) / 16 * 16;
    const size_t shared = bias_lut_bytes(p.nbuckets, p.maxd) + 16;
    int sets = 4 / RW;
    while (sets > 1 && shared + sets * set > 163840) sets >>= 1;
    if (shared + sets * set > 163840) return fail(SCIPNP_EINVAL, "block_attn_backward: %zu bytes of LDS needed (fewer buckets or a smaller n_sel)", shared + set);
    static LdsAttrOnce once;
    if (const int rc = once.ensure((const void*)block_attn_dq_kernel<T, DP, RW>, 163840, "block_attn_dq")) return rc;
    const long long items = (long long)p.B * p.Hk * p.ng * p.chunks;
    const unsigned plans = (unsigned)(p.B * p.Hk);
    block_attn_dq_kernel<T, DP, RW><<<plans + xcd_grid((items + sets - 1) / sets), 64 * RW * sets, shared + sets * set, st>>>(p, sets, (int)set, (int)plans, CH);
    return SCIPNP_OK;
}
template <typename T, int DP>
static int bwd_launch(const Attn& p, const BwdPlan& bp, hipStream_t st) {
    const int rc = bp.rw == 1 ? dq_launch<T, DP, 1>(p, bp.CH, st) : bp.rw == 2 ? dq_launch<T, DP, 2>(p, bp.CH, st) : dq_launch<T, DP, 4>(p, bp.CH, st);
    if (rc) return rc;
    using C = DkvCfg<T, DP>;
    const size_t lds = (size_t)C::MAIN + (C::LIST + 8) * 4 + bias_lds(p.nbuckets, p.maxd, p.G);
    if (lds > 163840) return fail(SCIPNP_EINVAL, "block_attn_backward: %zu bytes of LDS needed", lds);
    static LdsAttrOnce once;
    if (const int rc2 = once.ensure((const void*)block_attn_dkv_kernel<T, DP>, 163840, "block_attn_dkv")) return rc2;
    const unsigned gk = (unsigned)((long long)p.B * p.Hk * p.max_chunks * bp.subs);
    block_attn_dkv_kernel<T, DP><<<gk, 256, lds, st>>>(p, bp.subs, div_magic(bp.R), div_magic(p.G));
    return SCIPNP_OK;
}

template <typename T>
static int bwd_run(const Attn& p, const BwdPlan& bp, hipStream_t st) {
    static LdsAttrOnce once;
    if (const int rc = once.ensure((const void*)attn_mark_kernel, 163840, "attn_mark")) return rc;
    const int cap = p.nb < MARK_CAP ? p.nb : MARK_CAP;
    attn_mark_kernel<<<dim3((unsigned)bp.words, (unsigned)(p.B * p.Hk)), 64 * MARK_WAVES, (size_t)(cap + MARK_WAVES * p.n) * 4, st>>>(p, cap);
    int rc;
    if (sizeof(T) == 4 && p.D > 32 && p.D <= 48) rc = bwd_launch<T, sizeof(T) == 4 ? 48 : 64>(p, bp, st);
    else rc = p.D <= 32 ? bwd_launch<T, 32>(p, bp, st) : p.D <= 64 ? bwd_launch<T, 64>(p, bp, st)
                 : p.D <= 96 ? bwd_launch<T, 96>(p, bp, st) : bwd_launch<T, 128>(p, bp, st);
    if (rc) return rc;
    const unsigned joins = (unsigned)(p.nb * bp.subs) * (unsigned)(p.B * p.Hk), parts = (unsigned)((2 * KB * (p.D / 4) + 255) / 256);
    attn_end_kernel<T><<<dim3(joins + (p.dbias ? (p.nbuckets * p.Hq + 3) / 4 : 0), parts), 256, 0, st>>>(p, bp.subs, joins);
    return launch_status("scipnp_block_attn_backward");
}

}  // namespace scipnp

using namespace scipnp;

extern "C" {

int scipnp_block_attn_backward(const scipnp_block_attn_args* a, scipnp_stream_t s) {
    if (const int rc = attn_check(a)) return rc;
    SCIPNP_REQUIRE(a->dout && a->dq && a->dk && a->dv && a->lse && a->lse_rest && a->out32, "backward needs dout, dq, dk, dv, lse, lse_rest and out32");
    SCIPNP_REQUIRE(!a->num_buckets || a->dbias, "backward with a bias needs dbias");
    SCIPNP_REQUIRE((long long)a->num_buckets * a->Hq < (1ll << 24), "too many buckets and query heads");
    SCIPNP_ALIGNED(a->dout); SCIPNP_ALIGNED(a->dq); SCIPNP_ALIGNED(a->dk); SCIPNP_ALIGNED(a->dv); SCIPNP_ALIGNED(a->out32);
    SCIPNP_STRIDES(a->dout_stride, a->dtype);
    const BwdPlan bp = bwd_plan(a);
    SCIPNP_REQUIRE((long long)a->B * a->Hk < 65536 && (long long)a->B * a->Hk * bp.max_chunks * bp.subs < (1ll << 23), "too many query groups or key blocks");
    SCIPNP_REQUIRE((long long)bp.ng * bp.R < (1ll << 30), "too many query rows");
    if (!a->workspace || a->workspace_bytes < bp.total) return fail(SCIPNP_EWORKSPACE, "block_attn_backward: workspace of %zu bytes needed", bp.total);
    SCIPNP_ALIGNED(a->workspace);
    Attn p = attn_params(a);
    char* const w = (char*)a->workspace;
    p.delta = (float*)w;
    p.zeros = (float*)(w + bp.o_member - 256);
    p.member = (unsigned*)(w + bp.o_member);
    p.words = bp.words;
    p.nb4 = (p.nb + 3) / 4 * 4;
    p.chunk_start = (int*)(w + bp.o_chunk);
    p.chunk_rows = p.chunk_start + (size_t)a->B * a->Hk * (p.nb + 1);
    p.max_chunks = bp.max_chunks;
    p.pkv = (float*)(w + bp.o_pkv);
    p.pbias = (double*)(w + bp.o_pbias);
    p.chunks = bp.chunks;
    return a->dtype == SCIPNP_BF16 ? bwd_run<__bf16>(p, bp, (hipStream_t)s)
                                   : bwd_run<float>(p, bp, (hipStream_t)s);
}

}
