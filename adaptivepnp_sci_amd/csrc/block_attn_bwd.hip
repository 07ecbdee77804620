// Attention over selected key blocks, backward, in a fixed order throughout (no floating-point atomics).
//   P = exp(S - lse);  dP = dO V^T;  dS = P (dP - delta),  delta = sum_d dO O (O unrounded)
//   dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO;  dbias[bucket][head] = sum of dS over the bucket's pairs
// Two passes recompute S and dP (7 products of the pairs instead of 5): one per query group for dQ and dbias, one per key block for dK
// and dV, which needs the selection the other way round: a bit for every (key block, query group), then the blocks' query rows cut
// into chunks of equal length, since a first block is chosen by every group and most blocks by few.
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

// ---- delta of every live row (16 lanes a row), and the membership bits cleared for the launch behind it
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(Attn a, float* delta, size_t member_words) {
    const size_t rows = (size_t)a.B * a.Lq * a.Hq;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < member_words; i += (size_t)gridDim.x * 256) a.member[i] = 0;
    for (size_t id = (size_t)blockIdx.x * 16 + (threadIdx.x >> 4); id < rows; id += (size_t)gridDim.x * 16) {
        const int head = (int)(id % a.Hq), tok = (int)(id / a.Hq % a.Lq), b = (int)(id / a.Hq / a.Lq), l16 = threadIdx.x & 15;
        float s = 0.f;
        if (tok < seq_of(a, b).qlen) {
            const T* g = (const T*)a.dout + b * a.sdo.b + (long long)tok * a.sdo.t + head * a.sdo.h;
            for (int d = 4 * l16; d < a.D; d += 64) {
                const f32x4a o = *(const f32x4a*)(a.out32 + id * a.D + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fmaf((float)g[d + e], o[e], s);
            }
        }
        s += __shfl_xor(s, 8, 16);
        s += __shfl_xor(s, 4, 16);
        s += __shfl_xor(s, 2, 16);
        s += __shfl_xor(s, 1, 16);
        if (l16 == 0) delta[((size_t)b * a.Hq + head) * a.Lq + tok] = s;
    }
}

// ---- the selection the other way round: one wave a query group sets its bit in each of its blocks (an OR: no order)
__global__ void __launch_bounds__(256) attn_mark_kernel(Attn a) {
    extern __shared__ int lists[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long item = (long long)blockIdx.x * 4 + wave;
    if (item >= (long long)a.B * a.Hk * a.ng) return;
    int* const list = lists + wave * a.n;
    const int g = (int)(item % a.ng), bh = (int)(item / a.ng);
    const Seq s = seq_of(a, bh / a.Hk);
    const int q0 = g * a.qb, nq = min(a.qb, s.qlen - q0);
    if (nq <= 0) return;
    const int far = a.causal ? min(s.klen, s.shift + q0 + nq) : s.klen;
    const int c = live_blocks(a, a.sel + (size_t)item * a.n, far, list, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = lane; i < c; i += 64) atomicOr(&a.member[((size_t)bh * a.nb + list[i]) * a.words + (g >> 5)], 1u << (g & 31));
}

// ---- chunks of every key block of one (sequence, key head): chunk_start[j] = chunks of the blocks before j
__global__ void __launch_bounds__(256) attn_plan_kernel(Attn a, int* chunk_start, int R, int CH) {
    __shared__ int wsum[4], carry;
    const int bh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* const cs = chunk_start + (size_t)bh * (a.nb + 1);
    if (tid == 0) carry = 0;
    __syncthreads();
    for (int base = 0; base < a.nb; base += 256) {
        const int j = base + tid;
        int c = 0;
        if (j < a.nb) {
            const unsigned* w = a.member + ((size_t)bh * a.nb + j) * a.words;
            for (int i = 0; i < a.words; ++i) c += __popc(w[i]);
            c = (int)(((long long)c * R + CH - 1) / CH);
        }
        int incl = c;
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(incl, off, 64);
            if (lane >= off) incl += o;
        }
        if (lane == 63) wsum[wave] = incl;
        __syncthreads();
        int at = carry + incl - c;
        for (int w = 0; w < wave; ++w) at += wsum[w];
        if (j < a.nb) cs[j] = at;
        __syncthreads();
        if (tid == 0) carry += wsum[0] + wsum[1] + wsum[2] + wsum[3];
        __syncthreads();
    }
    if (tid == 0) cs[a.nb] = carry;
}

// ---- dQ, dbias: the forward's workgroup and tiles
template <typename T, int DP, int RW>
struct DqCfg {
    static constexpr int KS = 4 / RW, NTH = 64 * RW, ST = row_stride<T, DP>();
    static constexpr int TILE = 2 * KT * ST * (int)sizeof(T);
    // private tiles need one buffer; the widest fp32 tiles leave room for one beside the bias sums (then a second barrier)
    static constexpr int BUFS = KS == 4 || (KS == 2 && sizeof(T) == 4 && DP >= 96) ? 1 : 2;
    static constexpr int OST = DP + 4;
    static constexpr int JOIN = KS > 1 ? RW * 32 * OST * 4 : 0;
    static constexpr int TILES = KS * BUFS * TILE;
    static constexpr int MAIN = TILES > JOIN ? TILES : JOIN;
    static constexpr int KP = KS * BUFS * KT * 4;
};
constexpr int HROW = 65;                                  // a bucket's 64 lane sums, rows shifted by a bank

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256) block_attn_dq_kernel(Attn a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = DqCfg<T, DP, RW>;
    using Frag = typename Mat<T>::Frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const long long total = (long long)a.B * a.Hk * a.ng * a.chunks, item = xcd_item(blockIdx.x, total);
    if (item < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, hi = lane >> 5;
    const int rw = wave % RW, ks = wave / RW, tsplit = rw * 64 + lane;
    const int chunk = (int)(item % a.chunks), g = (int)(item / a.chunks % a.ng), bh = (int)(item / a.chunks / a.ng), hk = bh % a.Hk, b = bh / a.Hk;
    const Seq sq = seq_of(a, b);
    const int R = a.qb * a.G, r0 = chunk * 32 * RW;
    const int row = r0 + rw * 32 + li, tok = g * a.qb + row / a.G, gl = row % a.G, head = hk * a.G + gl;
    const bool live = row < R && tok < sq.qlen;
    const int qkey = sq.shift + tok;
    const int lim = !live ? -1 : a.causal ? min(qkey, sq.klen - 1) : sq.klen - 1;
    const bool any = g * a.qb + r0 / a.G < sq.qlen;       // (uniform) a live row in this chunk

    char* const main = smem;
    int* const kp_lds = (int*)(smem + C::MAIN);
    int* const list = (int*)(smem + C::MAIN + C::KP);
    int* const nlist = list + a.n;
    char* const bias_at = smem + C::MAIN + C::KP + (a.n + 4) / 4 * 16;
    const int lut_bytes = bias_lut_bytes(a.nbuckets, a.maxd);
    const Bias bias = load_bias(a, (unsigned char*)bias_at, (float*)(bias_at + lut_bytes), hk, threadIdx.x, 256);
    float* const hist = (float*)(bias_at + lut_bytes + (a.nbuckets * a.G * 4 + 15) / 16 * 16);
    float* const mine = hist + wave * a.nbuckets * HROW + lane;
    for (int i = 0; i < a.nbuckets; ++i) mine[i * HROW] = 0.f;
    if (wave == 0) {
        int c = 0;
        if (any) {
            const int rows_end = min(min(R, r0 + 32 * RW), (sq.qlen - g * a.qb) * a.G);
            const int far = a.causal ? min(sq.klen, sq.shift + g * a.qb + (rows_end - 1) / a.G + 1) : sq.klen;
            c = live_blocks(a, a.sel + ((size_t)bh * a.ng + g) * a.n, far, list, lane);
        }
        if (lane == 0) *nlist = c;
    }
    Frag qf[DP / Mat<T>::K], gf[DP / Mat<T>::K];
    load_frags<T, DP>(live ? (const T*)a.q + b * a.sq.b + (long long)tok * a.sq.t + head * a.sq.h : nullptr, a.D, hi, qf);
    load_frags<T, DP>(live ? (const T*)a.dout + b * a.sdo.b + (long long)tok * a.sdo.t + head * a.sdo.h : nullptr, a.D, hi, gf);
    const size_t stat = ((size_t)b * a.Hq + head) * a.Lq + tok;
    const float lse = live ? a.lse[stat] * LOG2E : 0.f, delta = live ? a.delta[stat] : 0.f;
    const int qp = a.nbuckets && live ? (a.q_pos ? a.q_pos[(size_t)b * a.Lq + tok] : qkey) : 0;
    RowRange range = {live ? qp : INT_MAX, live ? qp : INT_MIN};
    int min_lim = live ? lim : INT_MAX, max_lim = lim;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        range.lo = min(range.lo, __shfl_xor(range.lo, off, 64));
        range.hi = max(range.hi, __shfl_xor(range.hi, off, 64));
        min_lim = min(min_lim, __shfl_xor(min_lim, off, 64));
        max_lim = max(max_lim, __shfl_xor(max_lim, off, 64));
    }
    range.lo = __builtin_amdgcn_readfirstlane(range.lo);
    range.hi = __builtin_amdgcn_readfirstlane(range.hi);
    min_lim = __builtin_amdgcn_readfirstlane(min_lim);
    max_lim = __builtin_amdgcn_readfirstlane(max_lim);
    __syncthreads();

    const int tpb = a.block / KT, ntiles = *nlist * tpb, iters = (ntiles + C::KS - 1) / C::KS;
    const T* const kb = (const T*)a.k + b * a.sk.b + hk * a.sk.h;
    const T* const vb = (const T*)a.v + b * a.sv.b + hk * a.sv.h;
    TileRegs<T, DP, C::NTH> kr, vr;
    int kpr = 0;
    auto key0_of = [&](int it) -> int {
        const int t = it * C::KS + ks;
        if (t >= ntiles) return -1;
        const int blk = t / tpb;
        return list[blk] * a.block + (t - blk * tpb) * KT;
    };
    auto load = [&](int key0) {
        if (key0 < 0) return;
        kr.load(tsplit, a.D, [&](int r) { return key0 + r < sq.klen ? kb + (long long)(key0 + r) * a.sk.t : nullptr; });
        vr.load(tsplit, a.D, [&](int r) { return key0 + r < sq.klen ? vb + (long long)(key0 + r) * a.sv.t : nullptr; });
        if (a.k_pos && tsplit < KT) kpr = key0 + tsplit < sq.klen ? a.k_pos[(size_t)b * a.Lk + key0 + tsplit] : 0;
    };
    f32x16a o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = 0.f;

    int key0 = iters ? key0_of(0) : -1;
    load(key0);
    for (int it = 0; it < iters; ++it) {
        const int buf = C::BUFS == 2 ? (it & 1) : 0;
        T* const kt = (T*)(main + (ks * C::BUFS + buf) * C::TILE);
        T* const vt = kt + KT * C::ST;
        int* const kp = kp_lds + (ks * C::BUFS + buf) * KT;
        if (key0 >= 0) {
            kr.template store<C::ST>(tsplit, kt);
            vr.template store<C::ST>(tsplit, vt);
            if (a.k_pos && tsplit < KT) kp[tsplit] = kpr;
        }
        if constexpr (C::KS < 4) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int cur = key0;
        key0 = it + 1 < iters ? key0_of(it + 1) : -1;
        load(key0);
        if (cur >= 0 && cur <= max_lim) {
            f32x16a s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
            s = mma_rows<T, DP>(kt + li * C::ST, qf, hi, s);
            dp = mma_rows<T, DP>(vt + li * C::ST, gf, hi, dp);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= a.scale2;
            int dist = -1;
            if (a.nbuckets) {
                dist = tile_distance(a, range, cur, a.k_pos ? kp : nullptr, lane);
                if (dist >= 0) {
                    const float bv = bias.tbl[bias.lut[dist] * a.G + gl];
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] += bv;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int k = a.k_pos ? kp[tile_key(r, hi)] : cur + tile_key(r, hi);
                        s[r] += bias.tbl[bias.lut[clamp_dist(k - qp, a.maxd)] * a.G + gl];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = __builtin_amdgcn_exp2f(s[r] - lse);
                s[r] = cur + tile_key(r, hi) <= lim ? p * (dp[r] - delta) : 0.f;
            }
            if (a.dbias) {
                if (dist >= 0) {
                    float sum = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += s[r];
                    mine[bias.lut[dist] * HROW] += sum;
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int k = a.k_pos ? kp[tile_key(r, hi)] : cur + tile_key(r, hi);
                        mine[bias.lut[clamp_dist(k - qp, a.maxd)] * HROW] += s[r];
                    }
                }
            }
            mma_cols<T, DP, C::ST>(kt, s, lane, o);
        }
        if constexpr (C::KS == 4) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else if constexpr (C::BUFS == 1) __syncthreads();
    }
    if (a.dbias) {                                        // the workgroup's sums: a (bucket, head) adds its lanes in order, in fp64
        __syncthreads();
        for (int i = threadIdx.x; i < a.nbuckets * a.G; i += 256) {
            const int n = i / a.G, h = i - n * a.G;
            double sum = 0.0;
            for (int w = 0; w < 4; ++w)
                for (int x = 0; x < 64; ++x)
                    if ((r0 + (w % RW) * 32 + (x & 31)) % a.G == h) sum += (double)hist[(w * a.nbuckets + n) * HROW + x];
            a.pbias[(size_t)item * a.nbuckets * a.G + i] = sum;
        }
    }
    if constexpr (C::KS > 1) {
        float* const obuf = (float*)main + rw * 32 * C::OST;
        __syncthreads();
        for (int k = C::KS - 1; k >= 0; --k) {
            if (ks == k) {
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4a* const p = (f32x4a*)(obuf + li * C::OST + 32 * db + 8 * q + 4 * hi);
                        f32x4a v = f32x4a{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]};
                        if (k < C::KS - 1) v += *p;
                        if (k > 0) *p = v;
                        else
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[db][4 * q + e] = v[e];
                    }
            }
            if (k > 0) __syncthreads();
        }
        if (ks > 0) return;
    }
    if (row >= R || tok >= a.Lq) return;
    T* const dst = (T*)a.dq + (((size_t)b * a.Lq + tok) * a.Hq + head) * a.D;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * db + 8 * q + 4 * hi;
            if (d >= a.D) continue;
            f32x4a v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = live ? o[db][4 * q + e] * a.scale : 0.f;
            if constexpr (sizeof(T) == 2) {
                bf16x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (__bf16)v[e];
                *(bf16x4*)(dst + d) = w;
            } else {
                *(f32x4a*)(dst + d) = v;
            }
        }
#endif
}

// dbias[n][head]: one wave sums the workgroups' partials, every 64th a lane
__global__ void __launch_bounds__(64) attn_dbias_kernel(Attn a) {
    const int n = blockIdx.x / a.Hq, head = blockIdx.x % a.Hq, hk = head / a.G, h = head % a.G, lane = threadIdx.x;
    const size_t per = (size_t)a.ng * a.chunks, row = (size_t)a.nbuckets * a.G;
    double s = 0.0;
    for (int b = 0; b < a.B; ++b) {
        const double* p = a.pbias + ((size_t)(b * a.Hk + hk) * per) * row + (size_t)n * a.G + h;
        for (size_t i = lane; i < per; i += 64) s += p[i * row];
    }
    s = wave_sum_f64(s);
    if (lane == 0) a.dbias[(size_t)n * a.Hq + head] = (float)s;
}

// ---- dK, dV of 64 keys over one chunk of the query rows that chose their block.  Waves: two halves of the keys x two of the row tiles;
// a wave keeps its 32 keys and values in registers (the B operands) and streams rows: S, dP with the rows as A, then dV += dO^T P and
// dK += Q^T dS with the transposed rows as A and the score registers as B.
template <typename T, int DP>
struct DkvCfg {
    static constexpr int ST = row_stride<T, DP>();
    static constexpr int INFO = KT * 20;                  // lse, delta, last key, position, head of each row
    static constexpr int TILE = 2 * KT * ST * (int)sizeof(T) + INFO;
    static constexpr int MAIN = 4 * TILE;                 // two row tiles, two buffers
    static constexpr int OST = DP + 4;
    static constexpr int JOIN = 2 * 32 * OST * 4;
    static_assert(JOIN <= MAIN, "the join reuses the tiles");
    static constexpr int LIST = 1032;                     // query groups of a chunk
};

template <typename T, int DP>
__global__ void __launch_bounds__(256) block_attn_dkv_kernel(Attn a, int CH, int subs, unsigned magic_r, unsigned magic_g) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = DkvCfg<T, DP>;
    using Frag = typename Mat<T>::Frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const long long total = (long long)a.B * a.Hk * a.max_chunks * subs, item = xcd_item(blockIdx.x, total);
    if (item < 0) return;
    const int sub = (int)(item % subs), c = (int)(item / subs % a.max_chunks), bh = (int)(item / subs / a.max_chunks), hk = bh % a.Hk, b = bh / a.Hk;
    const int* const cs = a.chunk_start + (size_t)bh * (a.nb + 1);
    if (c >= cs[a.nb]) return;                            // (uniform)
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 31, hi = lane >> 5, kw = wave & 1, rs = wave >> 1;
    const int tsplit = kw * 64 + lane;
    char* const main = smem;
    int* const list = (int*)(smem + C::MAIN);
    int* const misc = list + C::LIST;                     // block, scan
    char* const bias_at = smem + C::MAIN + (C::LIST + 8) * 4;
    const Bias bias = load_bias(a, (unsigned char*)bias_at, (float*)(bias_at + bias_lut_bytes(a.nbuckets, a.maxd)), hk, tid, 256);
    for (int j = tid; j < a.nb; j += 256)
        if (cs[j] <= c && c < cs[j + 1]) misc[0] = j;
    __syncthreads();
    const int j = misc[0], nchunks = cs[j + 1] - cs[j];
    const int R = a.qb * a.G;
    const Seq sq = seq_of(a, b);
    // the chunk's rows are x0 .. x1 of the block's groups laid end to end; their groups into the list
    const unsigned x0 = (unsigned)(c - cs[j]) * CH;
    int count = 0;
    {
        const unsigned* w = a.member + ((size_t)bh * a.nb + j) * a.words;
        const int e0 = (int)(x0 / R), e1 = (int)((x0 + CH + R - 1) / R);
        for (int base = 0; base < a.words; base += 256) {
            const unsigned bits = base + tid < a.words ? w[base + tid] : 0;
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
    const unsigned x1 = (unsigned)min((long long)x0 + CH, (long long)count * R);
    const int e0 = (int)(x0 / R);

    const int kbase = j * a.block + sub * KB + kw * 32, key = kbase + li;
    const bool klive = key < sq.klen;
    Frag kf[DP / Mat<T>::K], vf[DP / Mat<T>::K];
    load_frags<T, DP>(klive ? (const T*)a.k + b * a.sk.b + (long long)key * a.sk.t + hk * a.sk.h : nullptr, a.D, hi, kf);
    load_frags<T, DP>(klive ? (const T*)a.v + b * a.sv.b + (long long)key * a.sv.t + hk * a.sv.h : nullptr, a.D, hi, vf);
    const int kpos = a.k_pos ? (klive ? a.k_pos[(size_t)b * a.Lk + key] : 0) : key;

    f32x16a dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dk[db][r] = 0.f; dv[db][r] = 0.f; }

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
    TileRegs<T, DP, 128> qr, gr;
    float ilse = 0.f, idelta = 0.f;
    int ilim = -1, iqp = 0, ig = 0;
    auto load = [&](unsigned x) {                         // rows x .. x + 31
        qr.load(tsplit, a.D, [&](int r) -> const T* {
            int tok, gl;
            row_of(x + r, tok, gl);
            return tok < 0 ? nullptr : (const T*)a.q + b * a.sq.b + (long long)tok * a.sq.t + (hk * a.G + gl) * a.sq.h;
        });
        gr.load(tsplit, a.D, [&](int r) -> const T* {
            int tok, gl;
            row_of(x + r, tok, gl);
            return tok < 0 ? nullptr : (const T*)a.dout + b * a.sdo.b + (long long)tok * a.sdo.t + (hk * a.G + gl) * a.sdo.h;
        });
        if (tsplit < KT) {
            int tok, gl;
            row_of(x + tsplit, tok, gl);
            ilim = -1; ilse = idelta = 0.f; iqp = 0; ig = gl;
            if (tok >= 0) {
                const size_t stat = ((size_t)b * a.Hq + hk * a.G + gl) * a.Lq + tok;
                ilse = a.lse[stat] * LOG2E;
                idelta = a.delta[stat];
                ilim = a.causal ? min(sq.shift + tok, sq.klen - 1) : sq.klen - 1;
                iqp = a.q_pos ? a.q_pos[(size_t)b * a.Lq + tok] : sq.shift + tok;
            }
        }
    };
    const int iters = (int)((x1 - x0 + 2 * KT - 1) / (2 * KT));
    load(x0 + rs * KT);
    for (int it = 0; it < iters; ++it) {
        char* const at = main + (rs * 2 + (it & 1)) * C::TILE;
        T* const qt = (T*)at;
        T* const gt = qt + KT * C::ST;
        float* const info = (float*)(at + 2 * KT * C::ST * (int)sizeof(T));
        qr.template store<C::ST>(tsplit, qt);
        gr.template store<C::ST>(tsplit, gt);
        if (tsplit < KT) {
            info[tsplit] = ilse;
            info[KT + tsplit] = idelta;
            ((int*)info)[2 * KT + tsplit] = ilim;
            ((int*)info)[3 * KT + tsplit] = iqp;
            ((int*)info)[4 * KT + tsplit] = ig;
        }
        __syncthreads();
        if (it + 1 < iters) load(x0 + (it + 1) * 2 * KT + rs * KT);
        f32x16a s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
        s = mma_rows<T, DP>(qt + li * C::ST, kf, hi, s);
        dp = mma_rows<T, DP>(gt + li * C::ST, vf, hi, dp);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r4 = 8 * q + 4 * hi;
            const f32x4a lse = *(const f32x4a*)(info + r4), delta = *(const f32x4a*)(info + KT + r4);
            const int4 lim = *(const int4*)((int*)info + 2 * KT + r4);
            const int lims[4] = {lim.x, lim.y, lim.z, lim.w};
            float add[4] = {0.f, 0.f, 0.f, 0.f};
            if (a.nbuckets) {
                const int4 qp = *(const int4*)((int*)info + 3 * KT + r4), gh = *(const int4*)((int*)info + 4 * KT + r4);
                const int qps[4] = {qp.x, qp.y, qp.z, qp.w}, ghs[4] = {gh.x, gh.y, gh.z, gh.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) add[e] = bias.tbl[bias.lut[clamp_dist(kpos - qps[e], a.maxd)] * a.G + ghs[e]];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * q + e;
                const bool see = key <= lims[e];
                const float p = see ? __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, add[e] - lse[e])) : 0.f;
                s[r] = p;
                dp[r] = see ? p * (dp[r] - delta[e]) : 0.f;
            }
        }
        mma_cols<T, DP, C::ST>(gt, s, lane, dv);
        mma_cols<T, DP, C::ST>(qt, dp, lane, dk);
    }
    // the two row halves: 1 into LDS, 0 adds
    float* const obuf = (float*)main + kw * 32 * C::OST;
    auto join = [&](f32x16a (&x)[DP / 32]) {
        __syncthreads();
        if (rs == 1) {
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4a*)(obuf + li * C::OST + 32 * db + 8 * q + 4 * hi) = f32x4a{x[db][4 * q], x[db][4 * q + 1], x[db][4 * q + 2], x[db][4 * q + 3]};
        }
        __syncthreads();
        if (rs == 0) {
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4a v = *(const f32x4a*)(obuf + li * C::OST + 32 * db + 8 * q + 4 * hi);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[db][4 * q + e] += v[e];
                }
        }
    };
    join(dv);
    join(dk);
    if (rs == 1) return;
    const size_t slot = ((size_t)bh * a.max_chunks + c) * subs + sub;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * db + 8 * q + 4 * hi;
                if (d >= a.D) continue;
                f32x4a v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = which ? dv[db][4 * q + e] : dk[db][4 * q + e] * a.scale;
                if (nchunks > 1) {
                    *(f32x4a*)(a.pkv + ((slot * 2 + which) * KB + kw * 32 + li) * a.D + d) = v;
                } else if (key < a.Lk) {
                    T* const dst = (T*)(which ? a.dv : a.dk) + (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D + d;
                    if constexpr (sizeof(T) == 2) {
                        bf16x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = (__bf16)v[e];
                        *(bf16x4*)dst = w;
                    } else {
                        *(f32x4a*)dst = v;
                    }
                }
            }
#endif
}

// blocks that more than one chunk worked on (their partials in order), and blocks that nobody chose (zeros)
template <typename T>
__global__ void __launch_bounds__(256) attn_dkv_join_kernel(Attn a, int subs) {
    const int j = blockIdx.x / subs, sub = blockIdx.x % subs, bh = blockIdx.y, hk = bh % a.Hk, b = bh / a.Hk;
    const int* const cs = a.chunk_start + (size_t)bh * (a.nb + 1);
    const int c0 = cs[j], n = cs[j + 1] - c0;
    if (n == 1) return;
    const int per = a.D / 4;
    for (int i = threadIdx.x; i < KB * per; i += 256) {
        const int k = i / per, d = 4 * (i - k * per), key = j * a.block + sub * KB + k;
        if (key >= a.Lk) continue;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            f32x4a s = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < n; ++c) {
                const size_t slot = ((size_t)bh * a.max_chunks + c0 + c) * subs + sub;
                s += *(const f32x4a*)(a.pkv + ((slot * 2 + which) * KB + k) * a.D + d);
            }
            T* const dst = (T*)(which ? a.dv : a.dk) + (((size_t)b * a.Lk + key) * a.Hk + hk) * a.D + d;
            if constexpr (sizeof(T) == 2) {
                bf16x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (__bf16)s[e];
                *(bf16x4*)dst = w;
            } else {
                *(f32x4a*)dst = s;
            }
        }
    }
}

struct BwdPlan {
    int R, rw, chunks, subs, CH, max_chunks, words, ng, nb;
    size_t o_member, o_chunk, o_pkv, o_pbias, total;      // offsets in the workspace (delta first)
};
static BwdPlan bwd_plan(const scipnp_block_attn_args* a) {
    BwdPlan p = {};
    p.R = a->query_block * (a->Hq / a->Hk);
    p.rw = p.R <= 32 ? 1 : p.R <= 64 ? 2 : 4;
    if (p.rw == 1 && a->dtype == SCIPNP_F32 && a->D > 64) p.rw = 2;       // four private fp32 tiles of 128 would not fit beside the bias sums
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
    size_t at = up((size_t)a->B * a->Hq * a->Lq * 4);
    p.o_member = at; at += up(bh * p.nb * p.words * 4);
    p.o_chunk = at; at += up(bh * (p.nb + 1) * 4);
    p.o_pkv = at; at += up(bh * p.max_chunks * p.subs * 2 * KB * a->D * 4);
    p.o_pbias = at; at += a->num_buckets ? up(bh * p.ng * p.chunks * a->num_buckets * (a->Hq / a->Hk) * 8) : 0;
    p.total = at;
    return p;
}
size_t attn_backward_workspace(const scipnp_block_attn_args* a) { return bwd_plan(a).total; }

template <typename T, int DP, int RW>
static int dq_launch(const Attn& p, unsigned grid, hipStream_t st) {
    using C = DqCfg<T, DP, RW>;
    const size_t lds = (size_t)C::MAIN + C::KP + (size_t)(p.n + 4) / 4 * 16 + bias_lds(p.nbuckets, p.maxd, p.G) + (size_t)4 * p.nbuckets * HROW * 4;
    if (lds > 163840) return fail(SCIPNP_EINVAL, "block_attn_backward: %zu bytes of LDS needed (fewer buckets or a smaller n_sel)", lds);
    static LdsAttrOnce once;
    if (const int rc = once.ensure((const void*)block_attn_dq_kernel<T, DP, RW>, 163840, "block_attn_dq")) return rc;
    block_attn_dq_kernel<T, DP, RW><<<grid, 256, lds, st>>>(p);
    return SCIPNP_OK;
}
template <typename T, int DP>
static int bwd_launch(const Attn& p, const BwdPlan& bp, hipStream_t st) {
    const unsigned gq = xcd_grid((long long)p.B * p.Hk * p.ng * p.chunks);
    int rc;
    if constexpr (sizeof(T) == 4 && DP > 64) rc = bp.rw == 2 ? dq_launch<T, DP, 2>(p, gq, st) : dq_launch<T, DP, 4>(p, gq, st);
    else rc = bp.rw == 1 ? dq_launch<T, DP, 1>(p, gq, st) : bp.rw == 2 ? dq_launch<T, DP, 2>(p, gq, st) : dq_launch<T, DP, 4>(p, gq, st);
    if (rc) return rc;
    using C = DkvCfg<T, DP>;
    const size_t lds = (size_t)C::MAIN + (C::LIST + 8) * 4 + bias_lds(p.nbuckets, p.maxd, p.G);
    if (lds > 163840) return fail(SCIPNP_EINVAL, "block_attn_backward: %zu bytes of LDS needed", lds);
    static LdsAttrOnce once;
    if (const int rc2 = once.ensure((const void*)block_attn_dkv_kernel<T, DP>, 163840, "block_attn_dkv")) return rc2;
    const unsigned gk = xcd_grid((long long)p.B * p.Hk * p.max_chunks * bp.subs);
    block_attn_dkv_kernel<T, DP><<<gk, 256, lds, st>>>(p, bp.CH, bp.subs, div_magic(bp.R), div_magic(p.G));
    return SCIPNP_OK;
}

template <typename T>
static int bwd_run(const Attn& p, const BwdPlan& bp, float* delta, int* chunk_start, hipStream_t st) {
    const size_t rows = (size_t)p.B * p.Lq * p.Hq, words = (size_t)p.B * p.Hk * p.nb * p.words;
    const size_t want = (rows + 15) / 16;
    attn_delta_kernel<T><<<(unsigned)(want < 8192 ? want : 8192), 256, 0, st>>>(p, delta, words);
    const size_t groups = (size_t)p.B * p.Hk * p.ng;
    attn_mark_kernel<<<(unsigned)((groups + 3) / 4), 256, (size_t)4 * p.n * 4, st>>>(p);
    attn_plan_kernel<<<(unsigned)(p.B * p.Hk), 256, 0, st>>>(p, chunk_start, bp.R, bp.CH);
    const int rc = p.D <= 32 ? bwd_launch<T, 32>(p, bp, st) : p.D <= 64 ? bwd_launch<T, 64>(p, bp, st)
                 : p.D <= 96 ? bwd_launch<T, 96>(p, bp, st) : bwd_launch<T, 128>(p, bp, st);
    if (rc) return rc;
    attn_dkv_join_kernel<T><<<dim3((unsigned)(p.nb * bp.subs), (unsigned)(p.B * p.Hk)), 256, 0, st>>>(p, bp.subs);
    if (p.dbias) attn_dbias_kernel<<<(unsigned)(p.nbuckets * p.Hq), 64, 0, st>>>(p);
    return launch_status("scipnp_block_attn_backward");
}

}  // namespace scipnp

using namespace scipnp;

extern "C" {

int scipnp_block_attn_backward(const scipnp_block_attn_args* a, scipnp_stream_t s) {
    if (const int rc = attn_check(a)) return rc;
    SCIPNP_REQUIRE(a->dout && a->dq && a->dk && a->dv && a->lse && a->out32, "backward needs dout, dq, dk, dv, lse and out32");
    SCIPNP_REQUIRE(!a->num_buckets || a->dbias, "backward with a bias needs dbias");
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
    p.member = (unsigned*)(w + bp.o_member);
    p.words = bp.words;
    p.chunk_start = (int*)(w + bp.o_chunk);
    p.max_chunks = bp.max_chunks;
    p.pkv = (float*)(w + bp.o_pkv);
    p.pbias = (double*)(w + bp.o_pbias);
    p.chunks = bp.chunks;
    return a->dtype == SCIPNP_BF16 ? bwd_run<__bf16>(p, bp, (float*)w, (int*)(w + bp.o_chunk), (hipStream_t)s)
                                   : bwd_run<float>(p, bp, (float*)w, (int*)(w + bp.o_chunk), (hipStream_t)s);
}

}
