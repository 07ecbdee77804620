// Attention over selected key blocks, forward.  One workgroup of RW waves holds up to 32 * RW rows (queries x heads of a key head) of
// one query group, 32 a wave, and passes once over its part of the selected key tiles (32 keys of K and V, two buffers) with a running
// maximum and sum; the parts of a group (few rows, many keys: a decoding step) are joined by a second launch.
//
// The scores are in units of ln 2: p = exp2(fma(s, scale log2 e, bias log2 e - m)), one fused multiply-add and one v_exp_f32 a score
// where the tile has one bucket and no mask.  The maximum m is moved only when a tile exceeds it by 2^8: until then p <= 2^8, which
// costs no accuracy in floating point, and the accumulators are not rescaled.
//
// What it is bound by, measured (in a program that has run for a while: the first dozen launches behind a pause take a fifth longer):
//   bf16, 128 wide, 16384 queries of 32 heads over 8 key heads, groups of 16 queries, 16 blocks of 64 each: 451 us; 590 TFLOP/s of one score and
//     one value product a pair, 890 of the three it does (P in two parts), against 1150 of a large matrix product.  A tile is 768 cycles of
//     matrix work and about 190 vector instructions, 16 of them exponentials (one part: 512 and 140, 382 us); three waves a SIMD (168 registers,
//     50 KB of LDS a workgroup) overlap the two in part.  LDS is busy 18 % of the time and has no bank conflicts.  64 rows a wave
//     were slower: the accumulators no longer fit beside the operands.
//   fp32, 48 wide, 131072 tokens, 16 blocks of 64: 237 us, 109 TFLOP/s against 133; four workgroups a CU are a round of three and one of one.
//     56 wide (the non-local prior, 2 x 147968 tokens): 738 us, 92 TFLOP/s, and 105 with the padding to 64 that it multiplies.
//   bf16, 128 wide, one token of 16 sequences, 64 blocks of 64: 48 us + 4.9 of the join, 5.6 TB/s of the keys and values read.
//   fp32 of that: 166 us, 3.2 TB/s; the tiles of 128 columns leave LDS for two waves a CU.
//   Workgroups in contiguous eighths a die were an eighth faster at 2 x 4096 bf16 tokens, 16 heads of 64, than in turn over the dies.
#include <type_traits>
#include "block_attn.hpp"

namespace scipnp {

// LEAN, bf16 of 96 and 128 columns and two waves a pair of tiles: three waves a SIMD instead of two (191 instead of 199 us at 8192 queries of
// 32 heads of 96 in groups of 16, 452 instead of 465 for the first case above).  V is read behind the softmax, 64 columns at a time, which
// saves the registers, and there is one buffer of V, which saves the LDS: it is asked for when its tile's scores begin.  Not where
// there is no third workgroup for a CU (52 us instead of 49 at 4096 queries of 16 heads of 128), nor with P in three parts of 128 columns (30
// registers would go to scratch in the loop), nor for one wave a set (LDS), nor for four (101 us instead of 96 at 8192 queries of 16 heads of 96 in
// groups of 64, 119 instead of 109 at 128 wide).
template <typename T, int DP, int RW, bool SAVE>
constexpr bool can_be_lean() { return sizeof(T) == 2 && DP > 64 && RW == 2 && !(SAVE && DP == 128); }
template <typename T, int DP, int RW, bool LEAN>
struct FwdCfg {
    static constexpr bool ONE_V = LEAN;
    static constexpr int BYTES = DmaTile<T, DP>::BYTES;
    static constexpr int MAIN = (ONE_V ? 3 : 4) * BYTES;                      // two K, one or two V
    static constexpr int KP = 2 * KT * 4;
};

// A workgroup holds `sets` sets of RW waves, each with work of its own: four waves a workgroup land one on each SIMD of a CU, where
// workgroups of one or two leave some SIMDs with three waves and some with one.
template <typename T, int DP, int RW, bool SAVE, bool LEAN>          // SAVE: out32 wanted (a training pass)
__global__ void __launch_bounds__(256, LEAN || (sizeof(T) == 4 && DP == 64 && RW > 1) ? 3 : 2)   // (fp32 of 64: 168 registers, a few spilt outside the loop)
block_attn_kernel(Attn a, int sets, int set_bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = FwdCfg<T, DP, RW, LEAN>;
    using Frag = typename Mat<T>::Frag;
    constexpr int NB = (DP + 31) / 32;
    constexpr bool ONE_V = C::ONE_V;
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    const long long total = (long long)a.B * a.Hk * a.ng * a.chunks * a.splits;
    const long long first = xcd_item(blockIdx.x, (total + sets - 1) / sets);
    if (first < 0) return;
    const int lane = threadIdx.x & 63, li = lane & 31, hi = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int set = wave / RW, rw = wave % RW, tset = rw * 64 + lane;
    const bool there_is = first * sets + set < total;
    unsigned it0 = there_is ? (unsigned)(first * sets + set) : 0;
    const int part = it0 % a.splits; it0 /= a.splits;
    const int chunk = it0 % a.chunks; it0 /= a.chunks;
    const int g = it0 % a.ng, bh = it0 / a.ng, hk = bh % a.Hk, b = bh / a.Hk;
    const Seq sq = seq_of(a, b);
    const int R = a.qb * a.G, r0 = chunk * 32 * RW;
    const bool any = there_is && g * a.qb + r0 / a.G < sq.qlen;             // a live row in this chunk
    int row = r0 + rw * 32 + li, tok = g * a.qb + row / a.G, gl = row % a.G, head = hk * a.G + gl;
    bool live = there_is && row < R && tok < sq.qlen;
    const int qkey = sq.shift + tok;                      // key position of the row
    const int lim = !live ? -1 : a.causal ? min(qkey, sq.klen - 1) : sq.klen - 1;       // its last visible key

    unsigned char* const lut = (unsigned char*)smem_all;  // shared by the sets; then each set's own
    char* const smem = smem_all + bias_lut_bytes(a.nbuckets, a.maxd) + 16 + set * set_bytes;
    int* const longest = (int*)(smem_all + bias_lut_bytes(a.nbuckets, a.maxd));
    int* const kp_lds = (int*)(smem + C::MAIN);
    int* const list = (int*)(smem + C::MAIN + C::KP);
    int* const nlist = list + a.n;
    const Bias bias = load_bias(a, lut, (float*)(smem + C::MAIN + C::KP + (a.n + 4) / 4 * 16), hk, tset, 64 * RW);
    if (threadIdx.x == 0) longest[0] = longest[1] = 0;
    if (rw == 0) {
        int c = 0;
        if (any) {
            const int rows_end = min(min(R, r0 + 32 * RW), (sq.qlen - g * a.qb) * a.G);
            const int far = a.causal ? min(sq.klen, sq.shift + g * a.qb + (rows_end - 1) / a.G + 1) : sq.klen;
            c = live_tiles(a, a.sel + ((size_t)bh * a.ng + g) * a.n, far, list, lane);
        }
        if (lane == 0) *nlist = c;
    }
    Frag qf[DP / Mat<T>::K];
    load_frags<T, DP>(live ? (const T*)a.q + b * a.sq.b + (long long)tok * a.sq.t + head * a.sq.h : nullptr, a.D, hi, qf);
    const int qp = a.nbuckets && live ? (a.q_pos ? a.q_pos[(size_t)b * a.Lq + tok] : qkey) : 0;
    const RowRange range = {wave_min(live ? qp : INT_MAX), wave_max(live ? qp : INT_MIN)};
    const int min_lim = wave_min(live ? lim : INT_MAX);
    const unsigned ks = (unsigned)(a.sk.t * (long long)sizeof(T)), vs = (unsigned)(a.sv.t * (long long)sizeof(T));
    DmaOffsets<T, DP, RW> ko, vo;
    ko.init(rw, lane, ks, a.D);
    vo.init(rw, lane, vs, a.D);
    __syncthreads();

    const int tpb = a.block / KT, ntiles = __builtin_amdgcn_readfirstlane(*nlist);
    const int per = (ntiles + a.splits - 1) / a.splits, t_begin = part * per, count = max(0, min(ntiles, t_begin + per) - t_begin);
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
    int blk, off;                                         // the next tile to ask for
    auto next_key = [&]() -> int {
        const int key = __builtin_amdgcn_readfirstlane(list[blk]) * a.block + off;
        off += KT;
        if (off == a.block) { off = 0; ++blk; }
        return key;
    };
    auto issue = [&](int key0, int buf) {
        const int there = min(KT, sq.klen - key0);
        ko.issue(kb + (long long)key0 * a.sk.t, there, ks, a.D, smem + buf * C::BYTES, rw);
        if constexpr (!ONE_V) vo.issue(vb + (long long)key0 * a.sv.t, there, vs, a.D, smem + (2 + buf) * C::BYTES, rw);
        if (a.k_pos && rw == 0) issue_positions(a.k_pos + (size_t)b * a.Lk + key0, there, kp_lds + buf * KT, lane);
    };
    const int far = 2 * a.maxd;                           // the two ends, where most tiles lie: their bias in registers
    const float bias_lo = a.nbuckets ? bias.tbl[bias.lut[0] * a.G + gl] : 0.f, bias_hi = a.nbuckets ? bias.tbl[bias.lut[far] * a.G + gl] : 0.f;
    Acc<T, DP> sums;
    float m, l;
    f32x16a o[NB];
    // One pass, and a careful second one where the first left a sum that is no number.  An infinity or a NaN among the values meets weights of
    // zero (masked keys) and parts of a weight that are zero or negative, and 0 x inf is none: the second pass has zeros in their
    // place; they come behind it, to the rows that see their keys.  A score that is no number stays none when a bias of -infinity masks it:
    // the second pass replaces it.  (What the first pass costs for this is its test, 16 operations a column block.)
    bool masks = false;                                   // a bias of this key head masks (uniform)
    auto pass = [&](auto second) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(second)::value;
    sums.zero();
    m = -INFINITY, l = 0.f;
    blk = t_begin / tpb, off = (t_begin - blk * tpb) * KT;
    int key0 = 0;
    if (count > 0) {
        key0 = next_key();
        issue(key0, 0);
    }
    for (int t = 0; t < count; ++t) {
        const int buf = t & 1, cur = key0;
        int* const kp = kp_lds + buf * KT;
        dma_wait<RW>();                                   // this tile has landed, and everyone is done with the other buffer
        if constexpr (ONE_V) vo.issue(vb + (long long)cur * a.sv.t, min(KT, sq.klen - cur), vs, a.D, smem + 2 * C::BYTES, rw);
        if (t + 1 < count) {
            key0 = next_key();
            issue(key0, buf ^ 1);
        }
        const char* const kt = smem + buf * C::BYTES;
        char* const v_at = smem + (ONE_V ? 2 : 2 + buf) * C::BYTES;
        if constexpr (CAREFUL && !ONE_V) {
            scrub<T, DP, RW>(v_at, rw, lane);
            dma_wait<RW>();
        }
        // (a wave with products to issue goes before one in its softmax: 73.6 -> 69.5 us in training at 2 x 4096 tokens, 16 heads of 64)
        __builtin_amdgcn_s_setprio(1);
        f32x16a s = dma_rows<T, DP, LEAN>(kt, qf, lane);
        __builtin_amdgcn_s_setprio(0);
        ColTile<T, DP, LEAN && NB == 4 ? 2 : NB> vt;
        if constexpr (LEAN) vt.at(v_at, lane);
        else vt.read(v_at, lane);
        const int dist = a.nbuckets ? tile_distance(a, range, cur, a.k_pos ? kp : nullptr, lane) : 0;
        const bool masked = cur + KT - 1 > min_lim;
        float c = a.scale2, add = 0.f;
        if (dist >= 0 && a.nbuckets) add = !LEAN && dist == 0 ? bias_lo : !LEAN && dist == far ? bias_hi : bias.tbl[bias.lut[dist] * a.G + gl];
        if (dist < 0 || masked || c < 0.f || (CAREFUL && masks)) {              // the scores one by one
            if (dist < 0) {
                constexpr int N = LEAN ? 8 : 16;          // (half of them at a time takes fewer registers)
#pragma unroll
                for (int r0 = 0; r0 < 16; r0 += N) {
                    float x[N];
                    tile_bias(a, bias, cur, a.k_pos ? kp : nullptr, qp, gl, hi, x, r0);
                    if constexpr (CAREFUL)
#pragma unroll
                        for (int r = 0; r < N; ++r) s[r0 + r] = x[r] == -INFINITY ? 0.f : s[r0 + r];
#pragma unroll
                    for (int r = 0; r < N; ++r) s[r0 + r] = fmaf(s[r0 + r], c, x[r]);
                    if constexpr (LEAN) __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                if constexpr (CAREFUL)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = add == -INFINITY ? 0.f : s[r];
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, add);
            }
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = cur + tile_key(r, hi) <= lim ? s[r] : -INFINITY;
            }
            c = 1.f;
            add = 0.f;
        }
        float mt = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
        mt = fmaf(mt, c, add);
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        if (__ballot(mt > m + 8.f)) {
            const float mn = fmaxf(m, mt), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= alpha;
            sums.scale(alpha);
        }
        const float shift = add - (m == -INFINITY ? 0.f : m);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, shift));
            sum[r & 3] += s[r];
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // bf16: P in two parts, off by 2^-16 of each probability.  One part, 2^-8, is off by as much as the output's own rounding (16384 queries
        // of 32 x 128: error 0.0022 of the result instead of 0.0016).  With out32 wanted it is taken whole, in three: delta = sum dO O
        // enters every score's gradient, and the sums of dbias cancel down to its error
        if constexpr (ONE_V) {
            dma_wait_but<DmaOffsets<T, DP, RW>::N>(t + 1 < count);
            if constexpr (CAREFUL) {
                scrub<T, DP, RW>(v_at, rw, lane);
                dma_wait<RW>();
            }
        }
        __builtin_amdgcn_s_setprio(1);
        if constexpr (LEAN) vt.read(v_at, lane);
        const Weights<T, SAVE ? 3 : 2> w(s);
        vt.mma(w, sums);
        if constexpr (LEAN && NB == 4) {
            vt.read(v_at, lane, 2);
            vt.mma(w, sums, 2);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    for (int t = count; t < trips; ++t) {                 // (the other sets' barriers)
        dma_wait<RW>();
        if constexpr (ONE_V) dma_wait<RW>();
        if constexpr (CAREFUL) dma_wait<RW>();
    }
    l += __shfl_xor(l, 32, 64);
    sums.blocks(o);
    };
    pass(std::false_type{});
    bool careful;
    {
        float none[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) none[r & 3] = fmaf(o[db][r], 0.f, none[r & 3]);
        const bool number = l - l == 0.f;                 // (if not, the row is none unless masked keys made it so)
        careful = __ballot(live && (!number || (none[0] + none[1]) + (none[2] + none[3]) != 0.f)) != 0;
        if (careful) {
            for (int i = lane; i < a.nbuckets * a.G; i += 64) masks |= bias.tbl[i] == -INFINITY;
            masks = __ballot(masks) != 0;
            careful = masks || __ballot(live && number && (none[0] + none[1]) + (none[2] + none[3]) != 0.f) != 0;
        }
        if constexpr (RW > 1) {                           // waves that share tiles go through them together
            if (careful && lane == 0) longest[1] = 1;
            __syncthreads();
            careful = __builtin_amdgcn_readfirstlane(longest[1]) != 0;
        }
    }
    if (careful) pass(std::true_type{});
    const Attn& z = late_args();                          // (what only the end needs is read again there: the loop's scalars fit the registers)
    if constexpr (LEAN) {                                 // (the row's place as well: no register holds it through the loop)
        int x = li;
        asm volatile("" : "+v"(x));
        row = r0 + rw * 32 + x;
        tok = g * z.qb + row / z.G;
        gl = row % z.G;
        head = hk * z.G + gl;
        live = there_is && row < R && tok < sq.qlen;
    }
    // Values that are no numbers, to the rows that see their keys, by plain loads
    if (careful) {
        const T* const qr = (const T*)z.q + b * z.sq.b + tok * z.sq.t + head * z.sq.h;
        for (int t = t_begin; t < t_begin + count; ++t) {
            const int cur = __builtin_amdgcn_readfirstlane(list[t / tpb]) * z.block + t % tpb * KT, there = min(KT, sq.klen - cur);
            bool bad = false;
            for (int j = 0; j < there; ++j)
                for (int d = lane; d < z.D; d += 64) bad |= !(fabsf((float)vb[(cur + j) * z.sv.t + d]) < INFINITY);
            if (!__ballot(bad)) continue;
            for (int j = 0; j < there; ++j) {
                if (!live || cur + j > lim) continue;
                const T* const kr = kb + (cur + j) * z.sk.t;
                const T* const vr = vb + (cur + j) * z.sv.t;
                float x = 0.f, add = 0.f;
                if (z.nbuckets) {
                    const int kp = z.k_pos ? z.k_pos[(size_t)b * z.Lk + cur + j] : cur + j;
                    add = bias.tbl[bias.lut[clamp_dist(kp - qp, z.maxd)] * z.G + gl];
                    if (add == -INFINITY) continue;
                }
                for (int d = 0; d < z.D; ++d) x = fmaf((float)kr[d], (float)qr[d], x);
                const float p = __builtin_amdgcn_exp2f(fmaf(x, z.scale2, add) - (m == -INFINITY ? 0.f : m));
                each_four<T, DP>(hi, [&](int d, auto at) {
                    if (d >= z.D) return;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = (float)vr[d + e];
                        o[at(e) >> 4][at(e) & 15] = fmaf(p, fabsf(v) < INFINITY ? 0.f : v, o[at(e) >> 4][at(e) & 15]);
                    }
                });
            }
        }
    }

    const size_t id = ((size_t)b * z.Lq + tok) * z.Hq + head;
    if (!live) {                                          // (a row behind qlen; the join takes care of it where there is one)
        if (there_is && z.zero_rest && z.splits == 1 && row < R && tok < z.Lq) {
            T* const out = (T*)z.out + b * z.so.b + (long long)tok * z.so.t + head * z.so.h;
            for (int d = 4 * hi; d < z.D; d += 8) store_four(out + d, f32x4a{0.f, 0.f, 0.f, 0.f});
        }
        return;
    }
    if (z.splits > 1) {
        const size_t rows = (size_t)z.B * z.Lq * z.Hq;
        if (hi == 0) *(float2*)(z.pml + 2 * (part * rows + id)) = make_float2(m, l);
        float* const po = z.po + (part * rows + id) * z.D;
        each_four<T, DP>(hi, [&](int d, auto at) {
            if (d < z.D) *(f32x4a*)(po + d) = f32x4a{o[at(0) >> 4][at(0) & 15], o[at(1) >> 4][at(1) & 15], o[at(2) >> 4][at(2) & 15], o[at(3) >> 4][at(3) & 15]};
        });
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);             // (a NaN sum stays one)
    T* const out = (T*)z.out + b * z.so.b + (long long)tok * z.so.t + head * z.so.h;
    each_four<T, DP>(hi, [&](int d, auto at) {
        if (d >= z.D) return;
        f32x4a v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[at(e) >> 4][at(e) & 15] * inv;
        store_four(out + d, v);
        if constexpr (SAVE) *(f32x4a*)(z.out32 + id * z.D + d) = v;
    });
    if (z.lse && hi == 0) store_lse(z, ((size_t)b * z.Hq + head) * z.Lq + tok, m, l);
#endif
}

// joins the parts of a row's keys (at most 64: a lane each for their maxima and sums): one wave a row, the parts in order.  Latency:
// 4.8 us for 512 rows of 128 in 8 parts (8.6 with the maxima read one after the other)
template <typename T>
__global__ void __launch_bounds__(256) block_attn_join_kernel(Attn a) {
    const size_t rows = (size_t)a.B * a.Lq * a.Hq, id = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= rows) return;
    const int lane = threadIdx.x & 63, head = (int)(id % a.Hq), tok = (int)(id / a.Hq % a.Lq), b = (int)(id / a.Hq / a.Lq);
    T* const out = (T*)a.out + b * a.so.b + (long long)tok * a.so.t + head * a.so.h;
    if (tok >= seq_of(a, b).qlen) {
        if (a.zero_rest)
            for (int d = lane; d < a.D; d += 64) out[d] = (T)0.f;
        return;
    }
    const float2 ml = lane < a.splits ? *(const float2*)(a.pml + 2 * (lane * rows + id)) : make_float2(-INFINITY, 0.f);
    float M = ml.x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    const float Ms = M == -INFINITY ? 0.f : M, f = __builtin_amdgcn_exp2f(ml.x - Ms);
    float L = ml.y * f;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) L += __shfl_xor(L, off, 64);
    const float* po = a.po + id * a.D;
    float s[2] = {0.f, 0.f};
    for (int p0 = 0; p0 < a.splits; p0 += 8) {
        float v[8][2];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) v[u][i] = p0 + u < a.splits && lane + 64 * i < a.D ? po[(p0 + u) * rows * a.D + lane + 64 * i] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = __shfl(f, p0 + u, 64);
#pragma unroll
            for (int i = 0; i < 2; ++i) s[i] = p0 + u < a.splits ? fmaf(v[u][i], w, s[i]) : s[i];
        }
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + 64 * i;
        if (d >= a.D) continue;
        const float v = s[i] * inv;
        out[d] = (T)v;
        if (a.out32) a.out32[id * a.D + d] = v;
    }
    if (a.lse && lane == 0) store_lse(a, ((size_t)b * a.Hq + head) * a.Lq + tok, M, L);
}

static int row_waves(const scipnp_block_attn_args* a) {
    const int R = a->query_block * (a->Hq / a->Hk);
    return R <= 32 ? 1 : R <= 64 ? 2 : 4;
}

// parts of a group's keys: enough waves for four on every CU, none with fewer than two tiles (a serving step over 1024
// keys of 64: 11.9 + 4.0 us with four, 9.8 + 4.5 with two, 8.4 + 6.1 with one)
static int attn_splits(const scipnp_block_attn_args* a) {
    const int rw = row_waves(a), R = a->query_block * (a->Hq / a->Hk);
    const long long groups = (long long)a->B * a->Hk * ((a->Lq + a->query_block - 1) / a->query_block) * ((R + 32 * rw - 1) / (32 * rw));
    const int nb = (a->Lk + a->block - 1) / a->block;
    const long long tiles = (long long)(a->n_sel < nb ? a->n_sel : nb) * (a->block / KT);
    long long want = 1024 / (groups * rw), most = tiles / 2;
    if (want > most) want = most;
    if (want > 64) want = 64;
    return want < 1 ? 1 : (int)want;
}

int attn_check(const scipnp_block_attn_args* a) {
    SCIPNP_BLOCK_SIZE(a, scipnp_block_attn_args);
    SCIPNP_REQUIRE(a->dtype == SCIPNP_F32 || a->dtype == SCIPNP_BF16, "dtype %d: 0 (float32) or 1 (bfloat16)", a->dtype);
    SCIPNP_REQUIRE(a->B > 0 && a->Lq > 0 && a->Lk > 0 && a->Hk > 0 && a->Hq > 0, "B, Lq, Lk, Hq, Hk must be positive");
    SCIPNP_REQUIRE(a->Hq % a->Hk == 0, "%d query heads are no multiple of %d key heads", a->Hq, a->Hk);
    SCIPNP_REQUIRE(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, "head size %d: a multiple of 8 up to 128", a->D);
    SCIPNP_REQUIRE(a->block > 0 && a->block <= 65536 && a->block % 64 == 0, "block %d: a multiple of 64 up to 65536", a->block);
    SCIPNP_REQUIRE(a->query_block > 0 && a->query_block <= 1024, "query_block %d: 1 to 1024", a->query_block);
    SCIPNP_REQUIRE(a->n_sel > 0 && a->n_sel <= 1024, "n_sel %d: 1 to 1024", a->n_sel);
    SCIPNP_REQUIRE(a->Lk <= (1 << 30) && a->Lq <= (1 << 30), "sequences of at most 2^30 tokens");
    SCIPNP_REQUIRE(a->q && a->k && a->v && a->sel, "null q, k, v or sel");
    SCIPNP_REQUIRE(a->num_buckets >= 0 && a->num_buckets <= 64, "%d buckets: at most 64", a->num_buckets);
    if (a->num_buckets) {
        SCIPNP_REQUIRE(a->bias && a->bucket_of, "buckets need bias and bucket_of");
        SCIPNP_REQUIRE(a->max_distance > 0 && a->max_distance <= 4096, "max_distance %d: 1 to 4096", a->max_distance);
        SCIPNP_REQUIRE((long long)a->num_buckets * (a->Hq / a->Hk) <= 2048, "buckets times query heads of a key head: at most 2048");
    }
    SCIPNP_ALIGNED(a->q); SCIPNP_ALIGNED(a->k); SCIPNP_ALIGNED(a->v);
    SCIPNP_STRIDES(a->q_stride, a->dtype); SCIPNP_STRIDES(a->k_stride, a->dtype); SCIPNP_STRIDES(a->v_stride, a->dtype);
    SCIPNP_REQUIRE(a->k_stride[1] < (1 << 24) && a->v_stride[1] < (1 << 24), "token strides of k and v: below 2^24 elements");
    const long long rows = (long long)a->query_block * (a->Hq / a->Hk);
    SCIPNP_REQUIRE((long long)a->B * a->Hk * ((a->Lq + a->query_block - 1) / a->query_block) * ((rows + 31) / 32) < (1ll << 23), "too many query groups");
    return SCIPNP_OK;
}

Attn attn_params(const scipnp_block_attn_args* a) {
    Attn p = {};
    p.B = a->B; p.Lq = a->Lq; p.Lk = a->Lk; p.Hq = a->Hq; p.Hk = a->Hk; p.G = a->Hq / a->Hk; p.D = a->D; p.block = a->block;
    p.qb = a->query_block; p.n = a->n_sel; p.causal = a->causal; p.nbuckets = a->num_buckets; p.maxd = a->num_buckets ? a->max_distance : 0;
    p.nb = (a->Lk + a->block - 1) / a->block; p.ng = (a->Lq + a->query_block - 1) / a->query_block;
    p.chunks = p.splits = 1;
    p.scale = a->scale;
    p.scale2 = a->scale * LOG2E;
    p.zero_rest = a->zero_rest;
    p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out; p.dout = a->dout;
    p.sq = strides_of(a->q_stride); p.sk = strides_of(a->k_stride); p.sv = strides_of(a->v_stride); p.so = strides_of(a->out_stride);
    p.sdo = strides_of(a->dout_stride);
    p.sel = a->sel; p.qlen = a->qlen; p.klen = a->klen;
    p.bucket_of = a->bucket_of; p.q_pos = a->num_buckets ? a->q_pos : nullptr; p.k_pos = a->num_buckets ? a->k_pos : nullptr; p.bias = a->bias;
    p.lse = a->lse; p.lse_rest = a->lse_rest; p.out32 = a->out32;
    p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.dbias = a->num_buckets ? a->dbias : nullptr;
    return p;
}

template <typename T, int DP, int RW, bool SAVE, bool LEAN>
static int fwd_launch(const Attn& p, hipStream_t st) {
    using C = FwdCfg<T, DP, RW, LEAN>;
    const size_t set = ((size_t)C::MAIN + C::KP + (size_t)(p.n + 4) / 4 * 16 + (size_t)p.nbuckets * p.G * 4 + 15) / 16 * 16;
    const size_t shared = bias_lut_bytes(p.nbuckets, p.maxd) + 16;
    int sets = 4 / RW;
    while (sets > 1 && shared + sets * set > 163840) sets >>= 1;
    static LdsAttrOnce once;
    if (const int rc = once.ensure((const void*)block_attn_kernel<T, DP, RW, SAVE, LEAN>, 163840, "block_attn")) return rc;
    const long long items = (long long)p.B * p.Hk * p.ng * p.chunks * p.splits;
    block_attn_kernel<T, DP, RW, SAVE, LEAN><<<xcd_grid((items + sets - 1) / sets), 64 * RW * sets, shared + sets * set, st>>>(p, sets, (int)set);
    return SCIPNP_OK;
}
template <typename T, int DP, int RW, bool SAVE>
static int fwd_pick(const Attn& p, hipStream_t st) {
    if constexpr (can_be_lean<T, DP, RW, SAVE>()) {        // (more than two workgroups of four waves for each of 256 CUs)
        if ((long long)p.B * p.Hk * p.ng * p.chunks * p.splits > 512 * 2) return fwd_launch<T, DP, RW, SAVE, true>(p, st);
    }
    return fwd_launch<T, DP, RW, SAVE, false>(p, st);
}
template <typename T, int DP>
static int fwd_rows(const Attn& p, int rw, hipStream_t st) {
    if (p.out32) return rw == 1 ? fwd_pick<T, DP, 1, true>(p, st) : rw == 2 ? fwd_pick<T, DP, 2, true>(p, st) : fwd_pick<T, DP, 4, true>(p, st);
    return rw == 1 ? fwd_pick<T, DP, 1, false>(p, st) : rw == 2 ? fwd_pick<T, DP, 2, false>(p, st) : fwd_pick<T, DP, 4, false>(p, st);
}
template <typename T>
static int fwd_dim(const Attn& p, int rw, hipStream_t st) {
    if constexpr (sizeof(T) == 4)                          // fp32 products are the cost: 33 to 48 columns as 48 in the score product
        if (p.D > 32 && p.D <= 48) return fwd_rows<T, 48>(p, rw, st);
    return p.D <= 32 ? fwd_rows<T, 32>(p, rw, st) : p.D <= 64 ? fwd_rows<T, 64>(p, rw, st)
         : p.D <= 96 ? fwd_rows<T, 96>(p, rw, st) : fwd_rows<T, 128>(p, rw, st);
}

size_t attn_backward_workspace(const scipnp_block_attn_args* a);

}  // namespace scipnp

using namespace scipnp;

extern "C" {

size_t scipnp_block_attn_workspace_bytes(const scipnp_block_attn_args* a, int backward) {
    if (attn_check(a) != SCIPNP_OK) return 0;
    if (backward) return attn_backward_workspace(a);
    const int s = attn_splits(a);
    return s > 1 ? (size_t)s * a->B * a->Lq * a->Hq * (a->D + 2) * 4 : 0;
}

int scipnp_block_attn(const scipnp_block_attn_args* a, scipnp_stream_t s) {
    if (const int rc = attn_check(a)) return rc;
    SCIPNP_REQUIRE(a->out, "null out");
    SCIPNP_ALIGNED(a->out); SCIPNP_ALIGNED(a->out32);
    SCIPNP_STRIDES(a->out_stride, a->dtype);
    const hipStream_t st = (hipStream_t)s;
    Attn p = attn_params(a);
    const int rw = row_waves(a), R = p.qb * p.G;
    p.chunks = (R + 32 * rw - 1) / (32 * rw);
    p.splits = attn_splits(a);
    if (p.splits > 1) {
        if (!a->workspace || a->workspace_bytes < scipnp_block_attn_workspace_bytes(a, 0))
            return fail(SCIPNP_EWORKSPACE, "block_attn: workspace of %zu bytes needed", scipnp_block_attn_workspace_bytes(a, 0));
        SCIPNP_ALIGNED(a->workspace);
        p.po = (float*)a->workspace;
        p.pml = p.po + (size_t)p.splits * a->B * a->Lq * a->Hq * a->D;
    }
    if (const int rc = a->dtype == SCIPNP_BF16 ? fwd_dim<__bf16>(p, rw, st) : fwd_dim<float>(p, rw, st)) return rc;
    if (p.splits > 1) {
        const unsigned jg = (unsigned)(((size_t)p.B * p.Lq * p.Hq + 3) / 4);
        if (a->dtype == SCIPNP_BF16) block_attn_join_kernel<__bf16><<<jg, 256, 0, st>>>(p);
        else block_attn_join_kernel<float><<<jg, 256, 0, st>>>(p);
    }
    return launch_status("scipnp_block_attn");
}

}
