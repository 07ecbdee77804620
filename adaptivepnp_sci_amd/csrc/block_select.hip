// The cheap score of block attention: the mean key of every block, and the choice of each query group's blocks.
//   mean[j] = (1 / live) sum of the live keys of block j;   score[g][j] = (sum of the group's queries) . mean[j]
// Both in fp64: the n-th and the next score of a row of some hundred blocks are often 1e-5 apart, an fp32 sum would choose by its order.
#include "attn_common.hpp"

namespace scipnp {

// ---------------------------------------------------------------- mean keys
struct Summary {
    const void* k;
    Strides sk;
    const int32_t* klen;
    float* out;
    int B, Lk, Hk, D, block, newest, nb, chunks, cols, splits;
};

// One workgroup per (sequence, block, column tile): a thread owns 16 bytes of a key head's row and every splits-th key of the block,
// eight loads in flight; the splits are added in LDS in order.  Reads each key once: 16 x 32768 bf16 keys of 8 x 128 in 200 us,
// 5.4 TB/s (a large read reaches 6.0); 165 us, 5.0 TB/s, where lengths of half to all of them leave 78 % live.  fp32 5.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) block_summary_kernel(Summary a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ double red[256][E + 1];
    const int b = blockIdx.z;
    const int klen = a.klen ? min(max(a.klen[b], 0), a.Lk) : a.Lk;
    int j = blockIdx.x;
    if (a.newest) {
        if (klen == 0) return;
        j += max(0, klen - a.newest) / a.block;
        if (j > (klen - 1) / a.block) return;
    }
    const int k0 = j * a.block, live = min(a.block, max(0, klen - k0));
    const int col = threadIdx.x % a.cols, split = threadIdx.x / a.cols, chunk = blockIdx.y * a.cols + col;
    const bool on = split < a.splits && chunk < a.chunks;
    const int per_head = a.D / E, h = on ? chunk / per_head : 0, d = on ? (chunk - h * per_head) * E : 0;
    double s[E] = {};
    if (on) {
        const T* p = (const T*)a.k + b * a.sk.b + h * a.sk.h + d;
        auto row = [&](int i, T (&v)[E]) { *(f32x4a*)v = *(const f32x4a*)(p + (long long)(k0 + i) * a.sk.t); };
        int i = split;
        for (; i + 7 * a.splits < live; i += 8 * a.splits) {
            __attribute__((aligned(16))) T v[8][E];
#pragma unroll
            for (int u = 0; u < 8; ++u) row(i + u * a.splits, v[u]);
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] += (double)(float)v[u][e];
        }
        for (; i < live; i += a.splits) {
            __attribute__((aligned(16))) T v[E];
            row(i, v);
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] += (double)(float)v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) red[threadIdx.x][e] = s[e];
    __syncthreads();
    if (on && split == 0) {
        for (int u = 1; u < a.splits; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] += red[u * a.cols + col][e];
        float* o = a.out + (((size_t)b * a.nb + j) * a.Hk + h) * a.D + d;
        const double n = live > 0 ? (double)live : 1.0;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (float)(s[e] / n);
    }
}

// ---------------------------------------------------------------- selection
struct Select {
    const void* q;
    Strides sq;
    const float* summary;
    const int32_t *qlen, *klen;
    int32_t* sel;
    int B, Lq, Lk, Hq, Hk, D, block, qb, n, sink, local, causal, nb, ng;
    int gpw, tiles, kst, hist_at;                         // groups of a workgroup, workgroups of a (sequence, key head), keys of a row, LDS offset
};

constexpr int SEL_MAX_BLOCKS = 8192;

// A number as a whole number of the same order (64 and 32 bits): NaN lowest (1), 0 is free for "no candidate", all ones for "always"
__device__ __forceinline__ unsigned long long order_key(double v) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v + 0.0);          // (-0 becomes +0: they are equal)
    if (v != v) return 1;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);
    if (v != v) return 1;
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// One counting pass of a radix selection, from the greatest byte down: of the keys with `prefix` above the byte, the byte of the
// need-th greatest, how many are still needed among those with that byte, and how many there are.  key(j): 0 where there is none.
template <typename K, typename F>
__device__ __forceinline__ void radix_pass(F key, int nb, int shift, K& prefix, K& mask, int& need, bool& all, int* hist, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) hist[lane + 64 * i] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int j = lane; j < nb; j += 64) {
        const K k = key(j);
        if (k != 0 && (k & mask) == prefix) atomicAdd(&hist[(int)(k >> shift) & 255], 1);          // (counts: no order)
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int c[4], s = 0;                                       // sums from the greatest byte down, four counts a lane
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = hist[255 - (4 * lane + i)]; s += c[i]; }
    int incl = s;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
    }
    int before = incl - s, byte = -1, rest = 0, have = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (before < need && before + c[i] >= need) { byte = 255 - (4 * lane + i); rest = need - before; have = c[i]; }
        before += c[i];
    }
    const int src = __ffsll((unsigned long long)__ballot(byte >= 0)) - 1;                          // exactly one lane has it
    prefix |= (K)__shfl(byte, src, 64) << shift;
    mask |= (K)255 << shift;
    need = __shfl(rest, src, 64);
    all = need == __shfl(have, src, 64);
}

// the need-th greatest of the keys that count(t) counts from t on, bit by bit
template <typename F>
__device__ __forceinline__ unsigned nth_greatest(int need, F count) {
    unsigned t = 0;
#pragma unroll 4
    for (int bit = 31; bit >= 0; --bit)
        if (count(t | 1u << bit) >= need) t |= 1u << bit;
    return t;
}

// One wave writes the n best of the candidates 0 .. nb-1, ascending; ties to the lower index.  The scores are compared as fp32 keys
// first (half the LDS); only where the n-th and the next share one are those candidates compared in fp64, recomputed by exact(j).
// Up to 32 wanted of more than 256: the need-th greatest of the lanes' own greatest keys is a bound that few others reach (16 of 2048:
// about 18), and those few are sorted out in registers.  Otherwise a radix selection over all keys.  (16 of 2048 blocks, 2048 groups:
// 56 us with the radix passes, whose counters collide, 40 us by the bound; 16 of 128: 9.4 against 10.5 us, so there they stay)
constexpr int SHORT = 256;
template <typename F>
__device__ void select_best(const unsigned* keys, int nb, int n, int32_t* out, int* hist, unsigned short* list, int lane, F exact) {
    const unsigned long long below = (1ull << lane) - 1;
    int cand = 0;
    unsigned top = 0;
    for (int j = lane; j < nb; j += 64) {
        const unsigned k = keys[j];
        cand += k != 0;
        top = max(top, k);
    }
    for (int off = 32; off > 0; off >>= 1) cand += __shfl_xor(cand, off, 64);
    cand = __builtin_amdgcn_readfirstlane(cand);
    unsigned prefix = 0, mask = 0;                         // the threshold's known upper bytes
    int need = min(n, cand);                               // still to take among the keys with that prefix
    bool all = need == cand;                               // take every key with the prefix (and every greater one)
    int items = nb;                                        // the candidates that are still looked at: all, or those of the list
    bool listed = false;
    if (!all && nb > SHORT && need <= 32) {
        const unsigned bound = max(nth_greatest(need, [&](unsigned t) { return __popcll(__ballot(top >= t)); }), 1u);
        int c = 0;
        for (int base = 0; base < nb; base += 64) {
            const int j = base + lane;
            const bool in = j < nb && keys[j] >= bound;
            const unsigned long long m = __ballot(in);
            const int at = c + __popcll(m & below);
            if (in && at < SHORT) list[at] = (unsigned short)j;
            c += __popcll(m);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (c <= SHORT) {
            listed = true;
            items = c;
            unsigned r[SHORT / 64];
#pragma unroll
            for (int u = 0; u < SHORT / 64; ++u) r[u] = lane + 64 * u < c ? keys[list[lane + 64 * u]] : 0;
            auto from = [&](unsigned t) {
                int s = __popcll(__ballot(r[0] >= t));
                if (c > 64)
#pragma unroll
                    for (int u = 1; u < SHORT / 64; ++u) s += __popcll(__ballot(r[u] >= t));
                return s;
            };
            prefix = nth_greatest(need, from);
            mask = ~0u;
            const int more = prefix == ~0u ? 0 : from(prefix + 1);
            all = need == from(prefix);
            need -= more;
        }
    }
    if (!listed)
        for (int shift = 24; shift >= 0 && !all; shift -= 8)
            radix_pass<unsigned>([&](int j) { return keys[j]; }, nb, shift, prefix, mask, need, all, hist, lane);
    auto at_item = [&](int i) { return listed ? (int)list[i] : i; };
    unsigned long long prefix64 = 0, mask64 = 0;
    if (!all && prefix != ~0u && prefix != 1) {            // (the always chosen and the NaNs are equal among themselves)
        auto key64 = [&](int i) -> unsigned long long { const int j = at_item(i); return keys[j] == prefix ? order_key(exact(j)) : 0; };
        unsigned long long lo = ~0ull, hi = 0;
        for (int j = lane; j < items; j += 64) {
            const unsigned long long k = key64(j);
            if (k) { lo = min(lo, k); hi = max(hi, k); }
        }
        for (int off = 32; off > 0; off >>= 1) {
            lo = min(lo, (unsigned long long)__shfl_xor((long long)lo, off, 64));
            hi = max(hi, (unsigned long long)__shfl_xor((long long)hi, off, 64));
        }
        if (lo != hi)
            for (int shift = 56; shift >= 0 && !all; shift -= 8) radix_pass<unsigned long long>(key64, items, shift, prefix64, mask64, need, all, hist, lane);
    }
    // greater than the threshold: in; equal: the first `need` of them
    int eqs = 0, at = 0;
    for (int base = 0; base < items; base += 64) {
        const int j = base + lane < items ? at_item(base + lane) : 0;
        const unsigned k = base + lane < items ? keys[j] : 0;
        bool eq = k != 0 && (k & mask) == prefix, gt = k != 0 && (k & mask) > prefix;
        if (mask64 != 0 && eq) {
            const unsigned long long e = order_key(exact(j));
            eq = (e & mask64) == prefix64;
            gt = (e & mask64) > prefix64;
        }
        const unsigned long long be = __ballot(eq);
        const bool in = gt || (eq && (all || eqs + __popcll(be & below) < need));
        const unsigned long long bi = __ballot(in);
        if (in) out[at + __popcll(bi & below)] = j;
        eqs += __popcll(be);
        at += __popcll(bi);
    }
    for (int i = at + lane; i < n; i += 64) out[i] = -1;
}

// One workgroup of eight waves: up to 16 query groups of one (sequence, key head) -- as many as have room for their scores in LDS.
//   1. a wave sums the queries of one group (16 bytes a lane, the parts of its rows added in order);
//   2. the scores of 16 blocks x 16 groups at a time on the fp64 matrix unit (v_mfma_f64_16x16x4_f64: lane -> row lane & 15,
//      contraction lane >> 4; result register r: row 4 r + (lane >> 4), column lane & 15): a mean key is read once for all groups;
//   3. a wave chooses the blocks of one group.
// 16384 bf16 queries of 32 x 128 in groups of 16, 16 of 256 blocks: 52 us, of which the queries take 34 (their 134 MB 26 at the copy
// rate), the scores 11 (half the fp64 matrix rate) and the choice 9, one after the other in every workgroup.  2048 fp32 groups of 64 x 48, 16 of
// 2048 blocks: 39 us, 7 + 23 + 10; half the matrix columns are empty there, eight groups' scores fill the LDS.
typedef double f64x4a __attribute__((ext_vector_type(4)));
constexpr int SEL_WAVES = 8;

template <typename T, int ND>                              // ND * 16 >= D
__global__ void __launch_bounds__(64 * SEL_WAVES) select_blocks_kernel(Select a) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int E = 16 / sizeof(T);
    extern __shared__ __attribute__((aligned(16))) char smem_s[];
    const int qst = a.D + 2;                               // (rows two banks apart)
    double* const qs = (double*)smem_s;                    // [groups][qst]
    double* const scratch = qs + a.gpw * qst;              // step 1: the parts; then the keys [groups][kst]
    unsigned* const keys = (unsigned*)scratch;
    int* const hists = (int*)(smem_s + a.hist_at);
    unsigned short* const lists = (unsigned short*)(hists + SEL_WAVES * 256);
    const long long total = (long long)a.B * a.Hk * a.tiles, item = xcd_item(blockIdx.x, total);
    if (item < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g0 = (int)(item % a.tiles) * a.gpw, bh = (int)(item / a.tiles), hk = bh % a.Hk, b = bh / a.Hk;
    const int ngr = min(a.gpw, a.ng - g0);
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Lq) : a.Lq, klen = a.klen ? min(max(a.klen[b], 0), a.Lk) : a.Lk;
    const int G = a.Hq / a.Hk, nc = a.D / E, parts = 64 / nc;              // (D <= 256: at most 64 pieces of a row)
    for (int i = wave; i < a.gpw; i += SEL_WAVES) {
        const int q0 = (g0 + i) * a.qb, toks = i < ngr ? min(a.qb, qlen - q0) : 0;
        const int c = lane % nc, part = lane / nc;
        double s[E] = {};
        if (part < parts) {
            const T* base = (const T*)a.q + b * a.sq.b + (long long)q0 * a.sq.t + hk * G * a.sq.h + c * E;
            int tok = part / G, h = part - tok * G;
            const int dt = parts / G, dh = parts - dt * G;
            while (tok < toks) {
                __attribute__((aligned(16))) T v[8][E];
                int m = 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) {              // eight rows under way
                    const bool ok = tok < toks;
                    *(f32x4a*)v[u] = ok ? *(const f32x4a*)(base + (long long)tok * a.sq.t + h * a.sq.h) : f32x4a{0.f, 0.f, 0.f, 0.f};
                    m += ok;
                    h += dh;
                    tok += dt;
                    if (h >= G) { h -= G; ++tok; }
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (u < m)
#pragma unroll
                        for (int e = 0; e < E; ++e) s[e] += (double)(float)v[u][e];
            }
        }
        double* const mine = scratch + (size_t)wave * 64 * E;
#pragma unroll
        for (int e = 0; e < E; ++e) mine[lane * E + e] = s[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int d = lane; d < a.D; d += 64) {
            double v = 0.0;
            for (int p = 0; p < parts; ++p) v += mine[(p * nc + d / E) * E + d % E];
            qs[i * qst + d] = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    // key position of the group's last query (this lane's column)
    const int col = lane & 15, kq = lane >> 4, gc = g0 + col;
    const bool group = col < ngr && gc * a.qb < qlen;
    const int last = klen - qlen + min((gc + 1) * a.qb, qlen) - 1;
    const int own = last >= 0 ? last / a.block : -1 - (-1 - last) / a.block;        // (no sum here passes 32 bits, whatever the block)
    const int there = klen > 0 ? (klen - 1) / a.block + 1 : 0;
    const int seen = min(there, !a.causal ? a.nb : last < 0 ? 0 : last / a.block + 1);        // blocks it may choose
    // no group here sees a block from `nb` on (its own rows end with the last group's last query): neither scored nor looked at
    const int lastq = min((g0 + ngr) * a.qb, qlen), end = klen - qlen + lastq;
    const int nb = lastq <= g0 * a.qb ? 0 : min(there, !a.causal ? a.nb : end <= 0 ? 0 : (end - 1) / a.block + 1);
    const int nt = (nb + 15) / 16;
    const double* const qrow = qs + (col < a.gpw ? col : 0) * qst + 4 * kq;
    const float* const means = a.summary + ((size_t)b * a.nb * a.Hk + hk) * a.D;
    auto query = [&](int d, double (&q)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = 16 * d + 4 * kq < a.D ? qrow[16 * d + e] : 0.0;
    };
    constexpr bool HELD = ND <= 8;                         // the sums stay in registers while the tiles go by (16 columns: 128 VGPRs, read again)
    double held[HELD ? ND : 1][4];
    if constexpr (HELD)
#pragma unroll
        for (int d = 0; d < ND; ++d) query(d, held[d]);
    for (int jt = wave; jt < nt; jt += SEL_WAVES) {
        const int j = jt * 16 + col;                       // (A's row)
        f32x4a m[ND];
        const float* const row = means + (size_t)(j < nb ? j : 0) * a.Hk * a.D + 4 * kq;
#pragma unroll
        for (int d = 0; d < ND; ++d) m[d] = j < nb && 16 * d + 4 * kq < a.D ? *(const f32x4a*)(row + 16 * d) : f32x4a{0.f, 0.f, 0.f, 0.f};
        f64x4a s0 = {0.0, 0.0, 0.0, 0.0}, s1 = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (16 * d >= a.D) continue;                   // (uniform)
            double q[4];
            if constexpr (HELD) {
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = held[d][e];
            } else {
                query(d, q);
            }
            s0 = __builtin_amdgcn_mfma_f64_16x16x4f64((double)m[d][0], q[0], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f64_16x16x4f64((double)m[d][1], q[1], s1, 0, 0, 0);
            s0 = __builtin_amdgcn_mfma_f64_16x16x4f64((double)m[d][2], q[2], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f64_16x16x4f64((double)m[d][3], q[3], s1, 0, 0, 0);
        }
        if (col < a.gpw)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int jj = jt * 16 + 4 * r + kq;
                if (jj >= nb) continue;
                const bool must = jj < a.sink || abs(jj - own) < a.local;
                keys[(size_t)col * a.kst + jj] = !group || jj >= seen ? 0u : must ? ~0u : order_key((float)(s0[r] + s1[r]));
            }
    }
    __syncthreads();
    for (int i = wave; i < ngr; i += SEL_WAVES)
        select_best(keys + (size_t)i * a.kst, nb, a.n, a.sel + ((size_t)bh * a.ng + g0 + i) * a.n, hists + wave * 256, lists + wave * SHORT, lane, [&](int j) {
            const float* m = means + (size_t)j * a.Hk * a.D;
            double s = 0.0;
            for (int d = 0; d < a.D; d += 4) {
                const f32x4a v = *(const f32x4a*)(m + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma(qs[i * qst + d + e], (double)v[e], s);
            }
            return s;
        });
#endif
}

template <typename T>
static int select_launch(const Select& p, size_t lds, unsigned grid, hipStream_t st) {
    static LdsAttrOnce once[3];
    const int v = p.D <= 64 ? 0 : p.D <= 128 ? 1 : 2;
    const void* fn = v == 0 ? (const void*)select_blocks_kernel<T, 4> : v == 1 ? (const void*)select_blocks_kernel<T, 8> : (const void*)select_blocks_kernel<T, 16>;
    if (const int rc = once[v].ensure(fn, 163840, "select_blocks")) return rc;
    if (v == 0) select_blocks_kernel<T, 4><<<grid, 64 * SEL_WAVES, lds, st>>>(p);
    else if (v == 1) select_blocks_kernel<T, 8><<<grid, 64 * SEL_WAVES, lds, st>>>(p);
    else select_blocks_kernel<T, 16><<<grid, 64 * SEL_WAVES, lds, st>>>(p);
    return launch_status("scipnp_select_blocks");
}

}  // namespace scipnp

using namespace scipnp;

extern "C" {

int scipnp_block_summary(const void* k, const int64_t* k_stride, int dtype, const int32_t* klen, float* summary, int B, int Lk, int Hk,
                         int D, int block, int newest, scipnp_stream_t s) {
    SCIPNP_REQUIRE(k && k_stride && summary, "null k, k_stride or summary");
    SCIPNP_REQUIRE(dtype == SCIPNP_F32 || dtype == SCIPNP_BF16, "dtype %d: 0 (float32) or 1 (bfloat16)", dtype);
    SCIPNP_REQUIRE(B > 0 && B < 65536 && Lk > 0 && Hk > 0, "B, Lk, Hk must be positive (B below 65536)");
    SCIPNP_REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, "head size %d: a multiple of 8 up to 256", D);
    SCIPNP_REQUIRE(block > 0 && newest >= 0, "block must be positive, newest not negative");
    SCIPNP_ALIGNED(k);
    SCIPNP_ALIGNED(summary);
    SCIPNP_STRIDES(k_stride, dtype);
    Summary a = {};
    a.k = k; a.sk = strides_of(k_stride); a.klen = klen; a.out = summary;
    a.B = B; a.Lk = Lk; a.Hk = Hk; a.D = D; a.block = block; a.newest = newest;
    SCIPNP_REQUIRE((Lk - 1) / block + 1 < (1 << 24), "%d blocks: fewer than 2^24 (a larger block)", (Lk - 1) / block + 1);
    a.nb = (Lk - 1) / block + 1;                          // (no sum that a block or a length near 2^31 would carry past 32 bits)
    const long long chunks = (long long)Hk * (D / (16 / (int)attn_esize(dtype)));
    SCIPNP_REQUIRE(chunks < (1 << 24), "too many key heads");
    a.chunks = (int)chunks;
    a.cols = a.chunks < 256 ? a.chunks : 256;
    a.splits = 256 / a.cols;
    const int touched = newest ? (newest - 1) / block + 2 : a.nb;
    const int ny = (a.chunks + a.cols - 1) / a.cols;
    const dim3 grid((unsigned)(touched < a.nb ? touched : a.nb), (unsigned)ny, (unsigned)B);
    if (dtype == SCIPNP_BF16) block_summary_kernel<__bf16><<<grid, 256, 0, (hipStream_t)s>>>(a);
    else block_summary_kernel<float><<<grid, 256, 0, (hipStream_t)s>>>(a);
    return launch_status("scipnp_block_summary");
}

int scipnp_select_blocks(const scipnp_select_args* a, scipnp_stream_t s) {
    SCIPNP_BLOCK_SIZE(a, scipnp_select_args);
    SCIPNP_REQUIRE(a->q && a->summary && a->sel, "null q, summary or sel");
    SCIPNP_REQUIRE(a->dtype == SCIPNP_F32 || a->dtype == SCIPNP_BF16, "dtype %d: 0 (float32) or 1 (bfloat16)", a->dtype);
    SCIPNP_REQUIRE(a->B > 0 && a->Lq > 0 && a->Lk > 0 && a->Hk > 0 && a->Hq > 0, "B, Lq, Lk, Hq, Hk must be positive");
    SCIPNP_REQUIRE(a->Hq % a->Hk == 0, "%d query heads are no multiple of %d key heads", a->Hq, a->Hk);
    SCIPNP_REQUIRE(a->D >= 8 && a->D <= 256 && a->D % 8 == 0, "head size %d: a multiple of 8 up to 256", a->D);
    SCIPNP_REQUIRE(a->block > 0 && a->query_block > 0 && a->query_block <= 1024, "block must be positive, query_block 1 to 1024");
    SCIPNP_REQUIRE(a->n_sel > 0 && a->n_sel <= 1024, "n_sel %d: 1 to 1024", a->n_sel);
    SCIPNP_REQUIRE(a->sink >= 0 && a->local >= 0, "sink and local must not be negative");
    SCIPNP_ALIGNED(a->q);
    SCIPNP_ALIGNED(a->summary);
    SCIPNP_STRIDES(a->q_stride, a->dtype);
    Select p = {};
    p.nb = (a->Lk - 1) / a->block + 1;
    SCIPNP_REQUIRE(p.nb <= SEL_MAX_BLOCKS, "%d key blocks: at most %d (a larger block)", p.nb, SEL_MAX_BLOCKS);
    p.q = a->q; p.sq = strides_of(a->q_stride); p.summary = a->summary; p.qlen = a->qlen; p.klen = a->klen; p.sel = a->sel;
    p.B = a->B; p.Lq = a->Lq; p.Lk = a->Lk; p.Hq = a->Hq; p.Hk = a->Hk; p.D = a->D; p.block = a->block; p.qb = a->query_block;
    p.n = a->n_sel; p.sink = a->sink; p.local = a->local; p.causal = a->causal;
    p.ng = (a->Lq - 1) / a->query_block + 1;
    // groups of a workgroup: up to 16 (the columns of a matrix instruction) with at most 64 KB of scores, two workgroups a CU
    p.gpw = 65536 / (p.nb * 4);
    p.gpw = p.gpw > 16 ? 16 : p.gpw;
    if (p.gpw > p.ng) p.gpw = p.ng;
    p.tiles = (p.ng + p.gpw - 1) / p.gpw;
    p.kst = (p.nb + 31) / 32 * 32 + 4;                    // (16 groups' keys of a block in different banks)
    const size_t parts_bytes = (size_t)SEL_WAVES * 64 * (16 / attn_esize(a->dtype)) * 8, key_bytes = ((size_t)p.gpw * p.kst * 4 + 15) / 16 * 16;
    p.hist_at = (int)((size_t)p.gpw * (a->D + 2) * 8 + (parts_bytes > key_bytes ? parts_bytes : key_bytes));
    const long long items = (long long)a->B * a->Hk * p.tiles;
    SCIPNP_REQUIRE(items < (1ll << 22) && (long long)p.ng * a->query_block < (1ll << 30), "too many query groups");
    const size_t lds = (size_t)p.hist_at + SEL_WAVES * (256 * 4 + SHORT * 2);
    return a->dtype == SCIPNP_BF16 ? select_launch<__bf16>(p, lds, xcd_grid(items), (hipStream_t)s) : select_launch<float>(p, lds, xcd_grid(items), (hipStream_t)s);
}

}
