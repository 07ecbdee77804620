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
// eight loads in flight; the splits are added in LDS in order.
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
};

constexpr int SEL_MAX_BLOCKS = 8192;

// A double as a whole number of the same order: NaN lowest (1), 0 is free for "not a candidate"
__device__ __forceinline__ unsigned long long order_key(double v) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v + 0.0);          // (-0 becomes +0: they are equal)
    if (v != v) return 1;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// the keys of 0 .. nb-1 are in LDS (0: no candidate): writes the n best of them, ascending; ties to the lower index.
// Radix selection from the top byte: at most 8 counting passes, none once a byte's bucket is taken whole.
__device__ void select_best(const unsigned long long* keys, int nb, int n, int32_t* out, int* hist /* 256 + 16 */) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* const misc = hist + 256;
    int cand = 0;
    for (int j = tid; j < nb; j += 256) cand += keys[j] != 0;
    if (tid == 0) misc[0] = 0;
    __syncthreads();
    if (cand) atomicAdd(&misc[0], cand);                   // (a count: the order of the additions does not matter)
    __syncthreads();
    const int total = misc[0];
    unsigned long long prefix = 0, mask = 0;               // the threshold's known upper bytes
    int need = min(n, total);                              // still to take among the keys with that prefix
    bool all = need == total;                              // take every key with the prefix (and every greater one)
    for (int shift = 56; shift >= 0 && !all; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < nb; j += 256) {
            const unsigned long long k = keys[j];
            if (k != 0 && (k & mask) == prefix) atomicAdd(&hist[(int)(k >> shift) & 255], 1);
        }
        __syncthreads();
        // suffix sums over the 256 counts (from the greatest byte): one wave, four counts a lane
        if (wave == 0) {
            int c[4], s = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) { c[i] = hist[255 - (4 * lane + i)]; s += c[i]; }
            int incl = s;
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(incl, off, 64);
                if (lane >= off) incl += o;
            }
            int before = incl - s;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < need && before + c[i] >= need) {          // exactly one lane and count
                    misc[1] = 255 - (4 * lane + i);
                    misc[2] = need - before;
                    misc[3] = c[i];
                }
                before += c[i];
            }
        }
        __syncthreads();
        prefix |= (unsigned long long)misc[1] << shift;
        mask |= 255ull << shift;
        need = misc[2];
        all = need == misc[3];
    }
    // greater than the prefix: in; equal: the first `need` of them; written in order of the index
    if (tid == 0) { misc[4] = 0; misc[5] = 0; }
    __syncthreads();
    for (int base = 0; base < nb; base += 256) {
        const int j = base + tid;
        const unsigned long long k = j < nb ? keys[j] : 0;
        const bool eq = k != 0 && (k & mask) == prefix, gt = k != 0 && (k & mask) > prefix;
        const unsigned long long be = __ballot(eq);
        if (lane == 0) misc[8 + wave] = __popcll(be);
        __syncthreads();
        int eq_before = misc[4] + __popcll(be & ((1ull << lane) - 1));
        for (int w = 0; w < wave; ++w) eq_before += misc[8 + w];
        const bool in = gt || (eq && (all || eq_before < need));
        const unsigned long long bi = __ballot(in);
        if (lane == 0) misc[12 + wave] = __popcll(bi);
        __syncthreads();
        int at = misc[5] + __popcll(bi & ((1ull << lane) - 1));
        for (int w = 0; w < wave; ++w) at += misc[12 + w];
        if (in && at < n) out[at] = j;
        __syncthreads();
        if (tid == 0)
            for (int w = 0; w < 4; ++w) { misc[4] += misc[8 + w]; misc[5] += misc[12 + w]; }
        __syncthreads();
    }
    for (int i = misc[5] + tid; i < n; i += 256) out[i] = -1;
}

template <typename T>
__global__ void __launch_bounds__(256) select_blocks_kernel(Select a) {
    extern __shared__ __attribute__((aligned(16))) char smem_s[];
    double* const qs = (double*)smem_s;                                    // [D], then 256 more of scratch
    double* const red = qs + a.D;
    int* const hist = (int*)(red + 256);
    unsigned long long* const keys = (unsigned long long*)(hist + 256 + 16);
    const long long total = (long long)a.B * a.Hk * a.ng, item = xcd_item(blockIdx.x, total);
    if (item < 0) return;
    const int g = (int)(item % a.ng), bh = (int)(item / a.ng), hk = bh % a.Hk, b = bh / a.Hk;
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Lq) : a.Lq, klen = a.klen ? min(max(a.klen[b], 0), a.Lk) : a.Lk;
    int32_t* const out = a.sel + (size_t)item * a.n;
    const int q0 = g * a.qb, nq = min(a.qb, qlen - q0);
    if (nq <= 0) {                                                         // (uniform: the whole workgroup leaves)
        for (int i = threadIdx.x; i < a.n; i += 256) out[i] = -1;
        return;
    }
    // the group's summed queries: thread = (dimension, part of the rows), the parts added in order
    const int G = a.Hq / a.Hk, rows = nq * G, parts = max(1, 256 / a.D);
    {
        const int d = threadIdx.x % a.D, part = threadIdx.x / a.D;
        double s = 0.0;
        if (part < parts)
            for (int r = part; r < rows; r += parts)
                s += (double)(float)((const T*)a.q)[b * a.sq.b + (long long)(q0 + r / G) * a.sq.t + (hk * G + r % G) * a.sq.h + d];
        red[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x < a.D) {
            for (int p = 1; p < parts; ++p) s += red[p * a.D + threadIdx.x];
            qs[threadIdx.x] = s;
        }
        __syncthreads();
    }
    const int last = klen - qlen + q0 + nq - 1;                            // key position of the group's last query
    const int own = last >= 0 ? last / a.block : (last - a.block + 1) / a.block;
    // 16 lanes a block
    const int l16 = threadIdx.x & 15;
    for (int base = 0; base < a.nb; base += 16) {
        const int j = base + (threadIdx.x >> 4);
        const bool may = j < a.nb && (long long)j * a.block < klen && (!a.causal || (long long)j * a.block <= last);
        double s = 0.0;
        if (may) {
            const float* m = a.summary + (((size_t)b * a.nb + j) * a.Hk + hk) * a.D;
            for (int d = 4 * l16; d < a.D; d += 64) {
                const f32x4a v = *(const f32x4a*)(m + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) s += qs[d + e] * (double)v[e];
            }
        }
        s += dpp_f64<0xB1>(s);
        s += dpp_f64<0x4E>(s);
        s += dpp_f64<0x141>(s);
        s += dpp_f64<0x140>(s);
        if (l16 == 0 && j < a.nb) {
            const bool must = j < a.sink || abs(j - own) < a.local;
            keys[j] = !may ? 0 : must ? ~0ull : order_key(s);
        }
    }
    __syncthreads();
    select_best(keys, a.nb, a.n, out, hist);
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
    a.nb = (Lk + block - 1) / block;
    a.chunks = Hk * (D / (16 / (int)attn_esize(dtype)));
    a.cols = a.chunks < 256 ? a.chunks : 256;
    a.splits = 256 / a.cols;
    const int touched = newest ? (newest + block - 1) / block + 1 : a.nb;
    const int ny = (a.chunks + a.cols - 1) / a.cols;
    SCIPNP_REQUIRE(ny < 65536, "too many key heads");
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
    p.nb = (a->Lk + a->block - 1) / a->block;
    SCIPNP_REQUIRE(p.nb <= SEL_MAX_BLOCKS, "%d key blocks: at most %d (a larger block)", p.nb, SEL_MAX_BLOCKS);
    p.q = a->q; p.sq = strides_of(a->q_stride); p.summary = a->summary; p.qlen = a->qlen; p.klen = a->klen; p.sel = a->sel;
    p.B = a->B; p.Lq = a->Lq; p.Lk = a->Lk; p.Hq = a->Hq; p.Hk = a->Hk; p.D = a->D; p.block = a->block; p.qb = a->query_block;
    p.n = a->n_sel; p.sink = a->sink; p.local = a->local; p.causal = a->causal;
    p.ng = (a->Lq + a->query_block - 1) / a->query_block;
    const long long items = (long long)a->B * a->Hk * p.ng;
    SCIPNP_REQUIRE(items < (1ll << 30), "too many query groups");
    const size_t lds = (size_t)(a->D + 256) * 8 + (256 + 16) * 4 + (size_t)p.nb * 8;
    static LdsAttrOnce once[2];
    const void* fn = a->dtype == SCIPNP_BF16 ? (const void*)select_blocks_kernel<__bf16> : (const void*)select_blocks_kernel<float>;
    if (const int rc = once[a->dtype == SCIPNP_BF16].ensure(fn, (size_t)(256 + 256) * 8 + (256 + 16) * 4 + (size_t)SEL_MAX_BLOCKS * 8, "select_blocks")) return rc;
    if (a->dtype == SCIPNP_BF16) select_blocks_kernel<__bf16><<<xcd_grid(items), 256, lds, (hipStream_t)s>>>(p);
    else select_blocks_kernel<float><<<xcd_grid(items), 256, lds, (hipStream_t)s>>>(p);
    return launch_status("scipnp_select_blocks");
}

}
