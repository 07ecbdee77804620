// Attention over selected key blocks, forward.  One workgroup of four waves: up to 128 rows (queries x heads of a key head) of one query
// group; RW waves hold 32 rows each, the 4 / RW others of a row set take every other key tile and are joined at the end (few rows:
// a decoding step is 8 rows, four waves share its keys).  A pass over the selected tiles with running maximum and sum.
#include "block_attn.hpp"

namespace scipnp {

template <typename T, int DP, int RW>
struct FwdCfg {
    static constexpr int KS = 4 / RW, NTH = 64 * RW;
    static constexpr int KST = row_stride<T, DP>(), VST = col_stride<T, DP>();
    static constexpr int TILE = KT * (KST + VST) * (int)sizeof(T);            // K and V of one tile
    static constexpr int BUFS = KS == 4 ? 1 : 2;                              // four private tiles need no barrier and no second buffer
    static constexpr int OST = DP + 4;
    static constexpr int JOIN = KS > 1 ? RW * 32 * OST * 4 + KS * RW * 32 * 8 : 0;
    static constexpr int TILES = KS * BUFS * TILE;
    static constexpr int MAIN = TILES > JOIN ? TILES : JOIN;
    static constexpr int KP = KS * BUFS * KT * 4;
};

template <typename T, int DP, int RW>
__global__ void __launch_bounds__(256) block_attn_kernel(Attn a) {
#if defined(__HIP_DEVICE_COMPILE__)
    using C = FwdCfg<T, DP, RW>;
    using Frag = typename Mat<T>::Frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const long long total = (long long)a.B * a.Hk * a.ng * a.chunks * a.splits;
    const long long item = xcd_item(blockIdx.x, total);
    if (item < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, hi = lane >> 5;
    const int rw = wave % RW, ks = wave / RW, tsplit = rw * 64 + lane;
    long long it0 = item;
    const int part = (int)(it0 % a.splits); it0 /= a.splits;
    const int chunk = (int)(it0 % a.chunks); it0 /= a.chunks;
    const int g = (int)(it0 % a.ng), bh = (int)(it0 / a.ng), hk = bh % a.Hk, b = bh / a.Hk;
    const Seq sq = seq_of(a, b);
    const int R = a.qb * a.G, r0 = chunk * 32 * RW;
    if (g * a.qb + r0 / a.G >= sq.qlen) return;           // (uniform) nothing live in this chunk
    const int row = r0 + rw * 32 + li, tok = g * a.qb + row / a.G, gl = row % a.G, head = hk * a.G + gl;
    const bool live = row < R && tok < sq.qlen;
    const int qkey = sq.shift + tok;                      // key position of the row
    const int lim = !live ? -1 : a.causal ? min(qkey, sq.klen - 1) : sq.klen - 1;       // its last visible key

    char* const main = smem;
    int* const kp_lds = (int*)(smem + C::MAIN);
    int* const list = (int*)(smem + C::MAIN + C::KP);
    int* const nlist = list + a.n;
    const Bias bias = load_bias(a, smem + C::MAIN + C::KP + (a.n + 4) / 4 * 16, hk);
    if (wave == 0) {
        const int rows_end = min(min(R, r0 + 32 * RW), (sq.qlen - g * a.qb) * a.G);
        const int far = a.causal ? min(sq.klen, sq.shift + g * a.qb + (rows_end - 1) / a.G + 1) : sq.klen;
        const int c = live_blocks(a, a.sel + ((size_t)bh * a.ng + g) * a.n, far, list, lane);
        if (lane == 0) *nlist = c;
    }
    Frag qf[DP / Mat<T>::K];
    load_frags<T, DP>(live ? (const T*)a.q + b * a.sq.b + (long long)tok * a.sq.t + head * a.sq.h : nullptr, a.D, hi, qf);
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

    const int tpb = a.block / KT, ntiles = *nlist * tpb;
    const int per = (ntiles + a.splits - 1) / a.splits, t_begin = part * per, t_end = min(ntiles, t_begin + per);
    const int iters = t_end > t_begin ? (t_end - t_begin + C::KS - 1) / C::KS : 0;

    const T* const kb = (const T*)a.k + b * a.sk.b + hk * a.sk.h;
    const T* const vb = (const T*)a.v + b * a.sv.b + hk * a.sv.h;
    TileRegs<T, DP, C::NTH> kr, vr;
    int kpr = 0;
    auto key0_of = [&](int it) -> int {
        const int t = t_begin + it * C::KS + ks;
        if (t >= t_end) return -1;
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
    float m = -INFINITY, l = 0.f;

    int key0 = iters ? key0_of(0) : -1;
    load(key0);
    for (int it = 0; it < iters; ++it) {
        const int buf = C::BUFS == 2 ? (it & 1) : 0;
        T* const kt = (T*)(main + (ks * C::BUFS + buf) * C::TILE);
        T* const vt = kt + KT * C::KST;
        int* const kp = kp_lds + (ks * C::BUFS + buf) * KT;
        if (key0 >= 0) {
            kr.template store<C::KST>(tsplit, kt);
            vr.template store<C::VST>(tsplit, vt);
            if (a.k_pos && tsplit < KT) kp[tsplit] = kpr;
        }
        if constexpr (C::BUFS == 2) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int cur = key0;
        key0 = it + 1 < iters ? key0_of(it + 1) : -1;
        load(key0);
        if (cur >= 0 && cur <= max_lim) {
            f32x16a s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
            s = mma_rows<T, DP>(kt + li * C::KST, qf, hi, s);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= a.scale;
            if (a.nbuckets) {
                const int dist = tile_distance(a, range, cur, a.k_pos ? kp : nullptr, lane);
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
            if (cur + KT - 1 > min_lim) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = cur + tile_key(r, hi) <= lim ? s[r] : -INFINITY;
            }
            float mt = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
            const float mn = fmaxf(m, mt), ms = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f((m - ms) * LOG2E);
            m = mn;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = __builtin_amdgcn_exp2f((s[r] - ms) * LOG2E);
                sum += s[r];
            }
            l = fmaf(l, alpha, sum);
            if (__ballot(alpha != 1.f)) {
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
            }
            // P rounded to bf16 is off by 2^-8 of each probability, of the order of the output's own rounding; with out32 wanted it is
            // taken whole: delta = sum dO O enters every score's gradient, and the sums of dbias cancel down to its error
            mma_cols<T, DP, C::VST>(vt, s, lane, o, a.out32 != nullptr);
        }
        if constexpr (C::BUFS == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    l += __shfl_xor(l, 32, 64);

    if constexpr (C::KS > 1) {                            // the row set's other waves: maxima and sums first, then the sums of O in order
        float* const obuf = (float*)main + rw * 32 * C::OST;
        float2* const ml = (float2*)(main + RW * 32 * C::OST * 4) + rw * 32;
        __syncthreads();
        if (hi == 0) ml[ks * RW * 32 + li] = make_float2(m, l);
        __syncthreads();
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < C::KS; ++k) M = fmaxf(M, ml[k * RW * 32 + li].x);
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
#pragma unroll
        for (int k = 0; k < C::KS; ++k) L = fmaf(ml[k * RW * 32 + li].y, __builtin_amdgcn_exp2f((ml[k * RW * 32 + li].x - Ms) * LOG2E), L);
        const float f = __builtin_amdgcn_exp2f((m - Ms) * LOG2E);
        m = M;
        l = L;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] *= f;
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
    if (!live) return;
    const size_t id = ((size_t)b * a.Lq + tok) * a.Hq + head;
    if (a.splits > 1) {
        const size_t rows = (size_t)a.B * a.Lq * a.Hq;
        if (hi == 0) *(float2*)(a.pml + 2 * (part * rows + id)) = make_float2(m, l);
        float* const po = a.po + (part * rows + id) * a.D;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * db + 8 * q + 4 * hi;
                if (d < a.D) *(f32x4a*)(po + d) = f32x4a{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]};
            }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);             // (a NaN sum stays one)
    T* const out = (T*)a.out + b * a.so.b + (long long)tok * a.so.t + head * a.so.h;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * db + 8 * q + 4 * hi;
            if (d >= a.D) continue;
            f32x4a v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = o[db][4 * q + e] * inv;
            if constexpr (sizeof(T) == 2) {
                bf16x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (__bf16)v[e];
                *(bf16x4*)(out + d) = w;
            } else {
                *(f32x4a*)(out + d) = v;
            }
            if (a.out32) *(f32x4a*)(a.out32 + id * a.D + d) = v;
        }
    if (a.lse && hi == 0) a.lse[((size_t)b * a.Hq + head) * a.Lq + tok] = l == 0.f ? -INFINITY : m + __logf(l);
#endif
}

// joins the parts of a row's keys: one wave a row
template <typename T>
__global__ void __launch_bounds__(256) block_attn_join_kernel(Attn a) {
    const size_t rows = (size_t)a.B * a.Lq * a.Hq, id = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= rows) return;
    const int lane = threadIdx.x & 63, head = (int)(id % a.Hq), tok = (int)(id / a.Hq % a.Lq), b = (int)(id / a.Hq / a.Lq);
    if (tok >= seq_of(a, b).qlen) return;
    float M = -INFINITY;
    for (int p = 0; p < a.splits; ++p) M = fmaxf(M, a.pml[2 * (p * rows + id)]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, s[2] = {0.f, 0.f};
    for (int p = 0; p < a.splits; ++p) {
        const float2 ml = *(const float2*)(a.pml + 2 * (p * rows + id));
        const float f = __builtin_amdgcn_exp2f((ml.x - Ms) * LOG2E);
        L = fmaf(ml.y, f, L);
        const float* po = a.po + (p * rows + id) * a.D;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 64 * i < a.D) s[i] = fmaf(po[lane + 64 * i], f, s[i]);
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + 64 * i;
        if (d >= a.D) continue;
        const float v = s[i] * inv;
        ((T*)a.out)[b * a.so.b + (long long)tok * a.so.t + head * a.so.h + d] = (T)v;
        if (a.out32) a.out32[id * a.D + d] = v;
    }
    if (a.lse && lane == 0) a.lse[((size_t)b * a.Hq + head) * a.Lq + tok] = L == 0.f ? -INFINITY : M + __logf(L);
}

static int row_waves(const scipnp_block_attn_args* a) {
    const int R = a->query_block * (a->Hq / a->Hk);
    return R <= 32 ? 1 : R <= 64 ? 2 : 4;
}

// parts of a group's keys: enough workgroups for two on every CU, none with fewer than four tiles a wave
static int attn_splits(const scipnp_block_attn_args* a) {
    const int rw = row_waves(a), R = a->query_block * (a->Hq / a->Hk);
    const long long groups = (long long)a->B * a->Hk * ((a->Lq + a->query_block - 1) / a->query_block) * ((R + 32 * rw - 1) / (32 * rw));
    const int nb = (a->Lk + a->block - 1) / a->block;
    const long long tiles = (long long)(a->n_sel < nb ? a->n_sel : nb) * (a->block / KT);
    long long want = 512 / (groups > 0 ? groups : 1), most = tiles / (4 * (4 / rw));
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
    SCIPNP_REQUIRE(a->block > 0 && a->block <= 65536 && a->block % 64 == 0, "block %d: a multiple of 64", a->block);
    SCIPNP_REQUIRE(a->query_block > 0 && a->query_block <= 1024, "query_block %d: 1 to 1024", a->query_block);
    SCIPNP_REQUIRE(a->n_sel > 0 && a->n_sel <= 1024, "n_sel %d: 1 to 1024", a->n_sel);
    SCIPNP_REQUIRE(a->Lk <= (1 << 30) && a->Lq <= (1 << 30), "sequences of at most 2^30 tokens");
    SCIPNP_REQUIRE(a->q && a->k && a->v && a->sel, "null q, k, v or sel");
    SCIPNP_REQUIRE(a->num_buckets >= 0 && a->num_buckets <= 64, "%d buckets: at most 64", a->num_buckets);
    if (a->num_buckets) {
        SCIPNP_REQUIRE(a->bias && a->bucket_of, "buckets need bias and bucket_of");
        SCIPNP_REQUIRE(a->max_distance > 0 && a->max_distance <= 4096, "max_distance %d: 1 to 4096", a->max_distance);
        SCIPNP_REQUIRE(a->num_buckets * (a->Hq / a->Hk) <= 2048, "buckets times query heads of a key head: at most 2048");
    }
    SCIPNP_ALIGNED(a->q); SCIPNP_ALIGNED(a->k); SCIPNP_ALIGNED(a->v);
    SCIPNP_STRIDES(a->q_stride, a->dtype); SCIPNP_STRIDES(a->k_stride, a->dtype); SCIPNP_STRIDES(a->v_stride, a->dtype);
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
    p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out; p.dout = a->dout;
    p.sq = strides_of(a->q_stride); p.sk = strides_of(a->k_stride); p.sv = strides_of(a->v_stride); p.so = strides_of(a->out_stride);
    p.sdo = strides_of(a->dout_stride);
    p.sel = a->sel; p.qlen = a->qlen; p.klen = a->klen;
    p.bucket_of = a->bucket_of; p.q_pos = a->num_buckets ? a->q_pos : nullptr; p.k_pos = a->num_buckets ? a->k_pos : nullptr; p.bias = a->bias;
    p.lse = a->lse; p.out32 = a->out32;
    p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.dbias = a->num_buckets ? a->dbias : nullptr;
    return p;
}

template <typename T, int DP, int RW>
static int fwd_launch(const Attn& p, unsigned grid, hipStream_t st) {
    using C = FwdCfg<T, DP, RW>;
    const size_t fixed = (size_t)C::MAIN + C::KP, lds = fixed + (size_t)(p.n + 4) / 4 * 16 + bias_lds(p.nbuckets, p.maxd, p.G);
    static LdsAttrOnce once;
    const size_t most = fixed + 1028 * 4 + bias_lds(1, 4096, 1) + 2048 * 4;
    if (const int rc = once.ensure((const void*)block_attn_kernel<T, DP, RW>, most < 163840 ? most : 163840, "block_attn")) return rc;
    if (lds > 163840) return fail(SCIPNP_EINVAL, "block_attn: %zu bytes of LDS needed", lds);
    block_attn_kernel<T, DP, RW><<<grid, 256, lds, st>>>(p);
    return SCIPNP_OK;
}
template <typename T, int DP>
static int fwd_rows(const Attn& p, int rw, unsigned grid, hipStream_t st) {
    return rw == 1 ? fwd_launch<T, DP, 1>(p, grid, st) : rw == 2 ? fwd_launch<T, DP, 2>(p, grid, st) : fwd_launch<T, DP, 4>(p, grid, st);
}
template <typename T>
static int fwd_dim(const Attn& p, int rw, unsigned grid, hipStream_t st) {
    return p.D <= 32 ? fwd_rows<T, 32>(p, rw, grid, st) : p.D <= 64 ? fwd_rows<T, 64>(p, rw, grid, st)
         : p.D <= 96 ? fwd_rows<T, 96>(p, rw, grid, st) : fwd_rows<T, 128>(p, rw, grid, st);
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
    const unsigned grid = xcd_grid((long long)p.B * p.Hk * p.ng * p.chunks * p.splits);
    if (const int rc = a->dtype == SCIPNP_BF16 ? fwd_dim<__bf16>(p, rw, grid, st) : fwd_dim<float>(p, rw, grid, st)) return rc;
    if (p.splits > 1) {
        const unsigned jg = (unsigned)(((size_t)p.B * p.Lq * p.Hq + 3) / 4);
        if (a->dtype == SCIPNP_BF16) block_attn_join_kernel<__bf16><<<jg, 256, 0, st>>>(p);
        else block_attn_join_kernel<float><<<jg, 256, 0, st>>>(p);
    }
    return launch_status("scipnp_block_attn");
}

}
