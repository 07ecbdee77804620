// Norm of each query and key head with its learned weight and the rotation by the token's position, one pass; its gradient.
//   n = x * r * w,  r = 1 / sqrt(mean(x^2) + eps);   y_i = n_i c - n_{i+h} s,  y_{i+h} = n_{i+h} c + n_i s   (h = rot / 2)
//   g = the same rotation by the opposite angle of dy;  dw = sum g x r;  dx = r (g w - x r mean(g w x r))
//
// Everything between the load and the store is fp64 and rounded at the end (bf16: by way of fp32, half a step and 2^-25 off): a query's
// last bit can cross a border of the block selection that follows, and the keys of a cache must not depend on which call wrote them.  The kernel reads and writes each element once and
// costs about 8 fp64 operations per element against 4 bytes of traffic in bf16: 16384 tokens of 40 bf16 heads of 128 take 76 us, 4.4
// TB/s (a copy reaches 5.2); their arithmetic alone would take 38.  In fp32, 131072 tokens of 8 heads of 48: 83 us forward (4.8 TB/s),
// 132 backward (4.6 TB/s) and 6 for the sum of dw over the workgroups; backward of the first in bf16 139 (3.6 TB/s), in fp32 196 (5.1).  One
// token of 16 sequences: 5.8 us, latency.  (Rows asked for while the one before is computed were a fifth slower, fewer waves fit.)
//
// A row (one head of one token) is held by LPR = 2^k >= D / 8 lanes; a lane has two chunks of four elements, both halves of its
// pairs, so the rotation needs no exchange: lane l < rot/8 holds 4l.. and rot/2 + 4l.., the lanes behind it the unrotated rest.
// The cosines and sines of a token are computed once per workgroup into LDS (angle in turns, reduced exactly in fp64: a position
// of 10^6 keeps 2^-52 * 10^6 turns) and shared by its heads.
#include "attn_common.hpp"

namespace scipnp {

struct HeadNorm {
    int B, L, Hq, Hk, Hv, D, rot, first, Lout, TT;
    double eps, inv_d;
    const void *q, *k, *v;
    void *oq, *ok, *ov;
    const void *gq, *gk;
    Strides sq, sk, sv, soq, sok, sov, sgq, sgk;
    const float *wq, *wk;
    const double* turns;
    const int32_t *positions, *slots;
    double* part;                                         // backward: [workgroup][2][D]
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, double (&v)[4]) {
    if constexpr (sizeof(T) == 2) {
        const bf16x4 x = *(const bf16x4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (double)(float)x[i];
    } else {
        const f32x4a x = *(const f32x4a*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (double)x[i];
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const double (&v)[4]) {
    if constexpr (sizeof(T) == 2) {
        bf16x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (__bf16)(float)v[i];
        *(bf16x4*)p = x;
    } else {
        *(f32x4a*)p = f32x4a{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    }
}

// sum over the LPR lanes of a row, in every lane (fixed order): DPP inside a row of 16, a shuffle above
template <int LPR>
__device__ __forceinline__ double row_sum(double v) {
    if constexpr (LPR >= 2) v += dpp_f64<0xB1>(v);        // quad_perm [1,0,3,2]
    if constexpr (LPR >= 4) v += dpp_f64<0x4E>(v);        // quad_perm [2,3,0,1]
    if constexpr (LPR >= 8) v += dpp_f64<0x141>(v);       // row_half_mirror
    if constexpr (LPR >= 16) v += dpp_f64<0x140>(v);      // row_mirror
    if constexpr (LPR >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

// 1 / sqrt(x): the hardware's estimate and two Newton steps (its 2^-23 and more squares twice); 0 and infinity keep the estimate
__device__ __forceinline__ double rsqrt64(double x) {
    const double e = __builtin_amdgcn_rsq(x);
    double y = e * fma(-0.5 * x * e, e, 1.5);
    y = y * fma(-0.5 * x * y, y, 1.5);
    return y == y ? y : e;
}

// What the rows of a token share, once per workgroup in LDS: where its heads begin, and the cosines and sines of its position
struct Token { long long q, k, v, oq, ok, ov, gq, gk; int keep, pad[3]; };
struct NormLds {
    Token* tok;
    double2* cs;                                           // [token][pair] = (cos, sin)
};
__device__ __forceinline__ NormLds norm_lds(const HeadNorm& a, char* lds) { return NormLds{(Token*)lds, (double2*)(lds + a.TT * sizeof(Token))}; }
__device__ __forceinline__ void fill_tokens(const HeadNorm& a, const NormLds& s, long long t0, int nt) {
    const int half = a.rot >> 1;
    const int b0 = (int)((unsigned)t0 / (unsigned)a.L), l0 = (int)((unsigned)t0 - (unsigned)b0 * (unsigned)a.L);   // (uniform; fewer than 2^31 tokens)
    for (int i = threadIdx.x; i < nt; i += 256) {
        int b = b0, l = l0 + i;
        while (l >= a.L) { l -= a.L; ++b; }
        const int row = a.slots ? a.slots[t0 + i] : l;
        Token k;
        k.keep = row >= 0 && row < a.Lout;
        const long long r = k.keep ? row : 0;
        k.q = b * a.sq.b + l * a.sq.t;
        k.k = b * a.sk.b + l * a.sk.t;
        k.v = b * a.sv.b + l * a.sv.t;
        k.oq = b * a.soq.b + l * a.soq.t;
        k.ok = b * a.sok.b + r * a.sok.t;
        k.ov = b * a.sov.b + r * a.sov.t;
        k.gq = b * a.sgq.b + l * a.sgq.t;
        k.gk = b * a.sgk.b + l * a.sgk.t;
        s.tok[i] = k;
    }
    for (int i = threadIdx.x; i < nt * half; i += 256) {
        const int tok = nt == 1 ? 0 : i / half, pair = i - tok * half;
        int l = l0 + tok;
        while (l >= a.L) l -= a.L;
        const double pos = a.positions ? (double)a.positions[t0 + tok] : (double)(a.first + (long long)l);
        const double turn = pos * a.turns[pair];
        double sn, c;
        sincospi(2.0 * (turn - floor(turn)), &sn, &c);
        s.cs[i] = make_double2(c, sn);
    }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(256) head_norm_kernel(HeadNorm a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const NormLds s = norm_lds(a, lds);
    const int l = threadIdx.x % LPR, slot0 = threadIdx.x / LPR;
    constexpr int RPI = 256 / LPR;                        // rows per pass of the workgroup
    const long long tokens = (long long)a.B * a.L, t0 = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.TT;
    if (t0 >= tokens) return;                             // (uniform; the grid's last row)
    const int nt = (int)min((long long)a.TT, tokens - t0);
    const int nl = a.D >> 3, nr = a.rot >> 3, half = a.rot >> 1;
    const bool on = l < nl, turned = l < nr;
    const int o0 = turned ? 4 * l : a.rot + 8 * (l - nr), o1 = turned ? half + 4 * l : o0 + 4;
    const int heads = a.Hq + a.Hk + a.Hv;
    double w0q[4] = {}, w1q[4] = {}, w0k[4] = {}, w1k[4] = {};
    if (on) {
        load4(a.wq + o0, w0q);
        load4(a.wq + o1, w1q);
        if (a.Hk) { load4(a.wk + o0, w0k); load4(a.wk + o1, w1k); }
    }
    fill_tokens(a, s, t0, nt);
    __syncthreads();
    int tok = 0, hd = slot0;                              // row = (token, head); its LPR lanes share it, so the sums stay inside them
    while (hd >= heads) { hd -= heads; ++tok; }
    while (tok < nt) {
        const bool is_q = hd < a.Hq, is_v = hd >= a.Hq + a.Hk;
        const int h = is_q ? hd : is_v ? hd - a.Hq - a.Hk : hd - a.Hq;
        const Token& k = s.tok[tok];
        const T* in = (const T*)(is_q ? a.q : is_v ? a.v : a.k) + (is_q ? k.q : is_v ? k.v : k.k) + h * (is_q ? a.sq.h : is_v ? a.sv.h : a.sk.h);
        T* out = (T*)(is_q ? a.oq : is_v ? a.ov : a.ok) + (is_q ? k.oq : is_v ? k.ov : k.ok) + h * (is_q ? a.soq.h : is_v ? a.sov.h : a.sok.h);
        double x0[4] = {}, x1[4] = {};
        if (on) { load4(in + o0, x0); load4(in + o1, x1); }
        if (!is_v) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss = fma(x1[i], x1[i], fma(x0[i], x0[i], ss));
            ss = row_sum<LPR>(ss);
            const double rs = rsqrt64(fma(ss, a.inv_d, a.eps));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x0[i] *= rs * (is_q ? w0q[i] : w0k[i]);
                x1[i] *= rs * (is_q ? w1q[i] : w1k[i]);
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double2 c = s.cs[tok * half + 4 * l + i];
                    const double u = x0[i], v = x1[i];
                    x0[i] = fma(u, c.x, -(v * c.y));
                    x1[i] = fma(v, c.x, u * c.y);
                }
            }
        }
        if (on && (is_q || k.keep)) { store4(out + o0, x0); store4(out + o1, x1); }
        hd += RPI;
        while (hd >= heads) { hd -= heads; ++tok; }
    }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(256) head_norm_bwd_kernel(HeadNorm a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];        // the tile's tokens, then (reused) the workgroup's dw
    const NormLds s = norm_lds(a, lds);
    const int l = threadIdx.x % LPR, slot0 = threadIdx.x / LPR;
    constexpr int RPI = 256 / LPR;
    const long long tokens = (long long)a.B * a.L, tiles = (tokens + a.TT - 1) / a.TT;
    const int nl = a.D >> 3, nr = a.rot >> 3, half = a.rot >> 1;
    const bool on = l < nl, turned = l < nr;
    const int o0 = turned ? 4 * l : a.rot + 8 * (l - nr), o1 = turned ? half + 4 * l : o0 + 4;
    const int heads = a.Hq + a.Hk;
    double w0q[4] = {}, w1q[4] = {}, w0k[4] = {}, w1k[4] = {};
    double dq0[4] = {}, dq1[4] = {}, dk0[4] = {}, dk1[4] = {};
    if (on) {
        load4(a.wq + o0, w0q);
        load4(a.wq + o1, w1q);
        if (a.Hk) { load4(a.wk + o0, w0k); load4(a.wk + o1, w1k); }
    }
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long long t0 = tile * a.TT;
        const int nt = (int)min((long long)a.TT, tokens - t0);
        __syncthreads();
        fill_tokens(a, s, t0, nt);
        __syncthreads();
        int tok = 0, hd = slot0;
        while (hd >= heads) { hd -= heads; ++tok; }
        while (tok < nt) {
            const bool is_q = hd < a.Hq;
            const int h = is_q ? hd : hd - a.Hq;
            const Token& k = s.tok[tok];
            const T* in = (const T*)(is_q ? a.q : a.k) + (is_q ? k.q : k.k) + h * (is_q ? a.sq.h : a.sk.h);
            const T* gin = (const T*)(is_q ? a.gq : a.gk) + (is_q ? k.gq : k.gk) + h * (is_q ? a.sgq.h : a.sgk.h);
            T* out = (T*)(is_q ? a.oq : a.ok) + (is_q ? k.oq : k.ok) + h * (is_q ? a.soq.h : a.sok.h);
            double x0[4] = {}, x1[4] = {}, g0[4] = {}, g1[4] = {};
            if (on) { load4(in + o0, x0); load4(in + o1, x1); load4(gin + o0, g0); load4(gin + o1, g1); }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double2 c = s.cs[tok * half + 4 * l + i];
                    const double u = g0[i], v = g1[i];
                    g0[i] = fma(u, c.x, v * c.y);
                    g1[i] = fma(v, c.x, -(u * c.y));
                }
            }
            double ss = 0.0, gx = 0.0;                    // sum x^2, sum g w x
            double wg0[4], wg1[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wg0[i] = g0[i] * (is_q ? w0q[i] : w0k[i]);
                wg1[i] = g1[i] * (is_q ? w1q[i] : w1k[i]);
                ss = fma(x1[i], x1[i], fma(x0[i], x0[i], ss));
                gx = fma(wg1[i], x1[i], fma(wg0[i], x0[i], gx));
            }
            ss = row_sum<LPR>(ss);
            gx = row_sum<LPR>(gx);
            const double rs = rsqrt64(fma(ss, a.inv_d, a.eps)), back = -gx * a.inv_d * rs * rs * rs;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double u = x0[i] * rs, v = x1[i] * rs;
                if (is_q) { dq0[i] = fma(g0[i], u, dq0[i]); dq1[i] = fma(g1[i], v, dq1[i]); }
                else { dk0[i] = fma(g0[i], u, dk0[i]); dk1[i] = fma(g1[i], v, dk1[i]); }
                x0[i] = fma(rs, wg0[i], back * x0[i]);
                x1[i] = fma(rs, wg1[i], back * x1[i]);
            }
            if (on) { store4(out + o0, x0); store4(out + o1, x1); }
            hd += RPI;
            while (hd >= heads) { hd -= heads; ++tok; }
        }
    }
    // dw of the workgroup: the lanes that hold one column, in the order of their rows
    double* red = (double*)lds;                           // [RPI][D]
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (on) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                red[slot0 * a.D + o0 + i] = which ? dk0[i] : dq0[i];
                red[slot0 * a.D + o1 + i] = which ? dk1[i] : dq1[i];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += 256) {
            double v = 0.0;
            for (int r = 0; r < RPI; ++r) v += red[r * a.D + d];
            a.part[((size_t)blockIdx.x * 2 + which) * a.D + d] = v;
        }
    }
}

// dw[which][d] = sum over the workgroups, a fixed tree: 64 lanes take every 64th partial, then the wave sum
__global__ void __launch_bounds__(256) head_norm_dw_kernel(const double* __restrict__ part, float* dwq, float* dwk, int n, int D) {
    const int col = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (col >= 2 * D) return;
    double s = 0.0;
    for (int i = lane; i < n; i += 64) s += part[(size_t)i * 2 * D + col];
    s = wave_sum_f64(s);
    float* const dst = col < D ? dwq : dwk;
    if (lane == 0 && dst) dst[col < D ? col : col - D] = (float)s;
}

static int head_norm_check(const scipnp_head_norm_args* a, bool backward) {
    SCIPNP_BLOCK_SIZE(a, scipnp_head_norm_args);
    SCIPNP_REQUIRE(a->dtype == SCIPNP_F32 || a->dtype == SCIPNP_BF16, "dtype %d: 0 (float32) or 1 (bfloat16)", a->dtype);
    SCIPNP_REQUIRE(a->B > 0 && a->L > 0 && a->Hq > 0 && a->Hk >= 0, "B, L, Hq must be positive (got %d, %d, %d)", a->B, a->L, a->Hq);
    SCIPNP_REQUIRE(a->D >= 8 && a->D <= 256 && a->D % 8 == 0, "head size %d: a multiple of 8 up to 256", a->D);
    SCIPNP_REQUIRE(a->rot >= 0 && a->rot <= a->D && a->rot % 8 == 0, "%d rotated dimensions: a multiple of 8 up to the head size %d", a->rot, a->D);
    SCIPNP_REQUIRE(a->rot == 0 || a->turns, "rotated dimensions need turns");
    SCIPNP_REQUIRE((long long)a->B * a->L < (1ll << 31) && (long long)a->Hq + 2ll * a->Hk < 65536, "too many tokens or heads");
    SCIPNP_REQUIRE(a->eps >= 0.f, "eps must not be negative");
    SCIPNP_REQUIRE(a->q && a->out_q && a->wq, "null q, out_q or wq");
    SCIPNP_REQUIRE(!a->Hk == !a->k && (!a->k || (a->out_k && a->wk)), "k needs Hk, out_k and wk, and Hk needs k");
    SCIPNP_ALIGNED(a->q); SCIPNP_ALIGNED(a->out_q); SCIPNP_ALIGNED(a->k); SCIPNP_ALIGNED(a->out_k);
    SCIPNP_ALIGNED(a->wq); SCIPNP_ALIGNED(a->wk);
    SCIPNP_STRIDES(a->q_stride, a->dtype); SCIPNP_STRIDES(a->out_q_stride, a->dtype);
    if (a->k) { SCIPNP_STRIDES(a->k_stride, a->dtype); SCIPNP_STRIDES(a->out_k_stride, a->dtype); }
    if (!backward) {
        SCIPNP_REQUIRE(!a->v || (a->k && a->out_v), "v needs k and out_v");
        SCIPNP_REQUIRE(!a->slots || (a->k && a->Lout > 0), "slots need k and Lout");
        if (a->v) { SCIPNP_ALIGNED(a->v); SCIPNP_ALIGNED(a->out_v); SCIPNP_STRIDES(a->v_stride, a->dtype); SCIPNP_STRIDES(a->out_v_stride, a->dtype); }
    } else {
        SCIPNP_REQUIRE(a->g_q && a->dwq && (!a->k || (a->g_k && a->dwk)), "backward needs g_q, dwq (g_k, dwk)");
        SCIPNP_ALIGNED(a->g_q); SCIPNP_ALIGNED(a->g_k); SCIPNP_STRIDES(a->g_q_stride, a->dtype);
        if (a->k) SCIPNP_STRIDES(a->g_k_stride, a->dtype);
    }
    return SCIPNP_OK;
}

// tokens per workgroup: one while there are few (each is then its own workgroup), enough rows for eight passes of 256 threads otherwise (what a
// workgroup does once, weights and angles, weighs on two: 16384 tokens of 48 bf16 heads of 128 take 99 us with two, 79 with eight, 84 with 16)
static int head_norm_tokens(const scipnp_head_norm_args* a, int lpr) {
    const long long tokens = (long long)a->B * a->L;
    const int heads = a->Hq + a->Hk + (a->v ? a->Hk : 0), rows = 8 * 256 / lpr;
    int tt = (rows + heads - 1) / heads;
    if (tt > 16) tt = 16;
    while (tt > 1 && tokens / tt < 1024) tt >>= 1;
    return tt < 1 ? 1 : tt;
}
static int head_norm_lpr(int D) { int l = 1; while (l * 8 < D) l <<= 1; return l; }
static int head_norm_bwd_groups(const scipnp_head_norm_args* a) {
    const int tt = head_norm_tokens(a, head_norm_lpr(a->D));
    const long long tiles = ((long long)a->B * a->L + tt - 1) / tt;
    // three workgroups a CU, as many as the registers hold (149 to 165 in every form of the kernel; four: a second round a third full, 164 + 7
    // instead of 139 + 6 us at 131072 fp32 tokens of 8 heads of 48), each with its
    // share of dw
    return (int)(tiles < 768 ? tiles : 768);
}

static HeadNorm head_norm_params(const scipnp_head_norm_args* a) {
    HeadNorm p = {};
    p.B = a->B; p.L = a->L; p.Hq = a->Hq; p.Hk = a->Hk; p.Hv = a->v ? a->Hk : 0; p.D = a->D; p.rot = a->rot; p.first = a->first;
    p.Lout = a->slots ? a->Lout : a->L;
    p.eps = (double)a->eps; p.inv_d = 1.0 / a->D;
    p.q = a->q; p.k = a->k; p.v = a->v; p.oq = a->out_q; p.ok = a->out_k; p.ov = a->out_v; p.gq = a->g_q; p.gk = a->g_k;
    p.sq = strides_of(a->q_stride); p.sk = strides_of(a->k_stride); p.sv = strides_of(a->v_stride);
    p.soq = strides_of(a->out_q_stride); p.sok = strides_of(a->out_k_stride); p.sov = strides_of(a->out_v_stride);
    p.sgq = strides_of(a->g_q_stride); p.sgk = strides_of(a->g_k_stride);
    p.wq = a->wq; p.wk = a->wk; p.turns = a->turns; p.positions = a->positions; p.slots = a->slots;
    return p;
}

template <int LPR>
static void head_norm_launch(const HeadNorm& p, int dtype, bool backward, dim3 grid, hipStream_t st) {
    size_t lds = (size_t)p.TT * (sizeof(Token) + (p.rot / 2) * sizeof(double2));
    if (backward) {
        const size_t red = (size_t)(256 / LPR) * p.D * sizeof(double);
        lds = lds > red ? lds : red;
        if (dtype == SCIPNP_BF16) head_norm_bwd_kernel<__bf16, LPR><<<grid, 256, lds, st>>>(p);
        else head_norm_bwd_kernel<float, LPR><<<grid, 256, lds, st>>>(p);
    } else {
        if (dtype == SCIPNP_BF16) head_norm_kernel<__bf16, LPR><<<grid, 256, lds, st>>>(p);
        else head_norm_kernel<float, LPR><<<grid, 256, lds, st>>>(p);
    }
}
static void head_norm_dispatch(int lpr, const HeadNorm& p, int dtype, bool backward, dim3 grid, hipStream_t st) {
    switch (lpr) {
        case 1: head_norm_launch<1>(p, dtype, backward, grid, st); break;
        case 2: head_norm_launch<2>(p, dtype, backward, grid, st); break;
        case 4: head_norm_launch<4>(p, dtype, backward, grid, st); break;
        case 8: head_norm_launch<8>(p, dtype, backward, grid, st); break;
        case 16: head_norm_launch<16>(p, dtype, backward, grid, st); break;
        default: head_norm_launch<32>(p, dtype, backward, grid, st); break;
    }
}

}  // namespace scipnp

using namespace scipnp;

extern "C" {

int scipnp_head_norm_rotate(const scipnp_head_norm_args* a, scipnp_stream_t s) {
    if (const int rc = head_norm_check(a, false)) return rc;
    HeadNorm p = head_norm_params(a);
    const int lpr = head_norm_lpr(a->D);
    p.TT = head_norm_tokens(a, lpr);
    const long long tiles = ((long long)a->B * a->L + p.TT - 1) / p.TT;
    // (a dimension of the grid holds 2^32 threads: 2^24 workgroups, of which 2^28 tokens of one small head are too many)
    const long long row = tiles < (1 << 22) ? tiles : 1 << 22;
    head_norm_dispatch(lpr, p, a->dtype, false, dim3((unsigned)row, (unsigned)((tiles + row - 1) / row)), (hipStream_t)s);
    return launch_status("scipnp_head_norm_rotate");
}

size_t scipnp_head_norm_rotate_backward_workspace_bytes(const scipnp_head_norm_args* a) {
    if (!a || a->struct_size != sizeof(scipnp_head_norm_args) || a->B <= 0 || a->L <= 0 || a->Hq <= 0 || a->Hk < 0 || a->D <= 0 || a->D > 256) return 0;
    return (size_t)head_norm_bwd_groups(a) * 2 * a->D * sizeof(double);
}

int scipnp_head_norm_rotate_backward(const scipnp_head_norm_args* a, scipnp_stream_t s) {
    if (const int rc = head_norm_check(a, true)) return rc;
    if (!a->workspace || a->workspace_bytes < scipnp_head_norm_rotate_backward_workspace_bytes(a))
        return fail(SCIPNP_EWORKSPACE, "head norm backward: workspace of %zu bytes needed", scipnp_head_norm_rotate_backward_workspace_bytes(a));
    HeadNorm p = head_norm_params(a);
    const int lpr = head_norm_lpr(a->D);
    p.Hv = 0;
    p.TT = head_norm_tokens(a, lpr);
    p.part = (double*)a->workspace;
    const int n = head_norm_bwd_groups(a);
    head_norm_dispatch(lpr, p, a->dtype, true, dim3((unsigned)n), (hipStream_t)s);
    head_norm_dw_kernel<<<(2 * a->D + 3) / 4, 256, 0, (hipStream_t)s>>>(p.part, a->dwq, a->dwk, n, a->D);
    return launch_status("scipnp_head_norm_rotate_backward");
}

}
