// Tile pieces of the block-attention kernels: 32 x 32 products on the matrix cores from tiles in LDS.
//
// An accumulator f32x16 of v_mfma_f32_32x32x* is held as: lane (li = lane & 31, hi = lane >> 5), register r -> row 8*(r>>2) + 4*hi + (r&3),
// column li.  The scores are computed transposed, S^T[key][row] = K Q^T, so a lane holds 16 keys of ONE query row: the softmax needs
// one exchange (with lane ^ 32), and the registers of P^T are, in their order, the B operand of O^T = V^T P^T -- the order of the
// contraction's slots is free as long as V is read in the same one, so P never leaves its registers.
#pragma once
#include <climits>
#include "attn_common.hpp"

namespace scipnp {

constexpr int KT = 32;                                    // keys (rows) of a tile

template <typename T> struct Mat;
template <> struct Mat<__bf16> {
    typedef bf16x8 Frag;
    static constexpr int E = 8;                           // elements of 16 bytes
    static constexpr int K = 16;                          // contraction of one fragment
};
template <> struct Mat<float> {
    typedef f32x4a Frag;
    static constexpr int E = 4;
    static constexpr int K = 8;                           // four v_mfma_f32_32x32x2_f32 a fragment
};

// element stride of an LDS tile that is read row-wise (16 bytes of 32 rows): 4 banks further each row
template <typename T, int DP> constexpr int row_stride() { return DP + Mat<T>::E; }
// ... of one that is only read transposed: bf16 4 rows x 32 columns cover the 64 banks once; fp32 rows 4 apart are 32 banks apart
template <typename T, int DP> constexpr int col_stride() { return sizeof(T) == 2 ? (DP == 128 ? 160 : DP == 64 ? 96 : DP) : DP + 8; }

// acc += A B^T over DP: A = the tile's row li (LDS), B = fragments in registers
template <typename T, int DP>
__device__ __forceinline__ f32x16a mma_rows(const T* row, const typename Mat<T>::Frag (&b)[DP / Mat<T>::K], int hi, f32x16a acc) {
#pragma unroll
    for (int s = 0; s < DP / Mat<T>::K; ++s) {
        if constexpr (sizeof(T) == 2) {
            const bf16x8 a = *(const bf16x8*)(row + 16 * s + 8 * hi);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[s], acc, 0, 0, 0);
        } else {
            const f32x4a a = *(const f32x4a*)(row + 8 * s + 4 * hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[s][j], acc, 0, 0, 0);
        }
    }
    return acc;
}

// acc[db] += X^T P over the tile's 32 rows: X the tile (element stride ST), P in an accumulator's registers, rounded to T.
// exact (bf16): P as three bf16 numbers that add up to its 24 bits, three products
template <typename T, int DP, int ST>
__device__ __forceinline__ void mma_cols(const T* tile, const f32x16a& p, int lane, f32x16a (&acc)[DP / 32], bool exact = false) {
    const int li = lane & 31, hi = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        // transposing read: the 16 lanes of a group supply 4 rows x 16 columns (8 bytes each) and receive a column's 4 rows
        const int q = (lane >> 2) & 3, c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            bf16x8 b, b1, b2;
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = (__bf16)p[8 * k + i];
            if (exact) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r1 = p[8 * k + i] - (float)b[i];
                    b1[i] = (__bf16)r1;
                    b2[i] = (__bf16)(r1 - (float)b1[i]);
                }
            }
            const T* base = tile + (16 * k + 4 * hi + q) * ST + c;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                union { s16x4a s[2]; bf16x8 v; } u;
                u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4a*)(base + 32 * db));
                u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4a*)(base + 8 * ST + 32 * db));
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, b, acc[db], 0, 0, 0);
                if (exact) {
                    acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, b1, acc[db], 0, 0, 0);
                    acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, b2, acc[db], 0, 0, 0);
                }
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const T* x = tile + (8 * (r >> 2) + 4 * hi + (r & 3)) * ST + li;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[32 * db], p[r], acc[db], 0, 0, 0);
        }
    }
}

// fragments of one row in global memory (nullptr: zeros); columns past D are zero
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const T* row, int D, int hi, typename Mat<T>::Frag (&f)[DP / Mat<T>::K]) {
#pragma unroll
    for (int s = 0; s < DP / Mat<T>::K; ++s) {
        const int c = Mat<T>::K * s + Mat<T>::E * hi;
        if (row && c < D) f[s] = *(const typename Mat<T>::Frag*)(row + c);
        else
#pragma unroll
            for (int i = 0; i < Mat<T>::E; ++i) f[s][i] = (T)0.f;
    }
}

// ---- a tile on its way from global memory to LDS: 32 rows of DP elements, NTH threads, 16 bytes each
template <typename T, int DP, int NTH>
struct TileRegs {
    static constexpr int C = DP / Mat<T>::E;              // 16-byte chunks of a row
    static constexpr int N = (KT * C + NTH - 1) / NTH;
    static constexpr bool EVEN = KT * C % NTH == 0;
    f32x4a v[N];
    // row_of(i): address of row i's first element, nullptr for a row that is zeros
    template <typename F>
    __device__ __forceinline__ void load(int t, int D, F row_of) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = t + i * NTH, r = x / C, c = (x - r * C) * Mat<T>::E;
            const T* p = EVEN || r < KT ? row_of(r) : nullptr;
            v[i] = (p && c < D) ? *(const f32x4a*)(p + c) : f32x4a{0.f, 0.f, 0.f, 0.f};
        }
    }
    template <int ST>
    __device__ __forceinline__ void store(int t, T* tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = t + i * NTH, r = x / C, c = (x - r * C) * Mat<T>::E;
            if (EVEN || r < KT) *(f32x4a*)(tile + r * ST + c) = v[i];
        }
    }
};

// ---- a tile that the memory system writes into LDS itself (buffer_load ... lds: no registers, no address arithmetic per tile)
//
// 32 rows of LC = 2^n >= DP * sizeof(T) / 16 chunks of 16 bytes, packed (a wave's request writes 1 KB in lane order); chunk c of row r
// lies at chunk c ^ swz(r), so that both ways of reading meet every bank once: 16 rows at one chunk (the A operand of a score product),
// and, transposed, 4 rows x 4 chunks (bf16) or two rows 4 apart x 8 chunks (fp32).  Rows past the live ones and columns past D
// come back as zeros (requests outside the buffer descriptor), whatever lies behind them in memory.
template <typename T, int DP> constexpr int lds_chunks() {
    const int n = DP * (int)sizeof(T) / 16;
    return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;
}
template <typename T, int LC>
__device__ __forceinline__ int swz(int row) {
    if constexpr (sizeof(T) == 4) return LC >= 16 ? ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3) : (row >> 1) & 7;
    else return LC >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : LC == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
}
template <typename T, int DP>
struct DmaTile {
    static constexpr int LC = lds_chunks<T, DP>();
    static constexpr int BYTES = KT * LC * 16;
    static constexpr int PIECES = BYTES / 1024;
};
constexpr unsigned DMA_NONE = 0xFFFFFF00u;                // an offset outside every descriptor

// this lane's offsets of a wave's pieces (piece = first + i * step): row * stride + chunk * 16
template <typename T, int DP, int STEP>
struct DmaOffsets {
    static constexpr int N = (DmaTile<T, DP>::PIECES + STEP - 1) / STEP;
    unsigned off[N];
    __device__ __forceinline__ void init(int first, int lane, unsigned stride_bytes, int D) {
        constexpr int LC = DmaTile<T, DP>::LC;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int x = (first + i * STEP) * 64 + lane, row = x / LC, c = (x % LC) ^ swz<T, LC>(row);
            off[i] = c * Mat<T>::E < D && row < KT ? (unsigned)row * stride_bytes + 16u * c : DMA_NONE;
        }
    }
    // `base`: the tile's first row (wave-uniform); `live` rows of it exist
    __device__ __forceinline__ void issue(const void* base, int live, unsigned stride_bytes, int D, char* tile, int first) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)(live - 1) * stride_bytes + (unsigned)(D * (int)sizeof(T)), 0x00020000);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int piece = first + i * STEP;
            if (DmaTile<T, DP>::PIECES % STEP == 0 || piece < DmaTile<T, DP>::PIECES)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(tile + 1024 * piece), 16, off[i], 0, 0, 0);
        }
#endif
    }
};

// score products: acc += A B^T, A = row li of the tile
template <typename T, int DP>
__device__ __forceinline__ f32x16a dma_rows(const char* tile, const typename Mat<T>::Frag (&b)[DP / Mat<T>::K], int lane, f32x16a acc) {
    constexpr int LC = DmaTile<T, DP>::LC;
    const int li = lane & 31, x = (lane >> 5) ^ swz<T, LC>(li);
    const char* row = tile + li * LC * 16;
#pragma unroll
    for (int s = 0; s < DP / Mat<T>::K; ++s) {
        const typename Mat<T>::Frag a = *(const typename Mat<T>::Frag*)(row + ((x ^ (2 * s)) << 4));
        if constexpr (sizeof(T) == 2) {
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[s], acc, 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[s][j], acc, 0, 0, 0);
        }
    }
    return acc;
}

// transposing reads of one or two column blocks (4 rows and the 4 rows 8 below): the 16 lanes of a group supply 4 rows x 16 columns (8
// bytes each) and receive a column's 4 rows.  Written as assembly because the compiler takes the builtin for a reader of every request
// in flight and waits for the NEXT tile in front of it; each block waits for its own reads.
typedef unsigned u32x2a __attribute__((ext_vector_type(2)));
template <int OFF, int DOWN>
__device__ __forceinline__ void tr_read(unsigned a0, unsigned a1, bf16x8& x) {
#if defined(__HIP_DEVICE_COMPILE__)
    union { u32x2a s[2]; bf16x8 v; } u;
    asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%4\n\tds_read_b64_tr_b16 %1, %3 offset:%5\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(u.s[0]), "=&v"(u.s[1]) : "v"(a0), "v"(a1), "n"(OFF), "n"(OFF + DOWN));
    x = u.v;
#endif
}
template <int OFF, int DOWN>
__device__ __forceinline__ void tr_read2(unsigned a0, unsigned a1, unsigned b0, unsigned b1, bf16x8& x, bf16x8& y) {
#if defined(__HIP_DEVICE_COMPILE__)
    union { u32x2a s[2]; bf16x8 v; } u, w;
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%9\n\t"
                 "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%9\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(u.s[0]), "=&v"(u.s[1]), "=&v"(w.s[0]), "=&v"(w.s[1])
                 : "v"(a0), "v"(a1), "v"(b0), "v"(b1), "n"(OFF), "n"(OFF + DOWN));
    x = u.v;
    y = w.v;
#endif
}

// second products: acc[db] += X^T P over the tile's 32 rows, P in an accumulator's registers, rounded to T.  EXACT (bf16): P as three
// bf16 numbers that add up to its 24 bits, three products
template <typename T, int DP, bool EXACT = false>
__device__ __forceinline__ void dma_cols(const char* tile, const f32x16a& p, int lane, f32x16a (&acc)[(DP + 31) / 32]) {
    constexpr int LC = DmaTile<T, DP>::LC, NB = (DP + 31) / 32;
    const int li = lane & 31, hi = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int q = (lane >> 2) & 3, c0 = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), r0 = 4 * hi + q;
        const unsigned base = (unsigned)(size_t)(__attribute__((address_space(3))) const char*)tile + r0 * LC * 16 + 8 * (lane & 1);
        const int f0 = c0 ^ swz<T, LC>(r0), f1 = c0 ^ swz<T, LC>(r0 + 8);
        bf16x8 pb[2], p1[2], p2[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = p[8 * k + i];
                pb[k][i] = (__bf16)x;
                if constexpr (EXACT) {
                    const float r1 = x - (float)pb[k][i];
                    p1[k][i] = (__bf16)r1;
                    p2[k][i] = (__bf16)(r1 - (float)p1[k][i]);
                }
            }
        auto product = [&](int db, int k, const bf16x8& x) {
            acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pb[k], acc[db], 0, 0, 0);
            if constexpr (EXACT) {
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, p1[k], acc[db], 0, 0, 0);
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, p2[k], acc[db], 0, 0, 0);
            }
        };
        constexpr int STEP = 16 * LC * 16, DOWN = 8 * LC * 16;             // 16 rows, 8 rows
#pragma unroll
        for (int db = 0; db + 1 < NB; db += 2) {
            const unsigned a0 = base + ((f0 ^ (4 * db)) << 4), a1 = base + ((f1 ^ (4 * db)) << 4);
            const unsigned b0 = base + ((f0 ^ (4 * db + 4)) << 4), b1 = base + ((f1 ^ (4 * db + 4)) << 4);
            bf16x8 x, y;
            tr_read2<0, DOWN>(a0, a1, b0, b1, x, y);
            product(db, 0, x);
            product(db + 1, 0, y);
            tr_read2<STEP, DOWN>(a0, a1, b0, b1, x, y);
            product(db, 1, x);
            product(db + 1, 1, y);
        }
        if constexpr (NB & 1) {
            const unsigned a0 = base + ((f0 ^ (4 * (NB - 1))) << 4), a1 = base + ((f1 ^ (4 * (NB - 1))) << 4);
            bf16x8 x;
            tr_read<0, DOWN>(a0, a1, x);
            product(NB - 1, 0, x);
            tr_read<STEP, DOWN>(a0, a1, x);
            product(NB - 1, 1, x);
        }
    } else {
        const char* base = tile + 4 * hi * LC * 16 + 4 * (li & 3);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = 8 * (r >> 2) + (r & 3);        // + 4 hi
            const int f = (li >> 2) ^ swz<T, LC>(row + 4 * hi);
#pragma unroll
            for (int db = 0; db < NB; ++db) {
                const float x = *(const float*)(base + row * LC * 16 + ((f ^ (8 * db)) << 4));
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[r], acc[db], 0, 0, 0);
            }
        }
    }
}
// all of this wave's requests have landed; every wave's, with more than one
template <int WAVES>
__device__ __forceinline__ void dma_wait() {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (WAVES == 1) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}

// ---- what every kernel knows of the call
struct Attn {
    int B, Lq, Lk, Hq, Hk, G, D, block, qb, n, causal, nbuckets, maxd, nb, ng;
    int chunks, splits;                                   // forward: row chunks of a group, parts of its keys
    float scale, scale2;                                  // scale2 = scale * log2(e)
    const void *q, *k, *v, *dout;
    void* out;
    Strides sq, sk, sv, so, sdo;
    const int32_t *sel, *qlen, *klen, *bucket_of, *q_pos, *k_pos;
    const float* bias;
    float *lse, *out32;
    void *dq, *dk, *dv;
    float* dbias;
    float *po, *pml;                                      // forward, splits > 1: partial results, their maxima and sums
    // backward
    const float* delta;
    unsigned* member;                                     // [b, hk][key block][ng bits]
    int words;
    const int* chunk_start;                               // [b, hk][key block + 1]
    int max_chunks;
    float* pkv;                                           // partial dk, dv
    double* pbias;
};

struct Seq { int qlen, klen, shift; };                    // shift: key position of query 0
__device__ __forceinline__ Seq seq_of(const Attn& a, int b) {
    Seq s;
    s.qlen = a.qlen ? min(max(a.qlen[b], 0), a.Lq) : a.Lq;
    s.klen = a.klen ? min(max(a.klen[b], 0), a.Lk) : a.Lk;
    s.shift = s.klen - s.qlen;
    return s;
}

// the blocks of a selection that count, in order: one wave; returns their number.  `limit`: keys from there on are not wanted
__device__ __forceinline__ int live_blocks(const Attn& a, const int32_t* sel, int limit, int* list, int lane) {
    int count = 0, top = -1;
    for (int base = 0; base < a.n; base += 64) {
        int e = base + lane < a.n ? sel[base + lane] : -1;
        if (e >= a.nb) e = -1;
        int run = e;                                      // greatest entry up to this one
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(run, off, 64);
            if (lane >= off) run = max(run, o);
        }
        int before = __shfl_up(run, 1, 64);
        before = lane == 0 ? top : max(before, top);
        const bool ok = e >= 0 && e > before && (long long)e * a.block < limit;
        const unsigned long long m = __ballot(ok);
        if (ok) list[count + __popcll(m & ((1ull << lane) - 1))] = e;
        count += __popcll(m);
        top = max(top, __shfl(run, 63, 64));
    }
    return count;
}

// ---- scores of a tile: 32 keys of a lane's row, masked, with the bias
struct Bias {                                             // in LDS: the bucket of each clamped distance, the workgroup's heads
    const unsigned char* lut;
    const float* tbl;
};
// scores are kept in units of ln 2 (exp2 needs no product); a finite bias stays finite
__device__ __forceinline__ float bias_log2(float b) {
    const float x = b * LOG2E;
    return __builtin_isinf(x) && !__builtin_isinf(b) ? copysignf(3.402823466e38f, b) : x;
}
__device__ __forceinline__ Bias load_bias(const Attn& a, char* lds, int hk) {
    Bias s;
    unsigned char* lut = (unsigned char*)lds;
    float* tbl = (float*)(lds + (2 * a.maxd + 1 + 3) / 4 * 4);
    s.lut = lut;
    s.tbl = tbl;
    if (a.nbuckets) {
        for (int i = threadIdx.x; i < 2 * a.maxd + 1; i += blockDim.x) lut[i] = (unsigned char)min(max(a.bucket_of[i], 0), a.nbuckets - 1);
        for (int i = threadIdx.x; i < a.nbuckets * a.G; i += blockDim.x) tbl[i] = bias_log2(a.bias[(size_t)(i / a.G) * a.Hq + hk * a.G + i % a.G]);
    }
    return s;
}
__device__ __forceinline__ int clamp_dist(int d, int maxd) { return min(max(d, -maxd), maxd) + maxd; }
__device__ __forceinline__ int tile_key(int r, int hi) { return 8 * (r >> 2) + 4 * hi + (r & 3); }

// What the 32 keys of a tile and the rows of a wave have in common.  Distances are clamped, so a tile that lies beyond one end for
// every row, or whose positions are all equal (the frames of a picture), has ONE bucket a row: one LDS read instead of sixteen pairs.
struct RowRange { int lo, hi; };                          // positions of the wave's live rows
__device__ __forceinline__ int tile_distance(const Attn& a, RowRange q, int key0, const int* kp, int lane) {   // -1: not one bucket
    int klo = key0, khi = key0 + KT - 1;
    if (kp) {
        const int mine = kp[lane & 31];
        klo = khi = __builtin_amdgcn_readfirstlane(mine);
        if (__ballot(mine != klo)) return -1;
    }
    const int lo = clamp_dist(klo - q.hi, a.maxd), hi = clamp_dist(khi - q.lo, a.maxd);
    return lo == hi ? lo : -1;
}
// the bias of 16 scores of a lane's row, position by position
__device__ __forceinline__ void tile_bias(const Attn& a, const Bias& s, int key0, const int* kp, int qp, int gl, int hi, float (&x)[16]) {
    int d[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) d[r] = s.lut[clamp_dist((kp ? kp[tile_key(r, hi)] : key0 + tile_key(r, hi)) - qp, a.maxd)];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = s.tbl[d[r] * a.G + gl];
}
inline size_t bias_lds(int nbuckets, int maxd, int G) { return nbuckets ? ((size_t)(2 * maxd + 1 + 3) / 4 * 4 + (size_t)nbuckets * G * 4 + 15) / 16 * 16 : 0; }

}  // namespace scipnp
