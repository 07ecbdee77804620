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

// ---- a tile that the memory system writes into LDS itself (buffer_load ... lds: no registers, no address arithmetic per tile)
//
// 32 rows of LC >= DP * sizeof(T) / 16 chunks of 16 bytes, LC a power of two or 12, packed (a wave's request writes 1 KB in lane order); chunk c of row r
// lies at chunk c ^ swz(r), so that both ways of reading meet every bank once: 16 rows at one chunk (the A operand of a score product),
// and, transposed, 4 rows x 4 chunks (bf16) or two rows 4 apart x 8 chunks (fp32).  Rows past the live ones and columns past D
// come back as zeros (requests outside the buffer descriptor), whatever lies behind them in memory.
template <typename T, int DP> constexpr int lds_chunks() {
    const int n = DP * (int)sizeof(T) / 16;
    return n <= 4 ? 4 : n <= 8 ? 8 : sizeof(T) == 4 && n == 12 ? 12 : n <= 16 ? 16 : 32;
}
template <typename T, int LC>
__device__ __forceinline__ int swz(int row) {
    if constexpr (LC == 12) return (row >> 2) & 3;        // (rows begin 48 banks apart: four of them meet every 16th)
    else if constexpr (sizeof(T) == 4) return LC >= 16 ? ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3) : (row >> 1) & 7;
    else return LC >= 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : LC == 8 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
}
template <typename T, int DP>
struct DmaTile {
    static constexpr int LC = lds_chunks<T, DP>();
    static constexpr int BYTES = KT * LC * 16;
    static constexpr int PIECES = BYTES / 1024;
};
constexpr unsigned DMA_NONE = 0x80000000u;                // an offset outside every descriptor, and so with a tile's rows added (token strides are below 2^26 bytes)

// this lane's offsets of a wave's pieces (piece = first + i * step): row * stride + chunk * 16
template <typename T, int DP, int STEP>
struct DmaOffsets {
    static constexpr int N = (DmaTile<T, DP>::PIECES + STEP - 1) / STEP, LC = DmaTile<T, DP>::LC;
    // the swizzle repeats every 16 rows: pieces that far apart have one offset, but for those rows (held each for itself, the offsets of
    // 128 bf16 columns would be four registers more than three waves a SIMD have)
    static constexpr int period() {
        int p = 1;
        while (p < N && p * STEP * 64 % (16 * LC)) ++p;
        return p;
    }
    static constexpr int P = period(), ROWS = P * STEP * 64 / LC;
    unsigned off[P];
    __device__ __forceinline__ void init(int first, int lane, unsigned stride_bytes, int D) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
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
            unsigned at = off[i % P];
            if (i >= P) {
                asm volatile("" : "+v"(at));              // (or the compiler adds in front of the loop and holds the sums)
                at += i / P * ROWS * stride_bytes;
            }
            if (DmaTile<T, DP>::PIECES % STEP == 0 || piece < DmaTile<T, DP>::PIECES)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(tile + 1024 * piece), 16, at, 0, 0, 0);
        }
#endif
    }
};

// the positions of a tile's keys, the same way: `live` of 32, zeros behind them
__device__ __forceinline__ void issue_positions(const int* base, int live, int* to, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)live * 4u, 0x00020000);
    asm volatile("" : "+v"(lane));                        // (no register holds the offset between tiles)
    if (lane < KT) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)to, 4, 4 * lane, 0, 0, 0);
#endif
}

// score products: A B^T, A = row li of the tile.  read() brings the rows into registers (all reads under way at once), mma() multiplies
template <typename T, int DP>
struct RowTile {
    static constexpr int LC = DmaTile<T, DP>::LC, N = DP / Mat<T>::K;
    typename Mat<T>::Frag a[N];
    __device__ __forceinline__ void read(const char* tile, int lane) {
        const int li = lane & 31, x = (lane >> 5) ^ swz<T, LC>(li);
        const char* row = tile + li * LC * 16;
#pragma unroll
        for (int s = 0; s < N; ++s) a[s] = *(const typename Mat<T>::Frag*)(row + ((x ^ (2 * s)) << 4));
    }
    __device__ __forceinline__ f32x16a mma(const typename Mat<T>::Frag (&b)[N]) const {
        f32x16a acc;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll
        for (int s = 0; s < N; ++s) {
            if constexpr (sizeof(T) == 2) {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[s], b[s], acc, 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s][j], b[s][j], acc, 0, 0, 0);
            }
        }
        return acc;
    }
};
template <typename T, int DP, bool LEAN = false>          // LEAN: the compiler may read a part at a time, in fewer registers
__device__ __forceinline__ f32x16a dma_rows(const char* tile, const typename Mat<T>::Frag (&b)[DP / Mat<T>::K], int lane) {
    RowTile<T, DP> r;
    r.read(tile, lane);
    if constexpr (!LEAN) __builtin_amdgcn_sched_barrier(0);
    return r.mma(b);
}

// second products: acc += X^T P over the tile's 32 rows (P in an accumulator's registers, rounded to T), NB column blocks of 32.
// bf16: read() brings the transposed tile into registers, early, so that the reads overlap the score products and the softmax;
//   the 16 lanes of a group supply 4 rows x 16 columns (8 bytes each) and receive a column's 4 rows.  Assembly because the compiler
//   takes the builtin for a reader of every request in flight and waits for the NEXT tile in front of it; the block waits for its reads.
//   Column 32 db + m is row m of block db.  PARTS: the bf16 numbers that P is split into, a product each; 3 hold its 24 bits, 2 hold 16.
// fp32: with 2 or 4 blocks a lane reads 2 or 4 neighbouring columns at once: column NB m + db is row m of block db.
//   With 16 columns left over (48 wide) the blocks are 16 wide and nothing is multiplied with padding: two swaps of 16 lanes bring four
//   keys of 16 rows beside each other, which is the operand of v_mfma_f32_16x16x4_f32.
typedef unsigned u32x2a __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void swap16(float& x, float& y) {        // lanes 16-31 and 48-63 of x with lanes 0-15 and 32-47 of y
#if defined(__HIP_DEVICE_COMPILE__)
    const u32x2a z = __builtin_bit_cast(u32x2a, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false));
    x = __uint_as_float(z[0]);
    y = __uint_as_float(z[1]);
#endif
}
__device__ __forceinline__ void swap32(float& x, float& y) {        // lanes 32-63 of x with lanes 0-31 of y
#if defined(__HIP_DEVICE_COMPILE__)
    const u32x2a z = __builtin_bit_cast(u32x2a, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false));
    x = __uint_as_float(z[0]);
    y = __uint_as_float(z[1]);
#endif
}
// sums of second products; blocks() gives them as column blocks of 32
template <typename T, int DP>
struct Acc {
    static constexpr int NB = (DP + 31) / 32;
    static constexpr bool N16 = sizeof(T) == 4 && DP % 32 == 16;    // [16 columns][rows 0-15, 16-31]: row lane & 15, columns 4 (lane >> 4) + i
    f32x16a x[N16 ? 1 : NB];
    f32x4a y[N16 ? DP / 16 : 1][2];
    __device__ __forceinline__ void zero() {
        if constexpr (N16)
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) y[c][0] = y[c][1] = f32x4a{0.f, 0.f, 0.f, 0.f};
        else
#pragma unroll
            for (int db = 0; db < NB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[db][r] = 0.f;
    }
    __device__ __forceinline__ void scale(float f) {      // f: of row lane & 31
        if constexpr (N16) {
            float f0 = f, f1 = f;
            swap16(f0, f1);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) { y[c][0][i] *= f0; y[c][1][i] *= f1; }
        } else {
#pragma unroll
            for (int db = 0; db < NB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[db][r] *= f;
        }
    }
    __device__ __forceinline__ void blocks(f32x16a (&o)[NB]) const {
#pragma unroll
        for (int db = 0; db < NB; ++db) {
            if constexpr (!N16) o[db] = x[db];
            else
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
        }
        if constexpr (N16)
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float u = y[c][0][i], v = y[c][1][i];
                    swap16(u, v);
                    swap32(u, v);
                    o[c / 2][8 * (c & 1) + i] = u;
                    o[c / 2][8 * (c & 1) + 4 + i] = v;
                }
    }
};
// P in front of a second product: bf16, PARTS numbers a weight (each what the ones before it left over); fp32, as it is
template <typename T, int PARTS>
struct Weights {
    bf16x8 p[PARTS][2];
    __device__ __forceinline__ explicit Weights(const f32x16a& x) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                f32x2a rest = {x[8 * k + i], x[8 * k + i + 1]};
#pragma unroll
                for (int n = 0; n < PARTS; ++n) {
                    const bf16x2 y = __builtin_convertvector(rest, bf16x2);
                    p[n][k][i] = y[0];
                    p[n][k][i + 1] = y[1];
                    if (n + 1 < PARTS) {                  // (their floats from the pair's bits: the compiler would convert each a second time)
                        unsigned u = __builtin_bit_cast(unsigned, y);
                        rest[0] -= __uint_as_float(u << 16);
                        rest[1] -= __uint_as_float(u & 0xFFFF0000u);
                    }
                }
            }
    }
};
template <int PARTS>
struct Weights<float, PARTS> {
    const f32x16a& x;
    __device__ __forceinline__ explicit Weights(const f32x16a& x_) : x(x_) {}
};
template <typename T, int DP, int PART = (DP + 31) / 32>   // PART: column blocks held at a time (bf16)
struct ColTile {
    static constexpr int LC = DmaTile<T, DP>::LC, NB = PART;
    union Pair { u32x2a s[2]; bf16x8 v; };
    Pair u[sizeof(T) == 2 ? NB : 1][2];
    const char* tile;
    int lane;
    __device__ __forceinline__ void at(const char* tile_, int lane_) {
        tile = tile_;
        lane = lane_;
    }
    __device__ __forceinline__ void read(const char* tile_, int lane_, int first = 0) {
        at(tile_, lane_);
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (sizeof(T) == 2) {
            const int q = (lane >> 2) & 3, c0 = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), r0 = 4 * (lane >> 5) + q;
            const unsigned base = (unsigned)(size_t)(__attribute__((address_space(3))) const char*)tile + r0 * LC * 16 + 8 * (lane & 1);
            const int f0 = c0 ^ swz<T, LC>(r0), f1 = c0 ^ swz<T, LC>(r0 + 8);
            constexpr int STEP = 16 * LC * 16, DOWN = 8 * LC * 16;         // 16 rows, 8 rows
            unsigned from[2 * NB];
#pragma unroll
            for (int db = 0; db < NB; ++db) {
                from[2 * db] = base + ((f0 ^ (4 * (first + db))) << 4);
                from[2 * db + 1] = base + ((f1 ^ (4 * (first + db))) << 4);
            }
            read_blocks<STEP, DOWN>(from);
        }
#endif
    }
#if defined(__HIP_DEVICE_COMPILE__)
    template <int STEP, int DOWN>
    __device__ __forceinline__ void read_blocks(const unsigned (&at)[2 * NB]) {
        if constexpr (NB == 1)
            asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
                     "ds_read_b64_tr_b16 %1, %5 offset:%7\n\t"
                     "ds_read_b64_tr_b16 %2, %4 offset:%8\n\t"
                     "ds_read_b64_tr_b16 %3, %5 offset:%9\n\t"
                     "s_waitcnt lgkmcnt(0)"
                         : "=&v"(u[0][0].s[0]), "=&v"(u[0][0].s[1]), "=&v"(u[0][1].s[0]), "=&v"(u[0][1].s[1])
                         : "v"(at[0]), "v"(at[1]), "n"(0), "n"(DOWN), "n"(STEP), "n"(STEP + DOWN));
        if constexpr (NB == 2)
            asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %1, %9 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %5, %11 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %2, %8 offset:%14\n\t"
                     "ds_read_b64_tr_b16 %3, %9 offset:%15\n\t"
                     "ds_read_b64_tr_b16 %6, %10 offset:%14\n\t"
                     "ds_read_b64_tr_b16 %7, %11 offset:%15\n\t"
                     "s_waitcnt lgkmcnt(0)"
                         : "=&v"(u[0][0].s[0]), "=&v"(u[0][0].s[1]), "=&v"(u[0][1].s[0]), "=&v"(u[0][1].s[1]), "=&v"(u[1][0].s[0]), "=&v"(u[1][0].s[1]), "=&v"(u[1][1].s[0]), "=&v"(u[1][1].s[1])
                         : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(0), "n"(DOWN), "n"(STEP), "n"(STEP + DOWN));
        if constexpr (NB == 3)
            asm volatile("ds_read_b64_tr_b16 %0, %12 offset:%18\n\t"
                     "ds_read_b64_tr_b16 %1, %13 offset:%19\n\t"
                     "ds_read_b64_tr_b16 %4, %14 offset:%18\n\t"
                     "ds_read_b64_tr_b16 %5, %15 offset:%19\n\t"
                     "ds_read_b64_tr_b16 %8, %16 offset:%18\n\t"
                     "ds_read_b64_tr_b16 %9, %17 offset:%19\n\t"
                     "ds_read_b64_tr_b16 %2, %12 offset:%20\n\t"
                     "ds_read_b64_tr_b16 %3, %13 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %6, %14 offset:%20\n\t"
                     "ds_read_b64_tr_b16 %7, %15 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %10, %16 offset:%20\n\t"
                     "ds_read_b64_tr_b16 %11, %17 offset:%21\n\t"
                     "s_waitcnt lgkmcnt(0)"
                         : "=&v"(u[0][0].s[0]), "=&v"(u[0][0].s[1]), "=&v"(u[0][1].s[0]), "=&v"(u[0][1].s[1]), "=&v"(u[1][0].s[0]), "=&v"(u[1][0].s[1]), "=&v"(u[1][1].s[0]), "=&v"(u[1][1].s[1]), "=&v"(u[2][0].s[0]), "=&v"(u[2][0].s[1]), "=&v"(u[2][1].s[0]), "=&v"(u[2][1].s[1])
                         : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "n"(0), "n"(DOWN), "n"(STEP), "n"(STEP + DOWN));
        if constexpr (NB == 4)
            asm volatile("ds_read_b64_tr_b16 %0, %16 offset:%24\n\t"
                     "ds_read_b64_tr_b16 %1, %17 offset:%25\n\t"
                     "ds_read_b64_tr_b16 %4, %18 offset:%24\n\t"
                     "ds_read_b64_tr_b16 %5, %19 offset:%25\n\t"
                     "ds_read_b64_tr_b16 %8, %20 offset:%24\n\t"
                     "ds_read_b64_tr_b16 %9, %21 offset:%25\n\t"
                     "ds_read_b64_tr_b16 %12, %22 offset:%24\n\t"
                     "ds_read_b64_tr_b16 %13, %23 offset:%25\n\t"
                     "ds_read_b64_tr_b16 %2, %16 offset:%26\n\t"
                     "ds_read_b64_tr_b16 %3, %17 offset:%27\n\t"
                     "ds_read_b64_tr_b16 %6, %18 offset:%26\n\t"
                     "ds_read_b64_tr_b16 %7, %19 offset:%27\n\t"
                     "ds_read_b64_tr_b16 %10, %20 offset:%26\n\t"
                     "ds_read_b64_tr_b16 %11, %21 offset:%27\n\t"
                     "ds_read_b64_tr_b16 %14, %22 offset:%26\n\t"
                     "ds_read_b64_tr_b16 %15, %23 offset:%27\n\t"
                     "s_waitcnt lgkmcnt(0)"
                         : "=&v"(u[0][0].s[0]), "=&v"(u[0][0].s[1]), "=&v"(u[0][1].s[0]), "=&v"(u[0][1].s[1]), "=&v"(u[1][0].s[0]), "=&v"(u[1][0].s[1]), "=&v"(u[1][1].s[0]), "=&v"(u[1][1].s[1]), "=&v"(u[2][0].s[0]), "=&v"(u[2][0].s[1]), "=&v"(u[2][1].s[0]), "=&v"(u[2][1].s[1]), "=&v"(u[3][0].s[0]), "=&v"(u[3][0].s[1]), "=&v"(u[3][1].s[0]), "=&v"(u[3][1].s[1])
                         : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7]), "n"(0), "n"(DOWN), "n"(STEP), "n"(STEP + DOWN));
    }
#endif
    template <int PARTS>
    __device__ __forceinline__ void mma(const Weights<T, PARTS>& w, Acc<T, DP>& sums, int first = 0) const {
        auto& acc = sums.x;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int n = 0; n < PARTS; ++n)
#pragma unroll
                    for (int db = 0; db < NB; ++db) acc[first + db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u[db][k].v, w.p[n][k], acc[first + db], 0, 0, 0);
        } else if constexpr (Acc<T, DP>::N16) {
            const f32x16a& p = w.x;
            constexpr int NC = DP / 16;
            const int l = lane & 15, j = lane >> 4, first = (j & 1) + 4 * (j >> 1);
            const char* const base = tile + first * LC * 16 + 4 * (l & 3);
            float x[2][NC];
            auto fetch = [&](int i, float (&y)[NC]) {
                const int row = 8 * (i >> 1) + 2 * (i & 1), f = swz<T, LC>(first + row);
#pragma unroll
                for (int c = 0; c < NC; ++c) y[c] = *(const float*)(base + row * LC * 16 + ((((l >> 2) + 4 * c) ^ f) << 4));
            };
            fetch(0, x[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i < 7) fetch(i + 1, x[(i + 1) & 1]);
                float p0 = p[2 * i], p1 = p[2 * i + 1];
                swap16(p0, p1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    sums.y[c][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i & 1][c], p0, sums.y[c][0], 0, 0, 0);
                    sums.y[c][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i & 1][c], p1, sums.y[c][1], 0, 0, 0);
                }
            }
        } else {
            const f32x16a& p = w.x;
            constexpr int W = NB == 3 ? 1 : NB;            // floats of a read
            typedef float vec __attribute__((ext_vector_type(W == 1 ? 1 : W)));
            const int li = lane & 31, hi = lane >> 5;
            const char* base = tile + 4 * hi * LC * 16 + (W * 4 * li & 15);
            float x[2][4][NB];
            auto fetch = [&](int a, float (&y)[4][NB]) {   // rows 8 a + 4 hi + 0..3
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 8 * a + e, f = swz<T, LC>(row + 4 * hi);
                    if constexpr (W == 1) {
#pragma unroll
                        for (int db = 0; db < NB; ++db) y[e][db] = *(const float*)(base + row * LC * 16 + ((((li >> 2) + 8 * db) ^ f) << 4));
                    } else {
                        const vec v = *(const vec*)(base + row * LC * 16 + (((W * li >> 2) ^ f) << 4));
#pragma unroll
                        for (int db = 0; db < NB; ++db) y[e][db] = v[db];
                    }
                }
            };
            fetch(0, x[0]);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                if (a < 3) fetch(a + 1, x[(a + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int db = 0; db < NB; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[a & 1][e][db], p[4 * a + e], acc[db], 0, 0, 0);
            }
        }
    }
};
// zeros in the place of the tile's infinities and NaN, a wave's pieces
template <typename T, int DP, int STEP>
__device__ __forceinline__ void scrub(char* tile, int first, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef T vec __attribute__((ext_vector_type(Mat<T>::E)));
    asm volatile("" : "+v"(lane));                        // (no address of this stays in registers through the tiles of every call)
    for (int i = first; i < DmaTile<T, DP>::PIECES; i += STEP) {
        vec* const at = (vec*)(tile + i * 1024 + lane * 16);
        vec x = *at;
#pragma unroll
        for (int e = 0; e < Mat<T>::E; ++e) x[e] = fabsf((float)x[e]) < INFINITY ? x[e] : (T)0.f;
        *at = x;
    }
#endif
}
// the accumulators of a lane's row, four neighbouring columns at a time: f(column, values, block and register of each)
template <typename T, int DP, typename F>
__device__ __forceinline__ void each_four(int hi, F f) {
    constexpr int NB = Acc<T, DP>::NB;
    if constexpr (sizeof(T) == 4 && NB == 4) {
#pragma unroll
        for (int r = 0; r < 16; ++r) f(4 * (8 * (r >> 2) + 4 * hi + (r & 3)), [=](int e) { return e * 16 + r; });
    } else if constexpr (sizeof(T) == 4 && NB == 2 && !Acc<T, DP>::N16) {
#pragma unroll
        for (int r = 0; r < 16; r += 2) f(2 * (8 * (r >> 2) + 4 * hi + (r & 3)), [=](int e) { return (e & 1) * 16 + r + (e >> 1); });
    } else {
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q) f(32 * db + 8 * q + 4 * hi, [=](int e) { return db * 16 + 4 * q + e; });
    }
}
// all of this wave's requests have landed; every wave's, with more than one
template <int WAVES>
__device__ __forceinline__ void dma_wait() {
#if defined(__HIP_DEVICE_COMPILE__)
    // (the builtins, so that the compiler knows these loads to be done and puts no wait for all of them further on)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);                   // vmcnt(0) lgkmcnt(0)
    if constexpr (WAVES > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#endif
}

// ... all but the last N requests, where there were any behind them; every wave's
template <int N>
__device__ __forceinline__ void dma_wait_but(bool more) {
#if defined(__HIP_DEVICE_COMPILE__)
    static_assert(N < 16, "the low four bits of the count");
    asm volatile("" ::: "memory");
    if (more) __builtin_amdgcn_s_waitcnt(0x0F70 | N);     // vmcnt(N)
    else __builtin_amdgcn_s_waitcnt(0x0F70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#endif
}

// ---- what every kernel knows of the call
struct Attn {
    int B, Lq, Lk, Hq, Hk, G, D, block, qb, n, causal, nbuckets, maxd, nb, ng;
    int zero_rest, chunks, splits;                                 // forward: row chunks of a group, parts of its keys
    float scale, scale2;                                  // scale2 = scale * log2(e)
    const void *q, *k, *v, *dout;
    void* out;
    Strides sq, sk, sv, so, sdo;
    const int32_t *sel, *qlen, *klen, *bucket_of, *q_pos, *k_pos;
    const float* bias;
    float *lse, *lse_rest, *out32;
    void *dq, *dk, *dv;
    float* dbias;
    float *po, *pml;                                      // forward, splits > 1: partial results, their maxima and sums
    // backward
    float* delta;
    float* zeros;                                         // 256 bytes
    unsigned* member;                                     // [b, hk][32 groups][nb4 key blocks], a bit a group
    int words, nb4;
    int *chunk_start, *chunk_rows;                        // [b, hk][key block + 1], [b, hk][key block]
    int max_chunks;
    float* pkv;                                           // partial dk, dv
    double* pbias;
};
// the kernel's first argument, read once more from memory where this is called: nothing of it is held in registers until then
#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ const Attn& late_args() {
    auto p = (const __attribute__((address_space(4))) Attn*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Attn*)p;
}
#endif

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

// ... and the number of their tiles with a wanted key (the last block may end behind the limit)
__device__ __forceinline__ int live_tiles(const Attn& a, const int32_t* sel, int limit, int* list, int lane) {
    const int c = live_blocks(a, sel, limit, list, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return c == 0 ? 0 : (c - 1) * (a.block / KT) + (min(a.block, limit - list[c - 1] * a.block) + KT - 1) / KT;
}

// ln(sum of 2^score) of a row with maximum m and sum l (units of log 2), as two fp32 numbers: a row whose scores are around 50 would be
// off by 2^-19 of every weight in the backward pass if it came back as one
__device__ __forceinline__ void store_lse(const Attn& a, size_t at, float m, float l) {
    const double v = l == 0.f ? -INFINITY : ((double)m + log2((double)l)) * 0.6931471805599453094;
    const float h = (float)v;
    a.lse[at] = h;
    if (a.lse_rest) a.lse_rest[at] = l == 0.f ? 0.f : (float)(v - (double)h);
}
// minus that, in units of log 2 and in two parts again
struct Shift { float hi, lo; };
__device__ __forceinline__ Shift load_lse(float lse, float rest) {
    const double v = ((double)lse + (double)rest) * 1.4426950408889634074;
    const float h = (float)v;
    return {-h, (float)((double)h - v)};
}

// ---- scores of a tile: 32 keys of a lane's row, masked, with the bias
struct Bias {                                             // in LDS: the bucket of each clamped distance, the workgroup's heads
    const unsigned char* lut;
    const float* tbl;
};
// scores are kept in units of ln 2 (exp2 needs no product).  A bias below -1e30 -- a type's lowest value as much as -inf -- masks its
// keys: at that size a score's own digits are lost in it, and a row with nothing else has no weights to tell apart
__device__ __forceinline__ float bias_log2(float b) { return b < -1e30f ? -INFINITY : fminf(b * LOG2E, 3.402823466e38f) + (b - b); }
__host__ __device__ inline int bias_lut_bytes(int nbuckets, int maxd) { return nbuckets ? (2 * maxd + 1 + 15) / 16 * 16 : 0; }
// the table of buckets by the whole workgroup, a key head's biases by `n` threads
__device__ __forceinline__ Bias load_bias(const Attn& a, unsigned char* lut, float* tbl, int hk, int t, int n) {
    if (a.nbuckets) {
        for (int i = threadIdx.x; i < 2 * a.maxd + 1; i += blockDim.x) lut[i] = (unsigned char)min(max(a.bucket_of[i], 0), a.nbuckets - 1);
        for (int i = t; i < a.nbuckets * a.G; i += n) tbl[i] = bias_log2(a.bias[(size_t)(i / a.G) * a.Hq + hk * a.G + i % a.G]);
    }
    return Bias{lut, tbl};
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
// the bias of N of the 16 scores of a lane's row from the first-th on, position by position
template <int N>
__device__ __forceinline__ void tile_buckets(const Attn& a, const Bias& s, int key0, const int* kp, int qp, int hi, int (&d)[N], int first = 0) {
    if (kp) {
#pragma unroll
        for (int r = 0; r < N; ++r) d[r] = kp[tile_key(first + r, hi)];
    } else {
#pragma unroll
        for (int r = 0; r < N; ++r) d[r] = key0 + tile_key(first + r, hi);
    }
#pragma unroll
    for (int r = 0; r < N; ++r) d[r] = s.lut[clamp_dist(d[r] - qp, a.maxd)];
}
template <int N>
__device__ __forceinline__ void tile_bias(const Attn& a, const Bias& s, int key0, const int* kp, int qp, int gl, int hi, float (&x)[N], int first = 0) {
    int d[N];
    tile_buckets(a, s, key0, kp, qp, hi, d, first);
#pragma unroll
    for (int r = 0; r < N; ++r) x[r] = s.tbl[d[r] * a.G + gl];
}
inline size_t bias_lds(int nbuckets, int maxd, int G) { return (size_t)bias_lut_bytes(nbuckets, maxd) + ((size_t)nbuckets * G * 4 + 15) / 16 * 16; }

}  // namespace scipnp
