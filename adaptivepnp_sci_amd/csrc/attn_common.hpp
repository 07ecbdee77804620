// Shared pieces of the block-attention kernels (head_norm.hip, block_select.hip, block_attn.hip, block_attn_bwd.hip).
#pragma once
#include "common.hpp"

namespace scipnp {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2a __attribute__((ext_vector_type(2)));
typedef float f32x4a __attribute__((ext_vector_type(4)));
typedef float f32x16a __attribute__((ext_vector_type(16)));
typedef short s16x4a __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

// ---- host-side argument checks
inline size_t attn_esize(int dtype) { return dtype == SCIPNP_BF16 ? 2 : 4; }
inline bool attn_strides_ok(const int64_t* st, int dtype) {
    for (int i = 0; i < 3; ++i)
        if (st[i] < 0 || (st[i] * (int64_t)attn_esize(dtype)) % 16 != 0) return false;
    return true;
}
#define SCIPNP_STRIDES(st, dtype) \
    do { if (!::scipnp::attn_strides_ok(st, dtype)) return ::scipnp::fail(SCIPNP_EALIGN, #st ": strides must be non-negative multiples of 16 bytes"); } while (0)
#define SCIPNP_BLOCK_SIZE(a, type)                                                                                              \
    do {                                                                                                                        \
        SCIPNP_REQUIRE(a, "null argument block");                                                                               \
        SCIPNP_REQUIRE((a)->struct_size == sizeof(type), #type ".struct_size is %zu, this library's block has %zu bytes",       \
                       (a)->struct_size, sizeof(type));                                                                         \
    } while (0)

struct Strides { long long b, t, h; };                    // elements
inline Strides strides_of(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

// Workgroups are dealt to the 8 XCDs in turn, each with an L2 of its own: logical work item of workgroup x such that an XCD
// takes a contiguous eighth of the items (the items of one sequence and key head, which read the same keys, follow each other).
// The grid is 8 * ceil(total / 8); items past the last are -1.
__device__ __forceinline__ long long xcd_item(unsigned x, long long total) {
    const long long per = (total + 7) >> 3;
    const long long i = (long long)(x & 7) * per + (x >> 3);
    return ((long long)(x >> 3) < per && i < total) ? i : -1;
}
// four neighbouring results, rounded to T
__device__ __forceinline__ void store_four(float* p, f32x4a v) { *(f32x4a*)p = v; }
__device__ __forceinline__ void store_four(__bf16* p, f32x4a v) { *(bf16x4*)p = bf16x4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]}; }
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = min(v, __shfl_xor(v, off, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = max(v, __shfl_xor(v, off, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
inline unsigned xcd_grid(long long total) { return (unsigned)(((total + 7) >> 3) << 3); }

}  // namespace scipnp
