// Frames <-> patch tokens of the non-local prior (adaptivepnp_sci_amd/nonlocal_prior.py).
//
// A frame is cut into 4 x 4 patches of three colours (48 values), a tile of 8 x 8 neighbouring patches is one block of 64 tokens; the
// tokens of a clip run over frames, tile rows, tile columns, the tile's patches.  `shifts` copies of every clip are cut with grids
// moved by half a patch, (0,0) (2,2) (0,2) (2,0), and averaged on the way back, so no patch border is a border in all of them.
// Token: 48 values as c * 16 + row * 4 + column, one constant, zeros to 56: with the constant in the vector, its direction -- all
// that is left after the norm -- still tells dark from bright.
//
// Both are plain copies, bound by HBM (12 bytes a pixel and 224 a token): one float4 a thread, neighbours write neighbours.
#include "common.hpp"

namespace scipnp {

constexpr int NL_P = 4, NL_TILE = 32, NL_D = 56, NL_VEC = NL_D / 4;
struct NlGrid { int units, T, shifts, H, W, ty, tx; };
__device__ __forceinline__ int nl_off_y(int s) { return s == 1 || s == 3 ? 2 : 0; }
__device__ __forceinline__ int nl_off_x(int s) { return s == 1 || s == 2 ? 2 : 0; }

// one thread: four values of a token
__global__ void __launch_bounds__(256) patch_tokens_kernel(const float* __restrict__ frames, float* __restrict__ tokens, NlGrid g, float constant, float scale,
                                                           int replicate, size_t total) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int e = (int)(i % NL_VEC);
        size_t r = i / NL_VEC;
        float v[4] = {e == 12 ? constant : 0.f, 0.f, 0.f, 0.f};
        if (e < 12) {
            const int patch = (int)(r % 64);
            r /= 64;
            const int tx = (int)(r % g.tx);
            r /= g.tx;
            const int ty = (int)(r % g.ty);
            r /= g.ty;
            const int t = (int)(r % g.T), seq = (int)(r / g.T), u = seq / g.shifts, s = seq % g.shifts;
            const int c = e >> 2, y = ty * NL_TILE + (patch >> 3) * NL_P + (e & 3) - nl_off_y(s), x0 = tx * NL_TILE + (patch & 7) * NL_P - nl_off_x(s);
            const float* const plane = frames + (((size_t)t * g.units + u) * 3 + c) * g.H * g.W;
            const int yc = min(max(y, 0), g.H - 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int x = x0 + j, xc = min(max(x, 0), g.W - 1);
                if (replicate || (y == yc && x == xc)) v[j] = plane[(size_t)yc * g.W + xc] * scale;
            }
        }
        ((float4*)tokens)[i] = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// one thread: a pixel and colour, the mean over the shifts
__global__ void __launch_bounds__(256) patch_frames_kernel(const float* __restrict__ tokens, float* __restrict__ frames, NlGrid g, size_t total) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int x = (int)(i % g.W);
        size_t r = i / g.W;
        const int y = (int)(r % g.H);
        r /= g.H;
        const int c = (int)(r % 3);
        r /= 3;
        const int u = (int)(r % g.units), t = (int)(r / g.units);
        float sum = 0.f;
        for (int s = 0; s < g.shifts; ++s) {
            const int yy = y + nl_off_y(s), xx = x + nl_off_x(s);
            const size_t tile = (((size_t)(u * g.shifts + s) * g.T + t) * g.ty + yy / NL_TILE) * g.tx + xx / NL_TILE;
            const int patch = (yy % NL_TILE / NL_P) * 8 + xx % NL_TILE / NL_P;
            sum += tokens[(tile * 64 + patch) * NL_D + c * 16 + (yy % NL_P) * 4 + xx % NL_P];
        }
        frames[i] = sum / (float)g.shifts;
    }
}

static bool nl_grid(NlGrid& g, int B, int H, int W, int units, int shifts) {
    if (B <= 0 || H <= 0 || W <= 0 || units <= 0 || B % units || (shifts != 1 && shifts != 2 && shifts != 4) || H > (1 << 20) || W > (1 << 20)) return false;
    const int more = shifts > 1 ? 2 : 0;
    g = {units, B / units, shifts, H, W, (H + more + NL_TILE - 1) / NL_TILE, (W + more + NL_TILE - 1) / NL_TILE};
    return true;
}
static unsigned nl_blocks(size_t total) {
    const size_t b = (total + 255) / 256;
    return (unsigned)(b < 65536 ? b : 65536);
}

}  // namespace scipnp

using namespace scipnp;

extern "C" {

int scipnp_patch_tokens(const float* frames, float* tokens, int B, int H, int W, int units, int shifts, float constant, float scale, int replicate,
                        scipnp_stream_t s) {
    NlGrid g;
    SCIPNP_REQUIRE(frames && tokens, "null pointer");
    SCIPNP_REQUIRE(nl_grid(g, B, H, W, units, shifts), "bad shape: B frames of H x W in `units` clips, shifts 1, 2 or 4");
    SCIPNP_ALIGNED(tokens);
    const size_t total = (size_t)units * shifts * g.T * g.ty * g.tx * 64 * NL_VEC;
    patch_tokens_kernel<<<nl_blocks(total), 256, 0, (hipStream_t)s>>>(frames, tokens, g, constant, scale, replicate, total);
    return launch_status("patch_tokens_kernel");
}

int scipnp_patch_frames(const float* tokens, float* frames, int B, int H, int W, int units, int shifts, scipnp_stream_t s) {
    NlGrid g;
    SCIPNP_REQUIRE(frames && tokens, "null pointer");
    SCIPNP_REQUIRE(nl_grid(g, B, H, W, units, shifts), "bad shape: B frames of H x W in `units` clips, shifts 1, 2 or 4");
    const size_t total = (size_t)B * 3 * H * W;
    patch_frames_kernel<<<nl_blocks(total), 256, 0, (hipStream_t)s>>>(tokens, frames, g, total);
    return launch_status("patch_frames_kernel");
}

}
