// w8a8.hip -- layers with 8-bit weights and tokens: argument checks, kernel choice, and the generic kernel.
#include <hip/hip_runtime.h>

#include "w8a8.hpp"

namespace lava {

namespace {
constexpr int WG_TILE = 64, WG_K = 64, WG_PITCH = WG_K + 16;   // padded: the 16 rows of a fragment on distinct banks

// 16 bytes of a row from byte k on, zeros from `end` on; any alignment.
__device__ __forceinline__ uint4 load16(const int8_t* row, int k, int end) {
    uint4 v = {0, 0, 0, 0};
    if (k + 16 <= end) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < end) {
        uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (k + i < end) word[i >> 2] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i & 3));
        v = uint4{word[0], word[1], word[2], word[3]};
    }
    return v;
}
}  // namespace

// Any layout: 64 rows x 64 channels a workgroup of 4 wavefronts, K 64 at a time through registers and LDS, one 16x16x64
// MFMA a wavefront and block of 16 channels.  Of a gated layer's 64 channels each second block of 16 is the other half's, so that a
// lane holds a column's gate and its factor.  Bound by the latency of one chunk of K in flight: 333 rows x 14336 x 4096 72 us (540 TOP/s),
// with rows of 4095 bytes 100; one row x 4096 x 4096 28 us.
__global__ void __launch_bounds__(256) w8a8_generic_kernel(W8Args a, int tiles_n) {
    __shared__ __attribute__((aligned(16))) int8_t sx[WG_TILE * WG_PITCH], sw[WG_TILE * WG_PITCH];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int tn = blockIdx.x % tiles_n;
    W8Tile tile;
    if (!w8_find(a, WG_TILE, blockIdx.x / tiles_n, tile)) return;
    const int half = a.n >> 1;
    // channel of row r of the weights' tile, and the column of Y it goes to
    auto column = [&](int r) { return a.gated ? tn * 32 + (r >> 5) * 16 + (r & 15) : tn * WG_TILE + r; };
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride;

    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;   // what this thread stages: a row, 16 bytes of it
    int xr = -1, yr;
    if (r < tile.rows) w8_rows(a, tile, r, xr, yr);
    const int8_t* xrow = a.x + (int64_t)(xr < 0 ? 0 : xr) * a.ldx;
    const int col = column(r);
    const bool wok = col < a.n_out;
    const int8_t* wrow = wbase + (int64_t)(!wok ? 0 : a.gated && (r & 16) ? half + col : col) * a.ldw;

    i32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = i32x4{0, 0, 0, 0};
    for (int k0 = 0; k0 < a.k; k0 += WG_K) {
        const uint4 vx = load16(xrow, k0 + c, xr < 0 ? 0 : a.k), vw = load16(wrow, k0 + c, wok ? a.k : 0);
        __syncthreads();
        *reinterpret_cast<uint4*>(sx + r * WG_PITCH + c) = vx;
        *reinterpret_cast<uint4*>(sw + r * WG_PITCH + c) = vw;
        __syncthreads();
        const int at = (lane & 15) * WG_PITCH + (lane >> 4) * 16;
        const uint4 fx = *reinterpret_cast<const uint4*>(sx + 16 * w * WG_PITCH + at);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc[j] = Mfma16<int8_t>::run(*reinterpret_cast<const uint4*>(sw + 16 * j * WG_PITCH + at), fx, acc[j]);
    }

    // acc[j][i]: row 16 w + lane % 16, channel row 16 j + 4 (lane / 16) + i
    const int m = 16 * w + (lane & 15);
    if (m >= tile.rows) return;
    w8_rows(a, tile, m, xr, yr);
    if (yr < 0) return;
    const float xs = a.xs[xr];
    const int64_t sbase = (int64_t)tile.expert * a.n;
    auto value = [&](int j, int i) {
        const int row = 16 * j + 4 * (lane >> 4) + i, cc = column(row);
        const int64_t ch = sbase + (a.gated && (row & 16) ? half + cc : cc);
        return cc < a.n_out ? w8_value(acc[j][i], xs, a.ws[ch], a.bias ? a.bias[ch] : 0.f) : 0.f;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (a.gated && (j & 1)) continue;
        const int cc = column(16 * j + 4 * (lane >> 4));
        if (cc >= a.n_out) continue;
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = w8_act(a.act, value(j, i));
            if (a.gated) v[i] *= value(j | 1, i);
        }
        w8_store(a, (int64_t)yr * a.ldy + cc, a.n_out - cc, v);
    }
}

int launch_w8_generic(const W8Args& a, hipStream_t s) {
    const int64_t tiles_n = ((int64_t)a.n_out + (a.gated ? 31 : 63)) / (a.gated ? 32 : 64);
    const int64_t blocks = w8_row_tiles(a, WG_TILE) * tiles_n;
    LAVA_REQUIRE(blocks <= 0xffffff, LAVA_HIP_ERR_UNSUPPORTED, "w8a8_generic_kernel would need %lld workgroups",
                 (long long)blocks);
    hipLaunchKernelGGL(w8a8_generic_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a, (int)tiles_n);
    LAVA_LAUNCH_CHECK("w8a8_generic_kernel");
    return LAVA_HIP_OK;
}

namespace {

// The layer's own checks, and those of X and Y; fills what does not depend on the rows.
int check_layer(const char* name, const lava_hip_w8_layer* l, const int8_t* X, const float* x_scale, int64_t ldx,
                int y_dtype, void* Y, int64_t ldy, bool nothing, W8Args& a) {
    LAVA_ARG(l != nullptr, "%s: null layer", name);
    LAVA_ARG(l->n >= 0 && l->k >= 0, "%s: negative extent (n=%lld k=%lld)", name, (long long)l->n, (long long)l->k);
    LAVA_REQUIRE(l->n <= W8_MOST, LAVA_HIP_ERR_UNSUPPORTED, "%s: n = %lld is too large", name, (long long)l->n);
    LAVA_REQUIRE(l->k <= 131071, LAVA_HIP_ERR_UNSUPPORTED, "%s: the sums of k = %lld products of bytes may leave 32 bits (at most 131071)",
                 name, (long long)l->k);
    LAVA_ARG(l->act >= LAVA_HIP_ACT_NONE && l->act <= LAVA_HIP_ACT_SILU, "%s: unknown activation %d", name, l->act);
    LAVA_ARG(!l->gated || l->n % 2 == 0, "%s: a gated layer of an odd number of channels (%lld)", name, (long long)l->n);
    LAVA_ARG(y_dtype == LAVA_HIP_F32 || y_dtype == LAVA_HIP_F16 || y_dtype == LAVA_HIP_BF16,
             "%s: Y's dtype %d is not f32, f16 or bf16", name, y_dtype);
    const int64_t n_out = l->gated ? l->n / 2 : l->n;
    a.n = (int)l->n;
    a.n_out = (int)n_out;
    if (nothing || n_out == 0) return LAVA_HIP_OK;
    LAVA_ARG(l->scale != nullptr && x_scale != nullptr && Y != nullptr, "%s: null scale or Y", name);
    LAVA_ARG(l->k == 0 || (l->w != nullptr && X != nullptr), "%s: null X or w", name);
    LAVA_ARG(l->ldw >= l->k, "%s: ldw = %lld is smaller than k", name, (long long)l->ldw);
    LAVA_ARG(ldx >= l->k, "%s: ldx = %lld is smaller than k", name, (long long)ldx);
    LAVA_ARG(ldy >= n_out, "%s: ldy = %lld is smaller than Y's %lld columns", name, (long long)ldy, (long long)n_out);
    const size_t ysz = y_dtype == LAVA_HIP_F32 ? 4 : 2;
    LAVA_ARG(aligned(l->scale, 4) && aligned(l->bias, 4) && aligned(x_scale, 4) && aligned(Y, ysz),
             "%s: operands not aligned to their element size", name);
    a.x = X;
    a.xs = x_scale;
    a.w = l->w;
    a.ws = l->scale;
    a.bias = l->bias;
    a.y = Y;
    a.ldx = ldx;
    a.ldw = l->ldw;
    a.expert_stride = l->expert_stride;
    a.ldy = ldy;
    a.k = (int)l->k;
    a.act = l->act;
    a.gated = l->gated != 0;
    a.y_dtype = y_dtype;
    return LAVA_HIP_OK;
}

int run(const W8Args& a, void* stream) {
    const int rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    hipStream_t s = as_stream(stream);
    const int pin = kernel_override(LAVA_HIP_FAMILY_W8A8);
    if (pin == 1) return launch_w8_generic(a, s);
    if (w8_stream_fits(a) && (pin == 2 || (pin == 0 && w8_stream_preferred(a)))) return launch_w8_stream(a, s);
    const int tile = pin >= 3 && w8_tile_fits(a, pin - 3) ? pin - 3 : w8_tile_choice(a);
    return tile >= 0 ? launch_w8_tile(a, tile, s) : launch_w8_generic(a, s);
}

}  // namespace

}  // namespace lava

using namespace lava;

extern "C" {

int lava_hip_gemm_w8a8(const lava_hip_w8_layer* layer, const int8_t* X, const float* x_scale, int64_t tokens, int64_t ldx,
                       int y_dtype, void* Y, int64_t ldy, void* stream) {
    W8Args a = {};
    LAVA_ARG(tokens >= 0, "gemm_w8a8: negative tokens (%lld)", (long long)tokens);
    LAVA_REQUIRE(tokens <= W8_MOST, LAVA_HIP_ERR_UNSUPPORTED, "gemm_w8a8: %lld tokens are too many", (long long)tokens);
    const int rc = check_layer("gemm_w8a8", layer, X, x_scale, ldx, y_dtype, Y, ldy, tokens == 0, a);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG(layer->experts == 1, "gemm_w8a8: a layer of %d experts", layer->experts);
    if (tokens == 0 || a.n_out == 0) return LAVA_HIP_OK;
    a.rows = (int)tokens;
    a.top_k = a.experts = 1;
    return run(a, stream);
}

int lava_hip_experts_w8a8(const lava_hip_moe_plan* plan, const lava_hip_w8_layer* layer, const int8_t* X,
                          const float* x_scale, int64_t ldx, int y_dtype, void* Y, int64_t ldy, uint32_t flags,
                          void* stream) {
    W8Args a = {};
    const int rp = check_plan("experts_w8a8", plan, false);
    if (rp != LAVA_HIP_OK) return rp;
    LAVA_ARG(flags <= 3u, "experts_w8a8: flags %u has bits beyond X_SORTED and Y_SORTED", flags);
    const int64_t rows = plan->tokens * plan->top_k;
    const int rc = check_layer("experts_w8a8", layer, X, x_scale, ldx, y_dtype, Y, ldy, rows == 0, a);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG(layer->experts == plan->experts, "experts_w8a8: a layer of %d experts, a plan of %d", layer->experts,
             plan->experts);
    if (rows == 0 || a.n_out == 0) return LAVA_HIP_OK;
    LAVA_ARG(layer->experts == 1 || layer->expert_stride / layer->n >= layer->ldw,
             "experts_w8a8: expert_stride = %lld is smaller than n * ldw", (long long)layer->expert_stride);
    a.offsets = plan->offsets;
    a.order = plan->order;
    a.rows = (int)rows;
    a.top_k = plan->top_k;
    a.experts = plan->experts;
    a.x_sorted = (flags & LAVA_HIP_X_SORTED) != 0;
    a.y_sorted = (flags & LAVA_HIP_Y_SORTED) != 0;
    return run(a, stream);
}

}  // extern "C"
