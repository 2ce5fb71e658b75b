// w8a8.hip -- layers with 8-bit weights and tokens: argument checks, kernel choice, and the generic kernel.
#include <hip/hip_runtime.h>

#include "w8a8.hpp"

namespace lava {

namespace {
// 16 bytes of a row from byte at on, any alignment.
__device__ __forceinline__ uint4 load16(const int8_t* row, int at) {
    uint4 v;
    __builtin_memcpy(&v, row + at, 16);
    return v;
}
// The same, zeros from byte k on.
__device__ __forceinline__ uint4 load16(const int8_t* row, int at, int k) {
    if (at + 16 <= k) return load16(row, at);
    if (at >= k) return uint4{0, 0, 0, 0};
    unsigned __int128 v = 0;
    if (k >= 16) {   // the row's last 16 bytes, the first of them cut off
        __builtin_memcpy(&v, row + k - 16, 16);
        v >>= 8 * (at + 16 - k);
    } else {
        for (int i = k - 1; i >= at; --i) v = v << 8 | (uint8_t)row[i];
    }
    return __builtin_bit_cast(uint4, v);
}
}  // namespace

// Any layout: TILE rows x TILE channels a workgroup of 2 x 2 wavefronts, K bytes of K at a time through registers, which hold the next
// ones during the MFMAs, and LDS.  Of a gated layer's channels each second block of 16 is the other half's, so that a lane holds a
// column's gate and its factor.  Bound by the latency of one chunk of K in flight a workgroup and by rows that begin inside a
// 16-byte word.  us with K = 4095 / the other kernels with 4096: 4096 x 4096 149 (922 TOP/s) / 60, 333 x 14336 70 / 31, 16 x 14336 22.4 /
// 11.6, 1 x 4096 19.9 / 6.0.
template <int TILE, int K>
__global__ void __launch_bounds__(256) w8a8_generic_kernel(W8Args a, int tiles_n) {
    constexpr int PITCH = K + 16, F = TILE / 32;   // padded: the 16 rows of a fragment on distinct banks; fragments a wavefront
    __shared__ __attribute__((aligned(16))) int8_t sx[TILE * PITCH], sw[TILE * PITCH];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w >> 1, wn = w & 1;
    const int tn = blockIdx.x % tiles_n;
    W8Tile tile;
    if (!w8_find(a, TILE, blockIdx.x / tiles_n, tile)) return;
    const int half = a.n >> 1;
    // channel of row r of the weights' tile, and the column of Y it goes to
    auto column = [&](int r) { return a.gated ? tn * (TILE / 2) + (r >> 5) * 16 + (r & 15) : tn * TILE + r; };
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride;

    // What this thread stages: 16 bytes of 4 rows of each; rows that are none are the first one, and not stored.
    constexpr int ROWS = TILE * K / 16 / 256;
    const int first = threadIdx.x / (K / 16), c = threadIdx.x % (K / 16) * 16;
    const int8_t *xrow[ROWS], *wrow[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = first + i * (TILE / ROWS), col = column(r);
        int xr = -1, yr;
        if (r < tile.rows) w8_rows(a, tile, r, xr, yr);
        xrow[i] = a.x + (int64_t)(xr < 0 ? 0 : xr) * a.ldx;
        wrow[i] = wbase + (int64_t)(col >= a.n_out ? 0 : a.gated && (r & 16) ? half + col : col) * a.ldw;
    }
    uint4 vx[ROWS], vw[ROWS];
    auto stage = [&]() __attribute__((always_inline)) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int at = (first + i * (TILE / ROWS)) * PITCH + c;
            *reinterpret_cast<uint4*>(sx + at) = vx[i];
            *reinterpret_cast<uint4*>(sw + at) = vw[i];
        }
        __syncthreads();
    };
    i32x4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < K / 64; ++u) {
            const int at = (lane & 15) * PITCH + u * 64 + (lane >> 4) * 16;
            uint4 fx[F], fw[F];
#pragma unroll
            for (int i = 0; i < F; ++i) {
                fx[i] = *reinterpret_cast<const uint4*>(sx + (TILE / 2 * wm + 16 * i) * PITCH + at);
                fw[i] = *reinterpret_cast<const uint4*>(sw + (TILE / 2 * wn + 16 * i) * PITCH + at);
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = Mfma16<int8_t>::run(fw[j], fx[i], acc[i][j]);
        }
    };
    const int whole = a.k / K;
    if (whole > 0) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            vx[i] = load16(xrow[i], c);
            vw[i] = load16(wrow[i], c);
        }
    }
    for (int n = 1; n <= whole; ++n) {
        stage();
        const int at = min(n, whole - 1) * K + c;   // no branch around the loads: the compiler would wait where it joins
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            vx[i] = load16(xrow[i], at);
            vw[i] = load16(wrow[i], at);
        }
        multiply();
    }
    if (whole * K < a.k) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            vx[i] = load16(xrow[i], whole * K + c, a.k);
            vw[i] = load16(wrow[i], whole * K + c, a.k);
        }
        stage();
        multiply();
    }

    // acc[i][j][r]: row TILE / 2 wm + 16 i + lane % 16, channel row TILE / 2 wn + 16 j + 4 (lane / 16) + r
    const int64_t sbase = (int64_t)tile.expert * a.n;
#pragma unroll
    for (int i = 0; i < F; ++i) {
        const int m = TILE / 2 * wm + 16 * i + (lane & 15);
        if (m >= tile.rows) continue;
        int xr, yr;
        w8_rows(a, tile, m, xr, yr);
        if (yr < 0) continue;
        const float xs = a.xs[xr];
        auto value = [&](int j, int r) {
            const int row = TILE / 2 * wn + 16 * j + 4 * (lane >> 4) + r, cc = column(row);
            const int64_t ch = sbase + (a.gated && (row & 16) ? half + cc : cc);
            return cc < a.n_out ? w8_value(acc[i][j][r], xs, a.ws[ch], a.bias ? a.bias[ch] : 0.f) : 0.f;
        };
#pragma unroll
        for (int j = 0; j < F; ++j) {
            if (a.gated && (j & 1)) continue;
            const int cc = column(TILE / 2 * wn + 16 * j + 4 * (lane >> 4));
            if (cc >= a.n_out) continue;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = w8_act(a.act, value(j, r));
                if (a.gated) v[r] *= value(j | 1, r);
            }
            w8_store(a, (int64_t)yr * a.ldy + cc, a.n_out - cc, v);
        }
    }
}

template <int TILE, int K>
static int launch_generic(const W8Args& a, hipStream_t s) {
    const int cols = a.gated ? TILE / 2 : TILE;
    const int64_t tiles_n = ((int64_t)a.n_out + cols - 1) / cols, blocks = w8_row_tiles(a, TILE) * tiles_n;
    LAVA_REQUIRE(w8_launch_fits(a, TILE, cols, 256), LAVA_HIP_ERR_UNSUPPORTED, "w8a8_generic_kernel would need %lld workgroups",
                 (long long)blocks);
    hipLaunchKernelGGL((w8a8_generic_kernel<TILE, K>), dim3((unsigned)blocks), dim3(256), 0, s, a, (int)tiles_n);
    LAVA_LAUNCH_CHECK("w8a8_generic_kernel");
    return LAVA_HIP_OK;
}

// The large tile where every CU has one.  us of 64 x 64 / 128 x 128: 1024 x 4096 x 4095, 256 large tiles, 61 / 68; 333 x 14336 x 4095, 336,
// 86 / 69; 2048 x 4096 x 1111 48 / 41; 200 x 14336 x 777, 224, 21 / 28.
int launch_w8_generic(const W8Args& a, hipStream_t s) {
    return w8_tile_count(a, 128, 128) > 256 ? launch_generic<128, 128>(a, s) : launch_generic<64, 256>(a, s);
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
    if (pin >= 3 && w8_tile_fits(a, pin - 3)) return launch_w8_tile(a, pin - 3, s);
    // a pinned tile that cannot take the call leaves it to the choice without a pin
    if (w8_stream_fits(a) && (pin == 2 || w8_stream_preferred(a))) return launch_w8_stream(a, s);
    const int tile = w8_tile_choice(a);
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
