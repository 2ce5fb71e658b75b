// quantize.hip -- rows of values to 8 bits with a scale a row.
//
// q is the integer nearest to the real number 127 x / max |x|.  In 32 bits t = x * (127 / max) is off by at most 2 half
// ulps, 127 * 2 * 2^-24 < 1.6e-5, so t rounds to the right integer unless it lies that near to a border between two; there
// 254 |x| against (2 n + 1) max, products that are exact in 64 bits, decides (ties to even).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_common.hpp"
#include "lava_hip_internal.hpp"

namespace lava {

namespace {

// |x| as bits that compare like |x|; infinities and NaN are at least 0x7f800000
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct Scale {
    float top;     // max |x|
    float up, r;   // t = (x * up) * r: up lifts rows so small that 127 / top overflows
    bool ok;       // finite
};

__device__ __forceinline__ Scale make_scale(uint32_t bits) {
    Scale s;
    s.ok = bits < 0x7f800000u;
    s.top = __uint_as_float(bits);
    s.up = s.top < 0x1p-100f ? 0x1p100f : 1.f;
    s.r = s.top > 0.f && s.ok ? 127.f / (s.top * s.up) : 0.f;
    return s;
}

constexpr float NEAR_BORDER = 0.49998f;

// The integer for an x whose t lies near a border.
__device__ __forceinline__ float by_border(float x, float t, float top) {
    const float n = floorf(fabsf(t));
    const double a = 254.0 * (double)fabsf(x), border = (2.0 * (double)n + 1.0) * (double)top;
    return copysignf(a > border || (a == border && ((int)n & 1)) ? n + 1.f : n, x);
}

__device__ __forceinline__ float nearest(float x, const Scale& s) {
    const float t = (x * s.up) * s.r, q = rintf(t);
    if (__builtin_expect(fabsf(t - q) > NEAR_BORDER, 0)) return by_border(x, t, s.top);
    return q;
}

}  // namespace

// Rows held in registers, THREADS lanes a row, CH chunks of 8 values a lane, of any alignment.  Bound by the bytes: 40961 rows of
// 1408 bf16 30.8 us, 5.6 TB/s; a single row by its launch and a chain of reads, 2 to 3 us.
template <typename T, int THREADS, int CH>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
    quantize_rows_kernel(const T* __restrict__ X, int8_t* __restrict__ Q, float* __restrict__ scale, int k, int tokens, int64_t ldx,
                         int64_t ldq) {
    constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, WAVES = THREADS / 64;
    __shared__ uint32_t part[WAVES];
    typedef T T8 __attribute__((ext_vector_type(8)));
    typedef T8 T8u __attribute__((aligned(sizeof(T))));
    typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(1)));
    const int64_t row = (int64_t)blockIdx.x * (BLOCK / THREADS) + threadIdx.x / THREADS;
    if (row >= tokens) return;   // whole wavefronts: THREADS is a multiple of 64
    const int t = threadIdx.x % THREADS;
    const T* x = X + row * ldx;
    int8_t* q = Q + row * ldq;
    T8 v[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = 8 * (c * THREADS + t);
        if (at + 8 <= k) {
            v[c] = __builtin_nontemporal_load(reinterpret_cast<const T8u*>(x + at));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = at + i < k ? x[at + i] : (T)0.f;
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, mag((float)v[c][i]));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = max(top, part[i]);
    }
    const Scale s = make_scale(top);
    if (t == 0) scale[row] = s.ok ? s.top / 127.f : __builtin_nanf("");
    const bool plain = s.up == 1.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = 8 * (c * THREADS + t);
        if (at >= k) break;
        // t + 1.5 * 2^23 has the integer nearest to t in its low bits
        float y[8], off = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = (float)v[c][i] * s.r;
            y[i] = z + 12582912.f;
            off = fmaxf(off, fabsf(z - (y[i] - 12582912.f)));
        }
        if (__builtin_expect(!plain || !s.ok, 0)) {
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const float n = s.ok ? nearest((float)v[c][i], s) : 0.f;
                if (at + i < k) q[at + i] = (int8_t)(int)n;
            }
            continue;
        }
        if (__builtin_expect(off > NEAR_BORDER, 0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = (float)v[c][i] * s.r;
                if (fabsf(z - (y[i] - 12582912.f)) > NEAR_BORDER) y[i] = 12582912.f + by_border((float)v[c][i], z, s.top);
            }
        }
        uint32_t word[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[4 * h + 1]), __float_as_uint(y[4 * h]), 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[4 * h + 3]), __float_as_uint(y[4 * h + 2]), 0x0c0c0400u);
            word[h] = lo | hi << 16;
        }
        if (at + 8 <= k) {
            *reinterpret_cast<u32x2u*>(q + at) = u32x2u{word[0], word[1]};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + i < k) q[at + i] = (int8_t)(word[i >> 2] >> 8 * (i & 3));
        }
    }
}

// A workgroup a row, of any length; the row is read twice.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ X, int8_t* __restrict__ Q,
                                                       float* __restrict__ scale, int64_t k, int64_t ldx, int64_t ldq) {
    __shared__ uint32_t part[4];
    const T* x = X + blockIdx.x * ldx;
    int8_t* q = Q + blockIdx.x * ldq;
    uint32_t top = 0;
    for (int64_t j = threadIdx.x; j < k; j += 256) top = max(top, mag((float)x[j]));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
    const Scale s = make_scale(top);
    if (threadIdx.x == 0) scale[blockIdx.x] = s.ok ? s.top / 127.f : __builtin_nanf("");
    for (int64_t j = threadIdx.x; j < k; j += 256) q[j] = s.ok ? (int8_t)(int)nearest((float)x[j], s) : (int8_t)0;
}

template <typename T>
static int launch_quantize(const void* X, int8_t* Q, float* scale, int64_t k, int64_t tokens, int64_t ldx, int64_t ldq,
                           hipStream_t s) {
    const T* x = static_cast<const T*>(X);
    if (k == 0 || k > 65536) {
        hipLaunchKernelGGL(quantize_kernel<T>, dim3((unsigned)tokens), dim3(256), 0, s, x, Q, scale, k, ldx, ldq);
        LAVA_LAUNCH_CHECK("quantize_kernel");
        return LAVA_HIP_OK;
    }
    auto go = [&](auto kernel, int threads) {
        const int per = threads < 256 ? 256 / threads : 1;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((tokens + per - 1) / per)), dim3(threads < 256 ? 256 : threads), 0, s, x, Q, scale,
                           (int)k, (int)tokens, ldx, ldq);
    };
    // A wavefront a row where a lane has few values or there are rows for all CUs many times over, a workgroup of 256 for longer
    // rows, of 1024 for few long ones.  us with 64 / 256 / 1024 lanes a row of bf16: 40961 x 1408 30.8 / 48.9 / 161, 16384 x 2048
    // 20.8 / 23.3 / 66, 8192 x 4096 24.9 / 20.0 / 38.6, 1024 x 2048 6.7 / 4.5 / 6.2, 8192 x 8192 - / 34.8 / 47.6, 1024 x 14336 - /
    // 16.8 / 13.3, 1 x 14336 - / 5.9 / 4.0.
    const int threads = k <= 1024 || (k <= 2048 && tokens >= 8192) ? 64 : k > 16384 || (k > 4096 && tokens <= 1024) ? 1024 : 256;
    const int ch = (int)((k + 8 * threads - 1) / (8 * threads));
    auto by_ch = [&](auto ttag) {
        constexpr int N = decltype(ttag)::value;
        if (ch <= 1) go(quantize_rows_kernel<T, N, 1>, N);
        else if (ch <= 2) go(quantize_rows_kernel<T, N, 2>, N);
        else if (ch <= 3) go(quantize_rows_kernel<T, N, 3>, N);
        else if (N == 64 || ch <= 4) go(quantize_rows_kernel<T, N, 4>, N);   // 64 lanes have at most 2048 values
        else if constexpr (N > 64) ch <= 6 ? go(quantize_rows_kernel<T, N, 6>, N) : go(quantize_rows_kernel<T, N, 8>, N);
    };
    if (threads == 64) by_ch(std::integral_constant<int, 64>{});
    else if (threads == 256) by_ch(std::integral_constant<int, 256>{});
    else by_ch(std::integral_constant<int, 1024>{});
    LAVA_LAUNCH_CHECK("quantize_rows_kernel");
    return LAVA_HIP_OK;
}

}  // namespace lava

using namespace lava;

extern "C" int lava_hip_quantize_i8(int x_dtype, const void* X, int8_t* Q, float* scale, int64_t k, int64_t tokens,
                                    int64_t ldx, int64_t ldq, void* stream) {
    LAVA_ARG(x_dtype == LAVA_HIP_F32 || x_dtype == LAVA_HIP_F16 || x_dtype == LAVA_HIP_BF16,
             "quantize_i8: dtype %d is not f32, f16 or bf16", x_dtype);
    LAVA_ARG(k >= 0 && tokens >= 0, "quantize_i8: negative extent (k=%lld tokens=%lld)", (long long)k, (long long)tokens);
    if (tokens == 0) return LAVA_HIP_OK;
    LAVA_ARG(scale != nullptr && (k == 0 || (X != nullptr && Q != nullptr)), "quantize_i8: null pointer");
    LAVA_ARG(ldx >= k, "quantize_i8: ldx = %lld is smaller than k", (long long)ldx);
    LAVA_ARG(ldq >= k, "quantize_i8: ldq = %lld is smaller than k", (long long)ldq);
    LAVA_ARG(aligned(X, x_dtype == LAVA_HIP_F32 ? 4 : 2) && aligned(scale, 4),
             "quantize_i8: operands not aligned to their element size");
    LAVA_REQUIRE(tokens <= 0x7fffffff, LAVA_HIP_ERR_UNSUPPORTED, "quantize_i8: %lld tokens are too many", (long long)tokens);
    const int rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    hipStream_t s = as_stream(stream);
    if (x_dtype == LAVA_HIP_F32) return launch_quantize<float>(X, Q, scale, k, tokens, ldx, ldq, s);
    if (x_dtype == LAVA_HIP_F16) return launch_quantize<f16>(X, Q, scale, k, tokens, ldx, ldq, s);
    return launch_quantize<bf16>(X, Q, scale, k, tokens, ldx, ldq, s);
}
