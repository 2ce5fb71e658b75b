// w8a8_stream.hip -- layers with 8-bit weights on few tokens: bound by reading the weights once.
//
// A workgroup has 16 MB rows and 16 NB channels over all of K.  Its wavefronts take 256 bytes of K in turn, whole lines of 8
// channels a load (and rows of X, from L2), straight to the MFMA operand's registers: no LDS, no barrier until the end, and as
// many loads in flight as registers hold.  The wavefronts' sums are added in LDS, in whole numbers, so in any order.
#include <type_traits>

#include "lds_dma.hpp"
#include "w8a8.hpp"

namespace lava {

template <int MB, int NB, int WAVES, bool GATED>
__global__ void __launch_bounds__(64 * WAVES) w8a8_stream_kernel(W8Args a, int tiles_n) {
    static_assert(!GATED || NB == 2, "a gated tile is 16 channels of the gate and their 16 factors");
    constexpr int DEPTH = 16 / (MB + NB) > 4 ? 4 : 16 / (MB + NB) < 2 ? 2 : 16 / (MB + NB);   // chunks in flight
    constexpr int CHUNK = 256;
    static_assert(WAVES >= 3, "three wavefronts fetch what the finish needs");
    __shared__ i32x4 part[WAVES][MB * NB][64];
    __shared__ float s_ws[32], s_bias[32], s_xs[16 * MB];
    __shared__ int s_yr[16 * MB];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tn = blockIdx.x % tiles_n;
    W8Tile tile;
    if (!w8_find(a, 16 * MB, blockIdx.x / tiles_n, tile)) return;
    const int half = a.n >> 1;
    const int r16 = lane & 15;
    const int col0 = tn * (GATED ? 16 : 16 * NB);

    // Rows, channels and bytes of K that are none get an offset outside the buffer and read zero.
    const bool gather = a.offsets != nullptr && !a.x_sorted;
    const int xfirst = gather ? 0 : tile.first, xrows = gather ? a.rows / a.top_k : tile.rows;
    const auto rx = w8_buffer(a.x + (int64_t)xfirst * a.ldx, (int64_t)(xrows - 1) * a.ldx + a.k);
    const int cols_in = min(GATED ? 16 : 16 * NB, a.n_out - col0);
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride + (int64_t)col0 * a.ldw;
    const int64_t wbytes = (int64_t)(cols_in - 1) * a.ldw + a.k;
    const auto rw = w8_buffer(wbase, wbytes), ru = w8_buffer(GATED ? wbase + (int64_t)half * a.ldw : wbase, wbytes);
    // What the finish needs, requested first: channel row l's scale (lanes 0 ..) and bias (32 ..), row l's scale, row l of Y.
    float held = 0.f;
    if (w == 0) {
        const int c = (lane & 31) < 16 * NB ? (GATED ? lane & 15 : lane & 31) : 0;
        const int64_t ch = (int64_t)tile.expert * a.n + col0 + min(c, cols_in - 1) + (GATED && (lane & 16) ? half : 0);
        const float* p = lane < 32 ? a.ws : a.bias;
        if (p) held = p[ch];
    } else if (w <= 2 && lane < tile.rows) {
        int xr, yr;
        w8_rows(a, tile, lane, xr, yr);
        held = w == 2 ? __int_as_float(yr) : xr < 0 ? 0.f : a.xs[xr];
    }
    uint32_t xoff[MB], woff[NB][2];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        int xr = -1, yr;
        if (16 * i + r16 < tile.rows) w8_rows(a, tile, 16 * i + r16, xr, yr);
        xoff[i] = xr < 0 ? OOB_OFS : (uint32_t)((int64_t)(xr - xfirst) * a.ldx + 32 * (lane >> 4));
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = (GATED ? 0 : 16 * j) + 8 * h + (lane & 7);
            woff[j][h] = c < cols_in ? (uint32_t)(c * a.ldw + 16 * (lane >> 3)) : OOB_OFS;
        }
    }
    i32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    // Two pieces of 128 bytes of K: of a block of channels, v[p][j][0] is the first 8 channels' whole lines, lane l channel l % 8,
    // bytes 16 (l / 8); v[p][j][1] the other 8's.
    struct Chunk {
        i32x4 x[2][MB][2], v[2][NB][2];
    };
    // Rows of a power-of-two length lie on the same memory channels byte for byte: each workgroup begins at another chunk.
    const int chunks = (a.k + CHUNK - 1) / CHUNK;
    const int turn = (tn + (tn >> 3)) % chunks;
    // the wavefront's chunk n; from `chunks` on none
    auto load = [&](Chunk& c, int n) __attribute__((always_inline)) {
        const int at = n >= chunks ? a.k : (n + turn < chunks ? n + turn : n + turn - chunks) * CHUNK;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int k = at + 128 * p;
            const bool in = k + 16 * (lane >> 3) < a.k;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) c.v[p][j][h] = w8_load<true>(GATED && j ? ru : rw, in ? woff[j][h] : OOB_OFS, k);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool xin = k + 32 * (lane >> 4) + 16 * h < a.k;
#pragma unroll
                for (int i = 0; i < MB; ++i) c.x[p][i][h] = w8_load<false>(rx, xin ? xoff[i] : OOB_OFS, k + 16 * h);
            }
        }
    };
    auto multiply = [&](Chunk& c) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                i32x4 v0, v1;
                w8_whole_lines(c.v[p][j][0], c.v[p][j][1], v0, v1);
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v0, c.x[p][i][0], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v1, c.x[p][i][1], acc[i][j], 0, 0, 0);
                }
            }
    };
    // No branch around a load: the compiler would wait for all that are in flight where it joins.
    Chunk ring[DEPTH];
    const int turns = (chunks + WAVES - 1) / WAVES;   // of every wavefront
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(ring[d], w + d * WAVES);
    int n = 0;
    for (; n + DEPTH < turns; n += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            multiply(ring[d]);
            __builtin_amdgcn_sched_barrier(0);
            load(ring[d], w + (n + d + DEPTH) * WAVES);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) multiply(ring[d]);
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) part[w][i * NB + j][lane] = acc[i][j];
    if (w == 0) (lane < 32 ? s_ws : s_bias)[lane & 31] = held;
    else if (w == 1 && lane < 16 * MB) s_xs[lane] = held;
    else if (w == 2 && lane < 16 * MB) s_yr[lane] = __float_as_int(held);
    __syncthreads();

    // Block b of the results (16 rows, 16 columns of Y) is finished by wavefront b % WAVES; a lane has row lane % 16, columns
    // 4 (lane / 16) and the next three.
    constexpr int OB = GATED ? MB : MB * NB;
    for (int b = w; b < OB; b += WAVES) {
        const int i = GATED ? b : b / NB, j = GATED ? 0 : b % NB;
        const int m = 16 * i + r16, c = 16 * j + 4 * (lane >> 4);
        const int yr = m < tile.rows ? s_yr[m] : -1;
        if (yr < 0 || c >= cols_in) continue;
        const float xs = s_xs[m];
        auto values = [&](int jj, float (&v)[4]) {
            const int at = GATED ? 16 * jj + 4 * (lane >> 4) : c;
            i32x4 s = part[0][i * NB + jj][lane];
#pragma unroll
            for (int z = 1; z < WAVES; ++z) s += part[z][i * NB + jj][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = w8_value(s[r], xs, s_ws[at + r], s_bias[at + r]);
        };
        float v[4];
        values(j, v);
        w8_act4(a.act, v);
        if constexpr (GATED) {
            float u[4];
            values(1, u);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] *= u[r];
        }
        w8_store(a, (int64_t)yr * a.ldy + col0 + c, cols_in - c, v);
    }
}

bool w8_stream_fits(const W8Args& a) { return a.k > 0 && w8_chunks_fit(a) && w8_spans_fit(a, 64, 32); }

int launch_w8_stream(const W8Args& a, int rows, hipStream_t s) {
    const int MB = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    // 16 channels a workgroup of a small layer, so that all CUs have one; of a larger one 32, which reads X half as often
    const bool wide = !a.gated && (int64_t)a.n_out * a.experts > 8192;
    const int cols = wide ? 32 : 16;
    const int64_t tm = w8_row_tiles(a, 16 * MB), tn = ((int64_t)a.n_out + cols - 1) / cols;
    LAVA_REQUIRE(tm * tn <= 0xffffff, LAVA_HIP_ERR_UNSUPPORTED, "w8a8_stream_kernel would need %lld workgroups", (long long)(tm * tn));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(256), 0, s, a, (int)tn); };
    auto by_rows = [&](auto mtag) {
        constexpr int M = decltype(mtag)::value;
        if (a.gated) go(w8a8_stream_kernel<M, 2, 4, true>);
        else if (wide) go(w8a8_stream_kernel<M, 2, 4, false>);
        else go(w8a8_stream_kernel<M, 1, 4, false>);
    };
    if (MB == 1) by_rows(std::integral_constant<int, 1>{});
    else if (MB == 2) by_rows(std::integral_constant<int, 2>{});
    else by_rows(std::integral_constant<int, 4>{});
    LAVA_LAUNCH_CHECK("w8a8_stream_kernel");
    return LAVA_HIP_OK;
}

}  // namespace lava
