// w8a8_stream.hip -- layers with 8-bit weights on at most 16 rows and few channels: bound by reading the weights once, with
// every CU at it.
//
// A workgroup has 16 rows and 16 channels (of a gated layer a gate's and their factors) over all of K, so that 4096 channels are 256
// workgroups.  Its wavefronts take 256 bytes of K in turn, whole lines of 8 channels a load (and rows of X, from L2), straight
// to the MFMA operand's registers: no LDS, no barrier until the end, four chunks in flight a wavefront.  The wavefronts' sums are
// added in LDS, in whole numbers, so in any order.  One row x 4096 x 4096, calls in a row: 5.5 to 6.0 us, 2.8 to 3.0 TB/s; x 4096 x 14336
// 11.6 to 12.4, 4.7 to 5.1 TB/s.
#include "lds_dma.hpp"
#include "w8a8.hpp"

namespace lava {

template <bool GATED>
__global__ void __launch_bounds__(256) w8a8_stream_kernel(W8Args a, int tiles_n) {
    constexpr int NB = GATED ? 2 : 1, WAVES = 4;
    constexpr int CHUNK = 256, DEPTH = 4;   // bytes of K, chunks in flight
    __shared__ i32x4 part[WAVES][NB][64];
    __shared__ float s_ws[16 * NB], s_bias[16 * NB], s_xs[16];
    __shared__ int s_yr[16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tn = blockIdx.x % tiles_n;
    W8Tile tile;
    if (!w8_find(a, 16, blockIdx.x / tiles_n, tile)) return;
    const int half = a.n >> 1;
    const int col0 = tn * 16, cols_in = min(16, a.n_out - col0);

    // What the finish needs, requested first and held: a wavefront each for the channels' scales, their biases, the rows'
    // scales and the rows of Y.
    float held = 0.f;
    if (w < 2) {
        const int c = min(lane & 15, cols_in - 1);
        const int64_t ch = (int64_t)tile.expert * a.n + col0 + c + (GATED && (lane & 16) ? half : 0);
        const float* p = w == 0 ? a.ws : a.bias;
        if (p) held = p[ch];
    } else if (lane < tile.rows) {
        int xr, yr;
        w8_rows(a, tile, lane, xr, yr);
        held = w == 3 ? __int_as_float(yr) : xr < 0 ? 0.f : a.xs[xr];
    }

    // Rows, channels and bytes of K that are none get an offset outside the buffer and read zero.
    const bool gather = a.offsets != nullptr && !a.x_sorted;
    const int xfirst = gather ? 0 : tile.first, xrows = gather ? a.rows / a.top_k : tile.rows;
    const auto rx = w8_buffer(a.x + (int64_t)xfirst * a.ldx, (int64_t)(xrows - 1) * a.ldx + a.k);
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride + (int64_t)col0 * a.ldw;
    const int64_t wbytes = (int64_t)(cols_in - 1) * a.ldw + a.k;
    const auto rw = w8_buffer(wbase, wbytes), ru = w8_buffer(GATED ? wbase + (int64_t)half * a.ldw : wbase, wbytes);
    int xr = -1, yr;
    if ((lane & 15) < tile.rows) w8_rows(a, tile, lane & 15, xr, yr);
    const uint32_t xoff = xr < 0 ? OOB_OFS : (uint32_t)((int64_t)(xr - xfirst) * a.ldx + 32 * (lane >> 4));
    uint32_t woff[2];   // channels 0 .. 7 and 8 .. 15
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int c = 8 * h + (lane & 7);
        woff[h] = c < cols_in ? (uint32_t)(c * a.ldw + 16 * (lane >> 3)) : OOB_OFS;
    }
    // Two pieces of 128 bytes of K: of a block of channels, v[p][j][0] is the first 8 channels' whole lines, lane l channel l % 8,
    // bytes 16 (l / 8); v[p][j][1] the other 8's.
    struct Chunk {
        i32x4 x[2][2], v[2][NB][2];
    };
    // Rows of a power-of-two length lie on the same memory channels byte for byte: each workgroup begins at another chunk (one
    // row x 4096 x 4096 6.0 -> 5.6 us).
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
                for (int h = 0; h < 2; ++h) c.v[p][j][h] = w8_load<true>(j ? ru : rw, in ? woff[h] : OOB_OFS, k);
#pragma unroll
            for (int h = 0; h < 2; ++h) c.x[p][h] = w8_load<false>(rx, k + 32 * (lane >> 4) + 16 * h < a.k ? xoff : OOB_OFS, k + 16 * h);
        }
    };
    i32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = i32x4{0, 0, 0, 0};
    auto multiply = [&](Chunk& c) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                i32x4 v0, v1;
                w8_whole_lines(c.v[p][j][0], c.v[p][j][1], v0, v1);
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v0, c.x[p][0], acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v1, c.x[p][1], acc[j], 0, 0, 0);
            }
    };
    // No branch around a load: the compiler would wait for all that are in flight where it joins.
    Chunk ring[DEPTH];
    const int turns = (chunks + WAVES - 1) / WAVES;   // of every wavefront
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(ring[d], w + d * WAVES);
    for (int n = 0; n + DEPTH < turns; n += DEPTH) {
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
    for (int j = 0; j < NB; ++j) part[w][j][lane] = acc[j];
    if (w < 2 && lane < 16 * NB) (w == 0 ? s_ws : s_bias)[lane] = held;
    if (w == 2 && lane < 16) s_xs[lane] = held;
    if (w == 3 && lane < 16) s_yr[lane] = __float_as_int(held);
    __syncthreads();

    // One wavefront finishes: a lane has row lane % 16, columns 4 (lane / 16) and the next three.
    if (w != 0) return;
    const int m = lane & 15, c = 4 * (lane >> 4);
    if (m >= tile.rows || c >= cols_in || s_yr[m] < 0) return;
    auto values = [&](int j, float (&v)[4]) {
        i32x4 s = part[0][j][lane];
#pragma unroll
        for (int z = 1; z < WAVES; ++z) s += part[z][j][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = w8_value(s[r], s_xs[m], s_ws[16 * j + c + r], s_bias[16 * j + c + r]);
    };
    float v[4];
    values(0, v);
    w8_act4(a.act, v);
    if constexpr (GATED) {
        float u[4];
        values(1, u);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] *= u[r];
    }
    w8_store(a, (int64_t)s_yr[m] * a.ldy + col0 + c, cols_in - c, v);
}

bool w8_stream_fits(const W8Args& a) { return a.k > 0 && w8_chunks_fit(a) && w8_spans_fit(a, 16, 16) && w8_launch_fits(a, 16, 16, 256); }

// Up to 16 rows (of a plan: on average of an expert's that has any) on fewer tiles of 64 x 64 than half the CUs: those take as long
// as all CUs' would, as a CU reads HBM at some 25 bytes a ns at most.  us, here / on tiles: 16 rows x 4096 x 4096 7.2 / 9.2, x 4096 x
// 14336 16.6 / 22.8, one row 11.6 / 22.5; 16 x 8192 x 4096 10.9 / 9.5, x 14336 x 4096 15.8 / 11.9, one row 12.1 / 11.5.
bool w8_stream_preferred(const W8Args& a) { return a.rows <= 16 * w8_met(a) && w8_tile_count(a, 64, 64) <= 112; }

int launch_w8_stream(const W8Args& a, hipStream_t s) {
    const int64_t tm = w8_row_tiles(a, 16), tn = ((int64_t)a.n_out + 15) / 16;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(256), 0, s, a, (int)tn); };
    a.gated ? go(w8a8_stream_kernel<true>) : go(w8a8_stream_kernel<false>);
    LAVA_LAUNCH_CHECK("w8a8_stream_kernel");
    return LAVA_HIP_OK;
}

}  // namespace lava
