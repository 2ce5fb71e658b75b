// w8a8_stream.hip -- layers with 8-bit weights on few tokens: bound by reading the weights once.
//
// A workgroup has 16 MB rows and 16 NB channels over all of K.  Its wavefronts take 256 bytes of K in turn, each lane 16 bytes
// of a channel (and of a row of X, from L2) a load, in the MFMA operand's own layout: no LDS, no barrier until the end, and as
// many loads in flight as registers hold.  The wavefronts' sums are added in LDS, in whole numbers, so in any order.
#include "w8a8.hpp"

namespace lava {

template <int MB, int NB, int WAVES, bool GATED>
__global__ void __launch_bounds__(64 * WAVES) w8a8_stream_kernel(W8Args a, int tiles_n) {
    static_assert(!GATED || NB == 2, "a gated tile is 16 channels of the gate and their 16 factors");
    constexpr int DEPTH = 16 / (MB + NB) > 4 ? 4 : 16 / (MB + NB) < 2 ? 2 : 16 / (MB + NB);   // chunks in flight
    constexpr int CHUNK = 256;
    __shared__ i32x4 part[WAVES][MB * NB][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tn = blockIdx.x % tiles_n;
    W8Tile tile;
    if (!w8_find(a, 16 * MB, blockIdx.x / tiles_n, tile)) return;
    const int half = a.n >> 1;
    const int r16 = lane & 15, kofs = 16 * (lane >> 4);
    const int col0 = tn * (GATED ? 16 : 16 * NB);

    // Rows and channels that are none read the tile's first ones: their sums are not stored.
    const int8_t *xp[MB], *wp[NB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        int xr, yr;
        w8_rows(a, tile, min(16 * i + r16, tile.rows - 1), xr, yr);
        xp[i] = a.x + (int64_t)max(xr, 0) * a.ldx + kofs;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int c = min(col0 + (GATED ? 0 : 16 * j) + r16, a.n_out - 1) + (GATED && j ? half : 0);
        wp[j] = a.w + (int64_t)tile.expert * a.expert_stride + (int64_t)c * a.ldw + kofs;
    }
    i32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    struct Chunk {
        i32x4 x[4][MB], v[4][NB];
    };
    // Rows of a power-of-two length lie on the same memory channels byte for byte: each workgroup begins at another chunk.
    const int chunks = (a.k + CHUNK - 1) / CHUNK;
    const int turn = (tn + (tn >> 3)) % chunks;
    // 16 bytes are wholly inside K or outside (k is a multiple of 16); outside the first ones of the row are read, and X's count as zero
    auto load = [&](Chunk& c, int n) __attribute__((always_inline)) {
        n = n + turn < chunks ? n + turn : n + turn - chunks;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = n * CHUNK + 64 * s;
            const int at = k + kofs < a.k ? k : -kofs;
#pragma unroll
            for (int j = 0; j < NB; ++j) c.v[s][j] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(wp[j] + at));
#pragma unroll
            for (int i = 0; i < MB; ++i) c.x[s][i] = *reinterpret_cast<const i32x4*>(xp[i] + at);
        }
    };
    auto multiply = [&](Chunk& c, int n) __attribute__((always_inline)) {
        n = n + turn < chunks ? n + turn : n + turn - chunks;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const bool in = n * CHUNK + 64 * s + kofs < a.k;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const i32x4 x = in ? c.x[s][i] : i32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.v[s][j], x, acc[i][j], 0, 0, 0);
            }
        }
    };
    Chunk ring[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (w + d * WAVES < chunks) load(ring[d], w + d * WAVES);
    for (int n = w; n < chunks; n += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int at = n + d * WAVES;
            if (at < chunks) {
                multiply(ring[d], at);
                if (at + DEPTH * WAVES < chunks) load(ring[d], at + DEPTH * WAVES);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) part[w][i * NB + j][lane] = acc[i][j];
    __syncthreads();

    // Block b of the results (16 rows, 16 columns of Y) is finished by wavefront b % WAVES; a lane has row lane % 16, columns
    // 4 (lane / 16) and the next three.
    constexpr int OB = GATED ? MB : MB * NB;
    const int64_t sbase = (int64_t)tile.expert * a.n;
    for (int b = w; b < OB; b += WAVES) {
        const int i = GATED ? b : b / NB, j = GATED ? 0 : b % NB;
        const int m = 16 * i + r16, col = col0 + 16 * j + 4 * (lane >> 4);
        if (m >= tile.rows || col >= a.n_out) continue;
        int xr, yr;
        w8_rows(a, tile, m, xr, yr);
        if (yr < 0) continue;
        const float xs = a.xs[xr];
        auto values = [&](int blk, int64_t ch, float (&v)[4]) {
            i32x4 s = part[0][blk][lane];
#pragma unroll
            for (int z = 1; z < WAVES; ++z) s += part[z][blk][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (col + r < a.n_out) v[r] = w8_value(s[r], xs, a.ws[ch + r], a.bias ? a.bias[ch + r] : 0.f);
        };
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        values(i * NB + j, sbase + col, v);
        w8_act4(a.act, v);
        if constexpr (GATED) {
            float u[4] = {0.f, 0.f, 0.f, 0.f};
            values(i * NB + 1, sbase + half + col, u);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] *= u[r];
        }
        w8_store(a, (int64_t)yr * a.ldy + col, a.n_out - col, v);
    }
}

bool w8_stream_fits(const W8Args& a) { return a.k > 0 && w8_chunks_fit(a); }

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
