// w8a8_mid.hip -- layers with 8-bit weights on 17 to some hundred tokens (or rows an expert): between the weights' bytes and
// the matrix cores.
//
// A workgroup has 16 MB rows x 64 NB channels, its 4 wavefronts side by side in the channels, 16 NB each.  So a wavefront's
// weights are its own and go straight to registers, whole lines of 8 channels a load; only the rows of X, which all four
// need, go through LDS (128 bytes of K a stage, a ring of ST, filled by buffer_load ... lds, chunk c of row r at slot
// c ^ r % 8).  LDS then moves 16 MB rows x 128 bytes x 4 a stage and nothing for the weights: with both operands staged, as in
// the 128 x 128 tile kernel, LDS is what bounds this size.  One barrier a stage; weights are requested ST - 1 stages ahead,
// right behind the rows of the same stage.
#include <type_traits>

#include "lds_dma.hpp"
#include "w8a8.hpp"

namespace lava {

template <int MB, int NB, int ST, bool GATED>
__global__ void __launch_bounds__(256, MB * NB > 16 ? 1 : 2) w8a8_mid_kernel(W8Args a, int tiles_m, int tiles_n) {
    static_assert(MB % 2 == 0, "rows are requested 32 at a time");
    static_assert(!GATED || NB % 2 == 0, "a gated layer's blocks are gates and factors in turn");
    constexpr int KB = 128, BM = 16 * MB, BN = 64 * NB, STAGE = BM * KB, D = ST - 1;
    constexpr int XD = BM / 32, WL = 2 * NB;   // requests of a stage by a wavefront: for X, for W
    constexpr int COLS = GATED ? 8 * NB : 16 * NB;    // of Y, a wavefront's
    constexpr int PITCH = 16 * NB * 4 + 16;
    constexpr int LDS = ST * STAGE > 4 * 32 * PITCH ? ST * STAGE : 4 * 32 * PITCH;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[LDS];
    __shared__ float s_xs[BM], s_ws[BN], s_bias[BN];
    __shared__ int s_xr[BM], s_yr[BM];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    xcd_tile(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
    W8Tile tile;
    if (!w8_find(a, BM, tm, tile)) return;
    const int half = a.n >> 1;
    const int col0 = tn * 4 * COLS;
    const int cols_in = min(4 * COLS, a.n_out - col0);

    for (int i = threadIdx.x; i < BM; i += 256) {
        int xr = -1, yr = -1;
        if (i < tile.rows) w8_rows(a, tile, i, xr, yr);
        s_xr[i] = xr;
        s_yr[i] = yr;
        s_xs[i] = xr < 0 ? 0.f : a.xs[xr];
    }
    for (int i = threadIdx.x; i < BN; i += 256) {
        const int c = col0 + (GATED ? (i >> 5) * 16 + (i & 15) : i);
        const int64_t ch = (int64_t)tile.expert * a.n + (GATED && (i & 16) ? half + c : c);
        s_ws[i] = c < a.n_out ? a.ws[ch] : 0.f;
        s_bias[i] = c < a.n_out && a.bias ? a.bias[ch] : 0.f;
    }
    __syncthreads();

    const bool gather = a.offsets != nullptr && !a.x_sorted;
    const int xfirst = gather ? 0 : tile.first, xrows = gather ? a.rows / a.top_k : tile.rows;
    const v4i rx = make_rsrc(a.x + (int64_t)xfirst * a.ldx, (uint32_t)((int64_t)(xrows - 1) * a.ldx + a.k));
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride + (int64_t)col0 * a.ldw;
    const int64_t wbytes = (int64_t)(cols_in - 1) * a.ldw + a.k;
    const auto rw = w8_buffer(wbase, wbytes), ru = w8_buffer(GATED ? wbase + (int64_t)half * a.ldw : wbase, wbytes);

    // X: a request covers 8 rows, lane l row l / 8, slot l % 8, which holds chunk slot ^ row % 8; wavefront w's are rows
    // 8 XD w and on
    const int lr = lane >> 3, chunk = 16 * ((lane & 7) ^ lr);
    uint32_t xoff[XD];
#pragma unroll
    for (int i = 0; i < XD; ++i) {
        const int xr = s_xr[8 * (XD * w + i) + lr];
        xoff[i] = xr < 0 ? OOB_OFS : (uint32_t)((int64_t)(xr - xfirst) * a.ldx + chunk);
    }
    const uint32_t lds_x = lds_addr(smem) + 8 * XD * w * KB;
    // W: lane l channel l % 8 of 8, bytes 16 (l / 8) of a line
    uint32_t woff[NB][2];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * NB * w + 16 * j + 8 * h + (lane & 7);
            const int c = GATED ? (r >> 5) * 16 + (r & 15) : r;
            woff[j][h] = c < cols_in ? (uint32_t)(c * a.ldw + 16 * (lane >> 3)) : OOB_OFS;
        }

    i32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    struct Weights {
        i32x4 v[NB][2];
    };
    Weights ring[D];
    // stage t's rows into slot `slot` of the ring, and its weights; past K both read zero and the counts stay
    auto request = [&](Weights& c, int slot, int t) __attribute__((always_inline)) {
        const int at = t * KB;
        const bool xin = at + chunk < a.k;
#pragma unroll
        for (int i = 0; i < XD; ++i) dma16(rx, xin ? xoff[i] : OOB_OFS, at, lds_x + slot * STAGE + i * 1024);
        const bool in = at + 16 * (lane >> 3) < a.k;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) c.v[j][h] = w8_load<true>(GATED && (j & 1) ? ru : rw, in ? woff[j][h] : OOB_OFS, at);
    };
    const int ktiles = (a.k + KB - 1) / KB;
#pragma unroll
    for (int d = 0; d < D; ++d) request(ring[d], d, d);
    // fragments: row 16 i + lane % 16, the 16 bytes 32 (lane / 16) + 16 h, which are what the weights' lanes have (below)
    const int rd = (lane & 15) * KB;
    int slot16[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) slot16[h] = ((2 * (lane >> 4) + h) ^ (lane & 7)) * 16;
    int st = 0, fill = D;
    // multiplies the ring's stage d, which is the oldest; more: and requests stage t in its place
    auto step = [&](int d, bool more, int t) __attribute__((always_inline)) {
        // this wavefront's requests of the stage landed (those of the later ones may not have); everyone's, and everyone
        // has read the stage before
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((D - 1) * (XD + WL)) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t* base = smem + st * STAGE;
        i32x4 v[NB][2];
#pragma unroll
        for (int j = 0; j < NB; ++j) w8_whole_lines(ring[d].v[j][0], ring[d].v[j][1], v[j][0], v[j][1]);
        if (more) request(ring[d], fill, t);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const i32x4 x = *reinterpret_cast<const i32x4*>(base + rd + i * 16 * KB + slot16[h]);
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[j][h], x, acc[i][j], 0, 0, 0);
            }
        fill = st;
        st = st + 1 == ST ? 0 : st + 1;
    };
    int kt = 0;
    for (; kt + D <= ktiles; kt += D) {   // no branch inside: the compiler would wait for all loads where it joins
#pragma unroll
        for (int d = 0; d < D; ++d) step(d, true, kt + d + D);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (kt + d < ktiles) step(d, false, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();

    // ---- finish, as in the tile kernel: a wavefront's sums by rows through LDS of its own, a lane 8 columns
    constexpr int LANES = COLS / 8, PASS = 64 / LANES;   // lanes a row, rows a pass
    uint8_t* ep = smem + w * 32 * PITCH;
    const int cc = (lane % LANES) * 8, cr = GATED ? (cc >> 4) * 32 + (cc & 15) : cc;
    const int left = a.n_out - (col0 + w * COLS + cc);
    f32x4 ws[GATED ? 4 : 2], bs[GATED ? 4 : 2];
#pragma unroll
    for (int h = 0; h < (GATED ? 4 : 2); ++h) {
        const int c = w * 16 * NB + cr + (h >> 1) * 16 + (h & 1) * 4;
        ws[h] = *reinterpret_cast<const f32x4*>(s_ws + c);
        bs[h] = *reinterpret_cast<const f32x4*>(s_bias + c);
    }
    auto rows32 = [&](auto itag) __attribute__((always_inline)) {
        constexpr int i0 = decltype(itag)::value;
        if constexpr (i0 < MB) {
#pragma unroll
            for (int ii = 0; ii < 32 / 16; ++ii)
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    *reinterpret_cast<i32x4*>(ep + (16 * ii + (lane & 15)) * PITCH + (16 * j + 4 * (lane >> 4)) * 4) = acc[i0 + ii][j];
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the wavefront's sums are in LDS
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int row = lane / LANES; row < 32; row += PASS) {
                const float xs = s_xs[16 * i0 + row];
                const int yr = s_yr[16 * i0 + row];
                float v[8];
                w8_finish8<GATED>(a.act, reinterpret_cast<const i32x4*>(ep + row * PITCH + cr * 4), xs, ws, bs, v);
                if (yr >= 0 && left > 0) w8_store(a, (int64_t)yr * a.ldy + col0 + w * COLS + cc, left, v);
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);   // read before the next rows overwrite them
            __builtin_amdgcn_wave_barrier();
        }
    };
    rows32(std::integral_constant<int, 0>{});
    rows32(std::integral_constant<int, 2>{});
    rows32(std::integral_constant<int, 4>{});
    rows32(std::integral_constant<int, 6>{});
}

bool w8_mid_fits(const W8Args& a) { return a.k > 0 && w8_chunks_fit(a) && w8_spans_fit(a, 128, 256); }

int launch_w8_mid(const W8Args& a, int MB, int NB, hipStream_t s) {
    if (a.gated && NB == 1) NB = 2;   // blocks of gates and factors in turn
    const int cols = a.gated ? 32 * NB : 64 * NB;
    const int64_t tm = w8_row_tiles(a, 16 * MB), tn = ((int64_t)a.n_out + cols - 1) / cols;
    LAVA_REQUIRE(tm * tn <= 0xffffff, LAVA_HIP_ERR_UNSUPPORTED, "w8a8_mid_kernel would need %lld workgroups", (long long)(tm * tn));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(256), 0, s, a, (int)tm, (int)tn); };
    auto by_cols = [&](auto mtag) {
        constexpr int M = decltype(mtag)::value;
        if (NB == 4) a.gated ? go(w8a8_mid_kernel<M, 4, 5, true>) : go(w8a8_mid_kernel<M, 4, 5, false>);
        else if (NB == 2) a.gated ? go(w8a8_mid_kernel<M, 2, 6, true>) : go(w8a8_mid_kernel<M, 2, 6, false>);
        else go(w8a8_mid_kernel<M, 1, 7, false>);
    };
    if (MB == 2) by_cols(std::integral_constant<int, 2>{});
    else if (MB == 4) by_cols(std::integral_constant<int, 4>{});
    else by_cols(std::integral_constant<int, 8>{});
    LAVA_LAUNCH_CHECK("w8a8_mid_kernel");
    return LAVA_HIP_OK;
}

}  // namespace lava
