// w8a8_tile.hip -- layers with 8-bit weights and tokens on 256 x 256 or 128 x 128 tiles (rows x channels).
//
// The loop is the tile GEMM's (gemm_tn_kernel.hpp): 4 wavefronts, each 16 WM rows x 16 WN channels in 16x16x64 MFMAs; K 128
// bytes at a time, both operands' slices straight to LDS (buffer_load ... lds, 16-byte chunk c of row r at slot c ^ r % 8, so
// that a fragment's 16 rows lie on all banks), two stages, one barrier in the middle of a stage: the MFMAs of its first half
// run while the second half's fragments are read, those of the second half while the next stage's are read and the stage
// after it is requested.  What differs:
//  * a row of X is found by the plan, so a lane keeps one offset for each of its requests (rows and channels that are none,
//    and chunks past K, get an offset outside the buffer and read zero);
//  * a gated layer's tile has 16 channels of the gate and their 16 factors in turn, so that a lane has both of a column in its
//    accumulators;
//  * the sums go through LDS to lanes that have 8 columns of a row, which they finish, round to Y's type and store.
#include "gemm_tn_kernel.hpp"
#include "w8a8.hpp"

namespace lava {

template <int WM, int WN, int ST, bool GATED>
__global__ void __launch_bounds__(256, 1) w8a8_tile_kernel(W8Args a, int tiles_m, int tiles_n) {
    constexpr int BM = 32 * WM, BN = 32 * WN, XS = BM * TN_KB, STAGE = (BM + BN) * TN_KB;
    constexpr int Q = WM * WN, R = WM + WN;   // MFMAs of half a stage, and fragments read (and requests made) beside them
    __shared__ __attribute__((aligned(1024))) uint8_t smem[ST * STAGE];
    __shared__ float s_xs[BM], s_ws[BN], s_bias[BN];
    __shared__ int s_xr[BM], s_yr[BM];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    xcd_tile(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
    W8Tile tile;
    if (!w8_find(a, BM, tm, tile)) return;
    const int wm = w >> 1, wn = w & 1;
    const int half = a.n >> 1;
    const int col0 = tn * (GATED ? BN / 2 : BN);   // first column of Y

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

    // X: rows of the tokens by offsets from the first of all, or rows of the tile by offsets from its own first
    const bool gather = a.offsets != nullptr && !a.x_sorted;
    const int xfirst = gather ? 0 : tile.first;
    const int xrows = gather ? a.rows / a.top_k : tile.rows;
    const v4i rx = make_rsrc(a.x + (int64_t)xfirst * a.ldx, (uint32_t)((int64_t)(xrows - 1) * a.ldx + a.k));
    const int cols_in = min(GATED ? BN / 2 : BN, a.n_out - col0);
    const int8_t* wbase = a.w + (int64_t)tile.expert * a.expert_stride + (int64_t)col0 * a.ldw;
    const uint32_t wbytes = (uint32_t)((int64_t)(cols_in - 1) * a.ldw + a.k);
    const v4i rw = make_rsrc(wbase, wbytes);
    const v4i ru = make_rsrc(GATED ? wbase + (int64_t)half * a.ldw : wbase, wbytes);
    // a request covers 8 rows: lane l row l / 8, slot l % 8, which holds chunk slot ^ row % 8
    const int lr = lane >> 3, chunk = 16 * ((lane & 7) ^ lr);
    uint32_t xoff[WM], woff[WN], wsoff[WN];
#pragma unroll
    for (int i = 0; i < WM; ++i) {
        const int xr = s_xr[8 * WM * w + 8 * i + lr];
        xoff[i] = xr < 0 ? OOB_OFS : (uint32_t)((int64_t)(xr - xfirst) * a.ldx + chunk);
    }
#pragma unroll
    for (int i = 0; i < WN; ++i) {
        const int r = 8 * WN * w + 8 * i;
        const int c = GATED ? (r >> 5) * 16 + (r & 8) : r;
        wsoff[i] = (uint32_t)(c * a.ldw);
        woff[i] = c + lr < cols_in ? (uint32_t)(lr * a.ldw + chunk) : OOB_OFS;
    }
    const uint32_t lds_x = lds_addr(smem) + w * 8 * WM * TN_KB, lds_w = lds_addr(smem) + XS + w * 8 * WN * TN_KB;

    // request q (of WM for X and WN for W) of the stage at byte kofs of K
    auto dma = [&](int q, int stage, uint32_t kofs) __attribute__((always_inline)) {
        if (q < WM) {
            dma16(rx, xoff[q], kofs, lds_x + stage * STAGE + q * 1024);
        } else {
            const int i = q - WM;
            const bool up = GATED && ((i >> 1) & 1);   // 8 WN w + 8 i is in a block of factors (WN a multiple of 4)
            dma16(up ? ru : rw, woff[i], wsoff[i] + kofs, lds_w + stage * STAGE + i * 1024);
        }
    };
    // Before the last stage's requests: chunks past K get an offset that reads zero (once, in the kept offsets: a choice at
    // every request costs the compiler the accumulators' places, 1185 against 9xx us for 8192 gated rows).
    const int ktiles = (a.k + TN_KB - 1) / TN_KB;
    auto cut_k = [&]() __attribute__((always_inline)) {
        const bool in = (ktiles - 1) * TN_KB + chunk < a.k;
#pragma unroll
        for (int i = 0; i < WM; ++i) xoff[i] = in ? xoff[i] : OOB_OFS;
#pragma unroll
        for (int i = 0; i < WN; ++i) woff[i] = in ? woff[i] : OOB_OFS;
    };

    i32x4 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    // fragments of half a stage (64 bytes of K): x[i] rows 16 i, v[j] channels 16 j of the wavefront's
    struct Frag {
        uint4 x[WM], v[WN];
    };
    const int rd_x = (wm * 16 * WM + (lane & 15)) * TN_KB, rd_w = XS + (wn * 16 * WN + (lane & 15)) * TN_KB;
    int slot[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) slot[u] = ((4 * u + (lane >> 4)) ^ (lane & 7)) * 16;
    // fragment t in the order of its first use: x[0], v[0 ..], x[1 ..]
    auto read = [&](Frag& f, const uint8_t* stage, int u, int t) __attribute__((always_inline)) {
        if (t == 0 || t > WN) {
            const int i = t == 0 ? 0 : t - WN;
            f.x[i] = *reinterpret_cast<const uint4*>(stage + rd_x + i * 16 * TN_KB + slot[u]);
        } else {
            f.v[t - 1] = *reinterpret_cast<const uint4*>(stage + rd_w + (t - 1) * 16 * TN_KB + slot[u]);
        }
    };

#pragma unroll
    for (int t = 0; t < ST; ++t) {
        if (t + 1 == ktiles) cut_k();
#pragma unroll
        for (int q = 0; q < R; ++q) dma(q, t, (uint32_t)min(t, ktiles - 1) * TN_KB);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * R) : "memory");
    __syncthreads();
    Frag fa, fb;
#pragma unroll
    for (int t = 0; t < R; ++t) {
        read(fa, smem, 0, t);
        __builtin_amdgcn_sched_barrier(0);
    }
    int st = 0;
    for (int kt = 0; kt < ktiles; ++kt) {
        const int st1 = ST == 2 ? st ^ 1 : st + 1 == ST ? 0 : st + 1;
        const uint8_t *base = smem + st * STAGE, *next = smem + st1 * STAGE;
        const uint32_t kofs2 = (uint32_t)min(kt + ST, ktiles - 1) * TN_KB;
        if (kt + ST + 1 == ktiles) cut_k();
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            acc[q / WN][q % WN] = Mfma16<int8_t>::run(fa.v[q % WN], fa.x[q / WN], acc[q / WN][q % WN]);
#pragma unroll
            for (int t = q * R / Q; t < (q + 1) * R / Q; ++t) read(fb, base, 1, t);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 2) * R) : "memory");   // this wavefront's part of the next stage landed
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            acc[q / WN][q % WN] = Mfma16<int8_t>::run(fb.v[q % WN], fb.x[q / WN], acc[q / WN][q % WN]);
#pragma unroll
            for (int t = q * R / Q; t < (q + 1) * R / Q; ++t) {
                read(fa, next, 0, t);
                dma(t, st, kofs2);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        st = st1;
    }

    // ---- finish: acc[i][j][r] is row 16 WM wm + 16 i + lane % 16, channel row 16 WN wn + 16 j + 4 (lane / 16) + r.  A wavefront
    // stages the sums of 32 rows at a time in LDS of its own and reads them back by rows, a lane 8 columns of Y (of a gated layer
    // their 8 gates and 8 factors), which it finishes and stores.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    constexpr int COLS = GATED ? 8 * WN : 16 * WN;         // of Y, a wavefront's
    constexpr int PITCH = 16 * WN * 4 + 16;                // padded: the 16 rows of a store start on distinct banks
    static_assert(4 * 32 * PITCH <= ST * STAGE, "four wavefronts' rows in the stages' LDS");
    constexpr int LANES = COLS / 8, ROWS = 64 / LANES;     // lanes a row, rows a pass
    uint8_t* ep = smem + w * 32 * PITCH;
    const int cc = (lane % LANES) * 8;                     // this lane's first column of the wavefront's
    const int cr = GATED ? (cc >> 4) * 32 + (cc & 15) : cc;   // and channel row
    const int left = a.n_out - (col0 + wn * COLS + cc);    // columns of Y from there on
    f32x4 ws[GATED ? 4 : 2], bs[GATED ? 4 : 2];
#pragma unroll
    for (int h = 0; h < (GATED ? 4 : 2); ++h) {
        const int c = wn * 16 * WN + cr + (h >> 1) * 16 + (h & 1) * 4;
        ws[h] = *reinterpret_cast<const f32x4*>(s_ws + c);
        bs[h] = *reinterpret_cast<const f32x4*>(s_bias + c);
    }
    auto rows32 = [&](auto itag) __attribute__((always_inline)) {
        constexpr int i0 = decltype(itag)::value;
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
            for (int j = 0; j < WN; ++j)
                *reinterpret_cast<i32x4*>(ep + (16 * ii + (lane & 15)) * PITCH + (16 * j + 4 * (lane >> 4)) * 4) = acc[i0 + ii][j];
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the wavefront's sums are in LDS
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int t = 0; t < 32 / ROWS; ++t) {
            const int row = t * ROWS + lane / LANES, at = wm * 16 * WM + 16 * i0 + row;
            const float xs = s_xs[at];
            const int yr = s_yr[at];
            float v[8];
            w8_finish8<GATED>(a.act, reinterpret_cast<const i32x4*>(ep + row * PITCH + cr * 4), xs, ws, bs, v);
            if (yr >= 0 && left > 0) w8_store(a, (int64_t)yr * a.ldy + col0 + wn * COLS + cc, left, v);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);   // read before the next rows overwrite them
        __builtin_amdgcn_wave_barrier();
    };
    rows32(std::integral_constant<int, 0>{});
    rows32(std::integral_constant<int, 2>{});
    if constexpr (WM > 4) {
        rows32(std::integral_constant<int, 4 % WM>{});
        rows32(std::integral_constant<int, 6 % WM>{});
    }
}

bool w8_tile_fits(const W8Args& a, int BM) { return a.k > 0 && w8_chunks_fit(a) && w8_spans_fit(a, BM, BM); }

int launch_w8_tile(const W8Args& a, int BM, hipStream_t s) {
    const int cols = a.gated ? BM / 2 : BM;
    const int64_t tm = w8_row_tiles(a, BM), tn = ((int64_t)a.n_out + cols - 1) / cols;
    LAVA_REQUIRE(tm * tn <= 0xffffff, LAVA_HIP_ERR_UNSUPPORTED, "w8a8_tile_kernel would need %lld workgroups", (long long)(tm * tn));
    const dim3 grid((unsigned)(tm * tn));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, (int)tm, (int)tn); };
    if (BM == 256) {
        a.gated ? go(w8a8_tile_kernel<8, 8, 2, true>) : go(w8a8_tile_kernel<8, 8, 2, false>);
        LAVA_LAUNCH_CHECK("w8a8_tile_kernel<256>");
    } else {
        a.gated ? go(w8a8_tile_kernel<4, 4, 4, true>) : go(w8a8_tile_kernel<4, 4, 4, false>);
        LAVA_LAUNCH_CHECK("w8a8_tile_kernel<128>");
    }
    return LAVA_HIP_OK;
}

}  // namespace lava
