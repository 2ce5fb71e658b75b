// w8a8_tile.hip -- layers with 8-bit weights and tokens on tiles of 64 x 64 to 256 x 256 (rows x channels).
//
// The loop is the tile GEMM's (gemm_tn_kernel.hpp): 4 wavefronts, of tiles above 64 rows 8, each 16 WM rows x 16 WN channels in
// 16x16x64 MFMAs; K 128 bytes at a time, both operands' slices straight to LDS (buffer_load ... lds, 16-byte chunk c of row r at slot
// c ^ r % 8, so that a fragment's 16 rows lie on all banks), ST stages, one barrier in the middle of a stage: the MFMAs of its first
// half run while the second half's fragments are read, those of the second half while the next stage's are read and the one ST
// further on is requested.  What differs:
//  * a row of X is found by the plan, so a lane keeps one offset for each of its requests (rows and channels that are none,
//    and chunks past K, get an offset outside the buffer and read zero);
//  * a gated layer's tile has 16 channels of the gate and their 16 factors in turn, so that a lane has both of a column in its
//    accumulators;
//  * the sums go through LDS to lanes that have 8 columns of a row, which they finish, round to Y's type and store.
// Measured: 8192 rows x 28672 gated channels x 4096 735 to 825 us (770 in the middle, 2500 TOP/s) on 256 x 256 tiles, whose matrix cores are 0.66
// busy at a clock that falls to 1.8 GHz under them (with 4 wavefronts of 128 x 128 each 0.57 and 1.9, 760 to 780 us; 16384 rows x 8192 x 1024
// 181 us against 230); 16 rows x 14336 x 4096 11.6 us, 5.1 TB/s of weights; 32 tokens' 8 of 64 experts, gates and factors of 2816 x 2048,
// 65 us, 5.6 TB/s; one token's 11.0, 4.2 TB/s.  Between those, latency: of a tile's first requests and of its finish where K is short, of requests that miss
// L2 (two or three stages in flight a workgroup).
#include <math.h>

#include "gemm_tn_kernel.hpp"
#include "w8a8.hpp"

namespace lava {

// MW wavefronts along the rows, NW along the channels.
template <int MW, int NW, int WM, int WN, int ST, bool GATED>
__global__ void __launch_bounds__(64 * MW * NW, MW * NW == 4 || ST * 16 * (WM * MW + WN * NW) * TN_KB > 80 * 1024 ? 2 : 4)
    w8a8_tile_kernel(W8Args a, int tiles_m, int tiles_n) {
    constexpr int WAVES = MW * NW, BM = 16 * WM * MW, BN = 16 * WN * NW, XS = BM * TN_KB, STAGE = (BM + BN) * TN_KB;
    constexpr int Q = WM * WN, R = WM + WN;               // of a wavefront: MFMAs of half a stage, fragments read beside them
    constexpr int XD = 2 * WM / NW, D = XD + 2 * WN / MW;         // and its requests of a stage, those for X first
    static_assert(WM % 2 == 0 && (!GATED || WN % 2 == 0), "rows are finished 32 at a time, gates and factors are blocks of 16");
    static_assert(WN == 2 || WN == 4 || WN == 8, "a power of two of lanes finishes a row");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[ST * STAGE];
    __shared__ __attribute__((aligned(16))) float s_ws[BN], s_bias[BN];
    __shared__ float s_xs[BM];
    __shared__ int s_yr[BM];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    xcd_tile(blockIdx.x, tiles_m, tiles_n, 4, tm, tn);
    W8Tile tile;
    if (!w8_find(a, BM, tm, tile)) return;
    const int wm = w / NW, wn = w % NW;
    const int half = a.n >> 1;
    const int col0 = tn * (GATED ? BN / 2 : BN);   // first column of Y

    // What the finish needs, requested first and held until then: of row threadIdx.x its scale and row of Y, of channel row
    // threadIdx.x its scale and bias.
    static_assert(BM <= 64 * WAVES && BN <= 64 * WAVES, "a row and a channel a thread");
    float held_xs = 0.f, held_ws = 0.f, held_bias = 0.f;
    int held_yr = -1;
    if (threadIdx.x < (unsigned)tile.rows) {
        int xr;
        w8_rows(a, tile, threadIdx.x, xr, held_yr);
        if (xr >= 0) held_xs = a.xs[xr];
    }
    if (threadIdx.x < BN) {
        const int i = threadIdx.x, c = col0 + (GATED ? (i >> 5) * 16 + (i & 15) : i);
        const int64_t ch = (int64_t)tile.expert * a.n + (GATED && (i & 16) ? half + c : c);
        if (c < a.n_out) {
            held_ws = a.ws[ch];
            if (a.bias) held_bias = a.bias[ch];
        }
    }

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
    uint32_t xoff[XD], woff[D - XD], wsoff[D - XD];
#pragma unroll
    for (int i = 0; i < XD; ++i) {
        const int r = 8 * XD * w + 8 * i + lr;
        int xr = -1, yr;
        if (r < tile.rows) w8_rows(a, tile, r, xr, yr);
        xoff[i] = xr < 0 ? OOB_OFS : (uint32_t)((int64_t)(xr - xfirst) * a.ldx + chunk);
    }
#pragma unroll
    for (int i = 0; i < D - XD; ++i) {
        const int r = 8 * (D - XD) * w + 8 * i;
        const int c = GATED ? (r >> 5) * 16 + (r & 8) : r;
        wsoff[i] = (uint32_t)(c * a.ldw);
        woff[i] = c + lr < cols_in ? (uint32_t)(lr * a.ldw + chunk) : OOB_OFS;
    }
    const uint32_t lds_x = lds_addr(smem) + w * XD * 1024, lds_w = lds_addr(smem) + XS + w * (D - XD) * 1024;

    // request q of the stage at byte kofs of K
    auto dma = [&](int q, int stage, uint32_t kofs) __attribute__((always_inline)) {
        if (q < XD) {
            dma16(rx, xoff[q], kofs, lds_x + stage * STAGE + q * 1024);
        } else {
            const int i = q - XD;
            const bool up = GATED && ((8 * (D - XD) * w + 8 * i) & 16);   // a block of factors; uniform
            dma16(up ? ru : rw, woff[i], wsoff[i] + kofs, lds_w + stage * STAGE + i * 1024);
        }
    };
    // Before the last stage's requests: chunks past K get an offset that reads zero (once, in the kept offsets: a
    // choice at every request costs the compiler the accumulators' places, 8192 gated rows 1183 us against 780, with 4 wavefronts).
    const int ktiles = (a.k + TN_KB - 1) / TN_KB;
    auto cut_k = [&]() __attribute__((always_inline)) {
        const bool in = (ktiles - 1) * TN_KB + chunk < a.k;
#pragma unroll
        for (int i = 0; i < XD; ++i) xoff[i] = in ? xoff[i] : OOB_OFS;
#pragma unroll
        for (int i = 0; i < D - XD; ++i) woff[i] = in ? woff[i] : OOB_OFS;
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
        for (int q = 0; q < D; ++q) dma(q, t, (uint32_t)min(t, ktiles - 1) * TN_KB);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * D) : "memory");
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
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 2) * D) : "memory");   // this wavefront's part of the next stage landed
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            acc[q / WN][q % WN] = Mfma16<int8_t>::run(fb.v[q % WN], fb.x[q / WN], acc[q / WN][q % WN]);
#pragma unroll
            for (int t = q * R / Q; t < (q + 1) * R / Q; ++t) read(fa, next, 0, t);
#pragma unroll
            for (int t = q * D / Q; t < (q + 1) * D / Q; ++t) dma(t, st, kofs2);
            __builtin_amdgcn_sched_barrier(0);
        }
        st = st1;
    }

    // ---- finish: acc[i][j][r] is row 16 WM wm + 16 i + lane % 16, channel row 16 WN wn + 16 j + 4 (lane / 16) + r.  A wavefront
    // stages the sums of 32 rows at a time in LDS of its own and reads them back by rows, a lane 8 columns of Y (of a gated layer
    // their 8 gates and 8 factors), which it finishes and stores.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (threadIdx.x < BM) {
        s_xs[threadIdx.x] = held_xs;
        s_yr[threadIdx.x] = held_yr;
    }
    if (threadIdx.x < BN) {
        s_ws[threadIdx.x] = held_ws;
        s_bias[threadIdx.x] = held_bias;
    }
    __syncthreads();
    constexpr int COLS = GATED ? 8 * WN : 16 * WN;         // of Y, a wavefront's
    constexpr int PITCH = 16 * WN * 4 + 16;                // padded: the 16 rows of a store start on distinct banks
    constexpr int EI = WAVES * 32 * PITCH <= ST * STAGE ? 2 : 1;   // blocks of 16 rows at a time
    static_assert(WAVES * EI * 16 * PITCH <= ST * STAGE, "the wavefronts' rows in the stages' LDS");
    constexpr int LANES = COLS / 8, ROWS = 64 / LANES;     // lanes a row, rows a pass
    uint8_t* ep = smem + w * EI * 16 * PITCH;
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
    auto finish = [&](auto itag) __attribute__((always_inline)) {
        constexpr int i0 = decltype(itag)::value;
#pragma unroll
        for (int ii = 0; ii < EI; ++ii)
#pragma unroll
            for (int j = 0; j < WN; ++j)
                *reinterpret_cast<i32x4*>(ep + (16 * ii + (lane & 15)) * PITCH + (16 * j + 4 * (lane >> 4)) * 4) = acc[i0 + ii][j];
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the wavefront's sums are in LDS
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int t = 0; t < 16 * EI / ROWS; ++t) {
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
    finish(std::integral_constant<int, 0>{});
    if constexpr (WM > EI) finish(std::integral_constant<int, EI>{});
    if constexpr (WM > 2 * EI) finish(std::integral_constant<int, 2 * EI>{});
    if constexpr (WM > 3 * EI) finish(std::integral_constant<int, 3 * EI>{});
    static_assert(WM <= 4 * EI, "four times");
}

template <int MW, int NW, int WM, int WN, int ST>
int launch_tile(const W8Args& a, hipStream_t s, const char* name) {
    const int cols = (a.gated ? 8 : 16) * WN * NW;
    const int64_t tm = w8_row_tiles(a, 16 * MW * WM), tn = ((int64_t)a.n_out + cols - 1) / cols;   // w8_tile_fits: of them few enough
    const dim3 grid((unsigned)(tm * tn));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * MW * NW), 0, s, a, (int)tm, (int)tn); };
    a.gated ? go(w8a8_tile_kernel<MW, NW, WM, WN, ST, true>) : go(w8a8_tile_kernel<MW, NW, WM, WN, ST, false>);
    LAVA_LAUNCH_CHECK(name);
    return LAVA_HIP_OK;
}

// What a tile costs a CU: us before and behind the loop, us each 128 bytes of K, and, where a CU has several, the share of one at the
// end in which CUs wait for others (a CU runs several of the small ones at once, one of the two largest).  Fitted to the times of
// all five at 730 shapes of 40 to 8192 rows, 1024 to 20480 channels and K of 128 to 7168 and at 240 plans of 8 to 256 experts.
constexpr struct {
    int bm, bn, threads;
    float fixed, stage, end;
} W8_TILES[W8_TILE_KINDS] = {{64, 64, 256, 0.74f, 0.40f, 0.3f},
                             {64, 128, 256, 2.8f, 0.39f, 0.3f},
                             {128, 128, 512, 2.7f, 0.62f, 0.3f},
                             {128, 256, 512, 10.2f, 0.80f, 0.53f},
                             {256, 256, 512, 14.6f, 1.47f, 0.53f}};

bool w8_tile_fits(const W8Args& a, int tile) {
    const auto& t = W8_TILES[tile];
    return a.k > 0 && w8_chunks_fit(a) && w8_spans_fit(a, t.bm, t.bn) && w8_launch_fits(a, t.bm, a.gated ? t.bn / 2 : t.bn, t.threads);
}

double w8_met(const W8Args& a) { return a.offsets ? a.experts * -expm1(-(double)a.rows / a.experts) : 1; }

double w8_tile_count(const W8Args& a, int bm, int bn) {
    const double tn = (a.n_out + (a.gated ? bn / 2 : bn) - 1) / (a.gated ? bn / 2 : bn);
    if (a.offsets == nullptr) return ((a.rows + bm - 1) / bm) * tn;
    // of a plan: each expert that has rows has half a tile more than whole ones
    const double met = w8_met(a), whole = (double)a.rows / bm + 0.5 * met;
    return (met > whole ? met : whole) * tn;
}

// The least estimate: up to 256 tiles in the time of one, more in that of their share of a CU and the end.  Over those shapes 0.5 % behind
// the best of the five, over the plans 3.4 % (at worst half, at few tiles).  us of {64 x 64, 64 x 128, 128 x 128, 128 x 256, 256 x 256},
// the rule's in brackets: 64 rows x 14336 x 4096 {[16.8], 22.4, 23.2, 32.8, 54}, 333 rows {47, 41.3, 38.6, [34.4], 55}, 2048 x 4096 x
// 4096 {54, 51.9, 37.6, [35.9], 47}, 1024 rows {29.8, 26.1, [22.2], 29.4, 45.8}, 4096 rows {103, 86, 71, 64, [58]}; 5003 tokens and 4
// of 60 experts of 2048 x 1408 {168, 129, [123], 116, 132}, of 2816 x 2048 {298, 235, 220, [207], 208}.
int w8_tile_choice(const W8Args& a) {
    const double stages = (a.k + TN_KB - 1) / TN_KB;
    int best = -1;
    double least = 0;
    for (int i = 0; i < W8_TILE_KINDS; ++i) {
        if (!w8_tile_fits(a, i)) continue;
        const double per_cu = w8_tile_count(a, W8_TILES[i].bm, W8_TILES[i].bn) / 256;
        const double cost = (per_cu <= 1 ? 1 : per_cu + W8_TILES[i].end) * (W8_TILES[i].fixed + W8_TILES[i].stage * stages);
        if (best < 0 || cost < least) {
            best = i;
            least = cost;
        }
    }
    return best;
}

int launch_w8_tile(const W8Args& a, int tile, hipStream_t s) {
    // Where a CU has one tile at most, a stage more in flight; else more tiles a CU (128 x 128, us with 2 stages / 3: 1024 x 4096 x
    // 4096, 256 tiles, 26.7 / 22.1; 2048 rows 36.7 / 41.5).
    const bool lone = w8_tile_count(a, W8_TILES[tile].bm, W8_TILES[tile].bn) <= 256;
    // the log names a tile and its form with that many stages
#define LAVA_W8_TILE(MW, NW, WM, WN, ST, TILE) \
    launch_tile<MW, NW, WM, WN, ST>(a, s, "w8a8_tile_kernel<" TILE ">+w8a8_tile_kernel<" TILE "," #ST ">")
    switch (tile) {
    case 0: return lone ? LAVA_W8_TILE(2, 2, 2, 2, 4, "64,64") : LAVA_W8_TILE(2, 2, 2, 2, 3, "64,64");
    case 1: return lone ? LAVA_W8_TILE(2, 2, 2, 4, 3, "64,128") : LAVA_W8_TILE(2, 2, 2, 4, 2, "64,128");
    case 2: return lone ? LAVA_W8_TILE(4, 2, 2, 4, 3, "128,128") : LAVA_W8_TILE(4, 2, 2, 4, 2, "128,128");
    case 3: return LAVA_W8_TILE(2, 4, 4, 4, 3, "128,256");
    default: return LAVA_W8_TILE(4, 2, 4, 8, 2, "256,256");
    }
#undef LAVA_W8_TILE
}

}  // namespace lava
