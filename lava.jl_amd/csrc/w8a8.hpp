// w8a8.hpp -- what the kernels of layers with 8-bit weights and tokens share (internal): their arguments, the rows of a
// tile, and the finish of a sum.
//
// A tile is BM rows of one expert's run (of a plain layer: of the tokens) times BN channels.  A kernel's grid holds an
// upper bound of the row tiles -- the runs' lengths are device memory: rows / BM whole ones and one begun per expert --
// and a workgroup finds its own by a scan of the offsets (w8_find); those behind the last end at once.
#pragma once
#include <hip/hip_runtime.h>

#include "gemm_common.hpp"
#include "lava_hip_internal.hpp"

namespace lava {

// Channels and rows at most: the last tile's, up to 255 behind them, are counted in 32 bits too.
constexpr int64_t W8_MOST = 0x7fffff00;

struct W8Args {
    const int8_t* x;
    const float* xs;
    const int8_t* w;
    const float* ws;
    const float* bias;
    void* y;
    int64_t ldx, ldw, expert_stride, ldy;
    const int32_t* offsets;   // of a plan; null: a plain layer on rows 0 .. rows - 1
    const int32_t* order;
    int n;                    // channels
    int n_out;                // columns of Y
    int k;
    int rows;                 // tokens, or a plan's tokens * top_k
    int top_k, experts;
    int act, gated, y_dtype;
    int x_sorted, y_sorted;
};

struct W8Tile {
    int expert;
    int first;   // its first row, of the tokens or in the plan's order
    int rows;    // 1 .. BM
};

// Of lane l: the sum of v over lanes 0 .. l.
__device__ __forceinline__ int wave_sums(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8: within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15: lane 15's to 16 .. 31, 47's to 48 .. 63
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31: lane 31's to 32 .. 63
    return v;
}

// Row tile t of BM rows; false behind the last.  Every lane of the wavefront takes part and gets the same answer.
__device__ __forceinline__ bool w8_find(const W8Args& a, int BM, int t, W8Tile& out) {
    if (a.offsets == nullptr) {
        out.expert = 0;
        out.first = t * BM;
        out.rows = min(BM, a.rows - out.first);
        return out.rows > 0;
    }
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = min(e0 + lane, a.experts);
        const int lo = min(max(a.offsets[e], 0), a.rows), hi = min(max(a.offsets[min(e + 1, a.experts)], lo), a.rows);
        const int tiles = (hi - lo + BM - 1) / BM, sum = wave_sums(tiles);
        const uint64_t past = __ballot(sum > t);
        if (past != 0) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int at = t - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(tiles, l));   // which of the expert's tiles
            const int s = __builtin_amdgcn_readlane(lo, l), n = __builtin_amdgcn_readlane(hi, l) - s;
            out.expert = e0 + l;
            out.first = s + at * BM;
            out.rows = min(BM, n - at * BM);
            return true;
        }
        t -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The rows of X and Y of row i of a tile: -1 where the plan's entry is none.
__device__ __forceinline__ void w8_rows(const W8Args& a, const W8Tile& tile, int i, int& xr, int& yr) {
    const int at = tile.first + i;
    xr = yr = at;
    if (a.offsets == nullptr) return;
    const int slot = a.order[at];
    const bool ok = slot >= 0 && slot < a.rows;
    xr = !ok ? -1 : a.x_sorted ? at : slot / a.top_k;
    yr = !ok ? -1 : a.y_sorted ? at : slot;
}

// y of a finished sum: the same operations in every kernel, so that the choice of one moves no bit.
__device__ __forceinline__ float w8_value(int32_t sum, float xs, float ws, float bias) {
    return __builtin_fmaf((float)sum * xs, ws, bias);
}

// The activations, without the cancellation of 1 - 1 at negative x.
// v_exp_f32 and v_rcp_f32 are off by 1 ulp; the exponent's rounding adds |x| 2^-24.  -infinity times 0 is NaN, as in the formulas.
__device__ __forceinline__ float w8_act(int act, float x) {
    switch (act) {
    case LAVA_HIP_ACT_RELU: return x < 0.f ? 0.f : x;   // NaN stays
    case LAVA_HIP_ACT_SILU: return x * __builtin_amdgcn_rcpf(1.f + epi_exp(-x));
    case LAVA_HIP_ACT_GELU_TANH:   // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
        return x * __builtin_amdgcn_rcpf(1.f + epi_exp(-1.5957691216057308f * __builtin_fmaf(0.044715f * x * x, x, x)));
    case LAVA_HIP_ACT_GELU_ERF: {
        // x Phi(x); Phi(-a) is e / 2, e = erfc(a / sqrt 2) = 2^-E, E = a (log2(e) / 2 a + G), where G = -log2(erfcx(a / sqrt 2)) / a is a
        // polynomial in t - 1, t = 1 / (1 + 0.184 a), fitted by weighted least squares for a up to 14.5, behind which e is below the least
        // float.  As the exponent is a product with a, the roundings of t vanish with a.  At most 3.5 + 6 a + 1.5 a^2 half steps off at
        // x = -a, and less above zero.  Measured half steps, here / 0.5 x erfcf(-x / sqrt 2): |x| < 1 4.2 / 4.9, -3 .. -1 12.6 / 14.6, -6 .. -3
        // 35 / 48.  (erfcf: a layer of 19350 rows x 2048 x 128 98 us against 68.)
        const float a = fabsf(x), t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.184f, 1.f)), s = t - 1.f;
        float g = 0.47620046f;
        g = __builtin_fmaf(g, s, 1.2415534f);
        g = __builtin_fmaf(g, s, 1.1321958f);
        g = __builtin_fmaf(g, s, -0.012980224f);
        g = __builtin_fmaf(g, s, -0.54390675f);
        g = __builtin_fmaf(g, s, 0.12553921f);
        g = __builtin_fmaf(g, s, 1.4246567f);
        g = __builtin_fmaf(g, s, 1.1511052f);
        const float e = __builtin_amdgcn_exp2f(-(__builtin_fmaf(a, 0.72134752f, g) * a));
        return x * (x > 0.f ? __builtin_fmaf(e, -0.5f, 1.f) : 0.5f * e);
    }
    default: return x;
    }
}

__device__ __forceinline__ void w8_act4(int act, float (&v)[4]) {
    switch (act) {   // uniform: one branch for the four
    case LAVA_HIP_ACT_NONE: return;
#define LAVA_W8_ACT(A)                                            \
    case A:                                                       \
        _Pragma("unroll") for (int r = 0; r < 4; ++r) v[r] = w8_act(A, v[r]); \
        return;
        LAVA_W8_ACT(LAVA_HIP_ACT_RELU)
        LAVA_W8_ACT(LAVA_HIP_ACT_SILU)
        LAVA_W8_ACT(LAVA_HIP_ACT_GELU_TANH)
        LAVA_W8_ACT(LAVA_HIP_ACT_GELU_ERF)
#undef LAVA_W8_ACT
    }
}

// `left` columns of a row of Y, at most C (4 or 8), from element offset `at` on, of any alignment.
template <typename T, int C>
__device__ __forceinline__ void w8_put(const W8Args& a, int64_t at, int left, const float (&v)[C]) {
    typedef T Tv __attribute__((ext_vector_type(C)));
    typedef Tv Tvu __attribute__((aligned(sizeof(T))));
    T* p = static_cast<T*>(a.y) + at;
    if (left >= C) {
        Tv o;
#pragma unroll
        for (int r = 0; r < C; ++r) o[r] = narrow<T>(v[r]);
        __builtin_nontemporal_store((Tvu)o, reinterpret_cast<Tvu*>(p));
    } else {
#pragma unroll
        for (int r = 0; r < C; ++r)
            if (r < left) p[r] = narrow<T>(v[r]);
    }
}
template <int C>
__device__ __forceinline__ void w8_store(const W8Args& a, int64_t at, int left, const float (&v)[C]) {
    if (a.y_dtype == LAVA_HIP_F32) w8_put<float, C>(a, at, left, v);
    else if (a.y_dtype == LAVA_HIP_F16) w8_put<f16, C>(a, at, left, v);
    else w8_put<bf16, C>(a, at, left, v);
}

// 8 columns of a row of Y from their sums (of a gated layer the gates' and, 16 places on, the factors').
template <bool GATED>
__device__ __forceinline__ void w8_finish8(int act, const i32x4* sums, float xs, const f32x4* ws, const f32x4* bs, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const i32x4 g = sums[h];
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = w8_value(g[r], xs, ws[h][r], bs[h][r]);
        w8_act4(act, o);
        if constexpr (GATED) {
            const i32x4 u = sums[4 + h];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] *= w8_value(u[r], xs, ws[2 + h][r], bs[2 + h][r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[4 * h + r] = o[r];
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t w8_buffer(const int8_t* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p), 0, (int)bytes, 0x00020000);
}
// 16 bytes at voff + soff; STREAM: with the nontemporal hint, for what is read once
template <bool STREAM>
__device__ __forceinline__ i32x4 w8_load(__amdgpu_buffer_rsrc_t r, uint32_t voff, int soff) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, STREAM ? 2 : 0));
}

// lo and hi: whole 128-byte lines of K of 8 channels each, lane l channel l % 8, bytes 16 (l / 8).  An MFMA's lane l has
// channel l % 16 and 16 bytes of K, whichever they are, as X's lanes have the same: here those at 32 (l / 16) in v0 and the next
// 16 in v1, for which lanes 8 .. 15 of each 16 of lo change places with 0 .. 7 of hi.
__device__ __forceinline__ void w8_whole_lines(const i32x4& lo, const i32x4& hi, i32x4& v0, i32x4& v1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        v0[r] = __builtin_amdgcn_update_dpp(lo[r], hi[r], 0x128, 0xf, 0xc, false);   // row_ror:8 into lanes 8 .. 15
        v1[r] = __builtin_amdgcn_update_dpp(hi[r], lo[r], 0x128, 0xf, 0x3, false);
    }
}

// Row tiles of BM rows that a grid has to hold.
inline int64_t w8_row_tiles(const W8Args& a, int BM) {
    if (a.offsets == nullptr) return ((int64_t)a.rows + BM - 1) / BM;
    return (int64_t)a.rows / BM + (a.experts < a.rows ? a.experts : a.rows);
}

// Whether X and w can be read 16 bytes at a time.
inline bool w8_chunks_fit(const W8Args& a) {
    return a.k % 16 == 0 && a.ldx % 16 == 0 && a.ldw % 16 == 0 && (a.experts == 1 || a.expert_stride % 16 == 0) && aligned(a.x, 16) &&
           aligned(a.w, 16);
}

// Offsets from the buffers' bases are 32-bit: the rows of a tile, or all tokens where they are gathered, and the channels of
// a tile have to span less than 2 GiB.
inline bool w8_spans_fit(const W8Args& a, int rows, int channels) {
    const bool gather = a.offsets != nullptr && !a.x_sorted;
    const int64_t lim = (int64_t)1 << 31, xrows = gather ? a.rows / a.top_k : rows;
    return a.ldx < lim && a.ldw < lim && xrows * a.ldx < lim && channels * a.ldw < lim;
}

// Whether a launch holds the tiles of bm rows and bn columns of Y: fewer than 2^32 threads.
inline bool w8_launch_fits(const W8Args& a, int bm, int bn, int threads) {
    return w8_row_tiles(a, bm) <= 0xffffffffll / threads / (((int64_t)a.n_out + bn - 1) / bn);
}

int launch_w8_generic(const W8Args& a, hipStream_t s);
// Few rows (w8a8_stream.hip).
bool w8_stream_fits(const W8Args& a);
bool w8_stream_preferred(const W8Args& a);
int launch_w8_stream(const W8Args& a, hipStream_t s);
// Tiles (w8a8_tile.hip): 64 x 64, 64 x 128, 128 x 128, 128 x 256 and 256 x 256 rows and channels; the one to take, -1 if none fits;
// how many a call has (of a plan: is likely to have); the experts that are likely to have rows (w8_met).
constexpr int W8_TILE_KINDS = 5;
bool w8_tile_fits(const W8Args& a, int tile);
int w8_tile_choice(const W8Args& a);
double w8_tile_count(const W8Args& a, int bm, int bn);
double w8_met(const W8Args& a);
int launch_w8_tile(const W8Args& a, int tile, hipStream_t s);

// The checks of a plan (moe.hip); write: one that a call writes.
int check_plan(const char* name, const lava_hip_moe_plan* plan, bool write);

}  // namespace lava
