// paged_attn.hpp -- what the attention kernels over the paged cache share (internal).
//
// A query at position i and a key at position j score s = scale q.k, capped (cap tanh(s / cap)), less
// slope |i - j|, and are kept for j in one interval [lo, hi] of the query's: causal, window, bidirectional
// prefix and the sequence's end all narrow it, so every kernel masks by one comparison of a row's own
// two bounds.  Scores are in base 2 throughout (times log2 e).
//
// A sequence's keys come from up to two sources: the batch's shared prefix (positions 0 .. P - 1) and its own
// pages (positions P ..).
#pragma once
#include "paged.hpp"

namespace lava {

struct PaParams {
    PagedCache c;
    PagedBatch b;
    const void* Q;
    void* O;
    float* lse;
    int64_t qsh, qst, osh, ost;   // head and token strides
    int Hq, G;                    // query heads of the call (a token's rows of lse, row_o), those of a key head
    int o16;                      // O and its strides allow 16-byte stores
    FastDiv by_g;
    float mul;                    // scores to base 2; with a cap to 2 log2(e) s / cap
    float cap2;                   // cap log2(e), or 0
    float near, a[5];             // with a cap: |q.k| up to which pa_cap_near holds (-1: none), and its coefficients
    int causal, window;
    const float* slopes;
    const int* bidir;
    const int* ppages;            // the shared prefix's pages
    int P;                        // its length, 0: none
    // how the work is shared out (paged_plan.hpp)
    int row_limit;                // the tile kernel takes the sequences of more rows (new tokens times G)
    int whole;                    // and never splits them
    int stack;                    // the prefix is attended once, by the rows of many sequences together: 1 by the row
                                  // kernel beside the sequences, 2 by the tile kernel in a launch of its own
    FastDiv by_rows, by_tiles;    // workgroups of the row kernel's launch, of the tile kernel's that split
    // a launch's workspace: partial sums [workgroup][2 rows of a tile][DP], their (maximum, weight), arrivals of a tile's
    // parts at the workgroup it starts in (zero between calls)
    float* ws_o;
    float2* ws_ml;
    unsigned* ws_count;
    struct PaOpen* ws_open;       // per workgroup: the tile that starts in its share and leaves it
    // stack: the same for the prefix's launch, and rows' whole results [prefix, own][T * Hq][DP]
    float* pre_o;
    float2* pre_ml;
    float* row_o;
    float2* row_ml;
};

// A row tile in parts: those of the workgroup that keeps this and of the ones behind it (0: none).
struct PaOpen {
    int parts, live, row0, first, head;   // its rows, the first of them in the sequence, the sequence's first token, the key head
};

struct PaRange {
    int lo, hi;   // positions of the keys a query sees
};
// Leading keys that every query of sequence b sees (not less than 0: the last one's position follows from it).
__device__ __forceinline__ int pa_leading(const PaParams& p, int b) { return p.bidir && b >= 0 ? max(p.bidir[b], 0) : 0; }
// A query at position pos of a sequence whose last key is at end - 1.
__device__ __forceinline__ PaRange pa_range(const PaParams& p, int pos, int end, int bid) {
    const int hi = p.causal ? min(max(pos, bid - 1), end - 1) : end - 1;
    return {p.window > 0 ? max(0, pos - p.window + 1) : 0, hi};
}

// The capped score in base 2: cap tanh(z) = cap (1 - 2 / (1 + e^2z)), with x = 2 z log2 e: +-cap where e^2z leaves the range.
// Off by up to 2^-21 of the cap, not of the score: 2^-14 at PA_CAP_SMALL, of a size with a score's 32-bit sum; a larger cap's
// small scores take pa_cap_near.
__device__ __forceinline__ float pa_cap(float x, float cap2) {
    return fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x)), cap2);
}

// The capped score in base 2 from a product |q.k| <= near, where |scale q.k / cap| <= 1/2: an odd polynomial, coefficients with the
// least maximum error (3e-9 of the cap, from a fit to tanh on [0, 1/2]).  Six multiply-adds against the exponential, the
// reciprocal and three more that the whole range takes: a tile of scores that all lie there, as those of most do, costs two thirds.
__device__ __forceinline__ float pa_cap_near(float s, const float (&a)[5]) {
    const float u = s * s;
    return s * fmaf(fmaf(fmaf(fmaf(a[4], u, a[3]), u, a[2]), u, a[1]), u, a[0]);
}
// Caps in base 2 up to which the exact form alone serves scores of any size.
constexpr float PA_CAP_SMALL = 128.f;
// Scores of any size, each by the form that is right to its own last places.
__device__ __forceinline__ float pa_cap_each(float s, float exact, float near, const float (&a)[5]) {
    return fabsf(s) <= near ? pa_cap_near(s, a) : exact;
}

constexpr float PA_LN2 = 0.69314718055994530942f;
constexpr float PA_LOG2E = 1.44269504088896340736f;

// What a call runs, from what the host knows: sizes, not the lengths on the device.
struct PaShape {
    int dp;               // the head dimension rounded up to 64, 128 or 256
    int nr;               // row kernel: 16 nr rows a tile; 0: no launch
    unsigned row_grid;
    int qh;               // tile kernel: 128 qh rows a tile; 0: no launch for sequences
    int pre_qh;           // the stacked prefix's launch of the tile kernel; 0: none
    int heads;            // key heads a pass over these launches; 0: not even one, the generic kernel
    size_t count_bytes, bytes;   // workspace: arrivals, all of it
};
int paged_rows_launch(const PaParams& p, const PaShape& sh, int dtype, hipStream_t s);
bool paged_tile_takes(const PaParams& p);
int paged_tile_launch(const PaParams& p, int qh, bool prefix, int dtype, hipStream_t s);

constexpr int PA_CUS = 256;
constexpr int PR_BK = 128;                       // the row kernel's blocks of keys
constexpr int PT_BK = 64;                        // the tile kernel's
constexpr unsigned PT_LEAST = 8;                  // blocks of a workgroup that splits: what writing and reading a part's bytes costs
constexpr int PT_SPLIT = 20;                     // blocks' time that splitting its tiles costs, about
constexpr unsigned PA_MAX_GRID = 768;            // workgroups that leave parts
constexpr unsigned PT_GRID = PA_CUS;             // those of the tile kernel

}  // namespace lava
