// paged.hpp -- the paged key/value cache: descriptors as the kernels take them, host checks (internal).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "lava_coopmat.hpp"
#include "lava_hip_internal.hpp"

namespace lava {

// n / d for 0 <= n < 2^31 by a multiplication (round-up method: mul = ceil(2^(31 + s) / d) with
// s = ceil(log2 d), so mul d - 2^(31 + s) < 2^s and the quotient is exact over 31 bits).
struct FastDiv {
    uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while (((uint64_t)1 << s) < d) ++s;
    const uint64_t p = (uint64_t)1 << (31 + s);
    return {d, (uint32_t)((p + d - 1) / d), 31 + s};
}
__host__ __device__ __forceinline__ uint32_t div_of(uint32_t n, const FastDiv& f) {
    return (uint32_t)(((uint64_t)n * f.mul) >> f.shift);
}

// A launch of n workgroups: HIP takes fewer than 2^32 threads in a dimension, and of more it runs what is left modulo that,
// without an error.  Up to 2^22 workgroups (of up to 512 threads) lie in x, what is above in y; workgroups
// from n on, where y rounds up, find nothing to do.
constexpr uint32_t PG_GRID_X = 1u << 22;
inline dim3 pg_grid(int64_t n) {
    return n <= PG_GRID_X ? dim3((unsigned)n) : dim3(PG_GRID_X, (unsigned)((n + PG_GRID_X - 1) / PG_GRID_X));
}
__device__ __forceinline__ uint32_t pg_block() { return blockIdx.y * PG_GRID_X + blockIdx.x; }

struct PagedCache {
    void* k;
    void* v;
    int64_t sl, sh, sp;   // elements between tokens, heads, pages
    int D, page, heads;
    int pages;
    FastDiv by_page;
};

struct PagedBatch {
    const int* q_start;
    const int* kv_len;
    const int* table;
    int B, max_pages, T;
    int kv_max;           // max_pages * page: a longer kv_len is cut to it
};

// Rows [first, first + n) and cached tokens of sequence b, cut to what the buffers hold.
struct PagedSeq {
    int first, n, kv;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& p, int b) {
    const int s = min(max(p.q_start[b], 0), p.T), e = min(max(p.q_start[b + 1], s), p.T);
    return {s, e - s, min(max(p.kv_len[b], 0), p.kv_max)};
}

// The sequence that row t belongs to, found by one wavefront together: the first whose end lies
// behind t (sequences without rows end where they start).  B or more: none.
__device__ __forceinline__ int paged_find(const PagedBatch& p, int t, int lane) {
    int got = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const bool before = b0 + lane < p.B && min(p.q_start[b0 + lane + 1], p.T) <= t;
        const int n = __popcll(__builtin_amdgcn_ballot_w64(before));
        got += n;
        if (n < 64) break;
    }
    return __builtin_amdgcn_readfirstlane(got);
}

// Checks of the descriptors, before any GPU call; `fn` names the entry point in messages.
int paged_check(const char* fn, const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch, PagedCache* c,
                PagedBatch* b);
// An (E, H, T) tensor's strides: the head dimension contiguous, heads and tokens at least a head apart.
int paged_check_strides(const char* fn, const char* what, const int64_t* st, int64_t D, int64_t heads, int64_t tokens);
// With several GPUs: `stream` and `ptr` belong to the current one.
int paged_check_device(const char* fn, const void* ptr, void* stream);

}  // namespace lava
