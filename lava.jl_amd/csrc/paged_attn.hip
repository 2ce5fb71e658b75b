// paged_attn.hip -- attention over the paged cache: checks, choice of kernel, and the generic kernel.
//
//  * paged_rows_kernel (paged_attn_rows.hip): rows of a sequence's queries and heads that share a key head,
//    the work split evenly along the keys over the whole chip;
//  * paged_tile_kernel (paged_attn_tile.hip): tiles of 128 or 256 such rows, for prompts;
//  * paged_any_kernel: any head dimension, page size, strides and alignment; one wavefront a query and head.
#include "paged_attn.hpp"

#include <algorithm>
#include <cmath>

namespace lava {

int paged_check(const char* fn, const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch, PagedCache* c,
                PagedBatch* b) {
    LAVA_ARG(cache && batch, "%s: null descriptor", fn);
    LAVA_REQUIRE(cache->dtype == LAVA_HIP_F16 || cache->dtype == LAVA_HIP_BF16, LAVA_HIP_ERR_UNSUPPORTED,
                 "%s: the cache's dtype is %d, not f16 or bf16", fn, cache->dtype);
    LAVA_ARG(cache->head_dim >= 1, "%s: head_dim = %d", fn, cache->head_dim);
    LAVA_REQUIRE(cache->head_dim <= 256, LAVA_HIP_ERR_UNSUPPORTED, "%s: head_dim = %d > 256 is not supported", fn,
                 cache->head_dim);
    LAVA_ARG(cache->page_size >= 1 && cache->heads >= 1 && cache->heads <= 65535,
             "%s: page_size = %d, heads = %d (at least 1; at most 65535 heads)", fn, cache->page_size, cache->heads);
    LAVA_ARG(cache->pages >= 0 && cache->pages <= 0x7fffffff, "%s: pages = %lld", fn, (long long)cache->pages);
    LAVA_ARG(batch->sequences >= 0 && batch->tokens >= 0 && batch->max_pages >= 0 && batch->max_q >= 0,
             "%s: negative extent", fn);
    LAVA_ARG(batch->tokens <= 0x7fffffff, "%s: tokens = %lld is too large", fn, (long long)batch->tokens);
    LAVA_REQUIRE((int64_t)batch->max_pages * cache->page_size <= 0x40000000, LAVA_HIP_ERR_UNSUPPORTED,
                 "%s: a sequence of up to %lld tokens (max_pages * page_size) is longer than 2^30", fn,
                 (long long)batch->max_pages * cache->page_size);
    const int64_t* st = cache->strides;
    LAVA_ARG(st[0] == 1, "%s: the head dimension (E) of the cache must be contiguous", fn);
    const int64_t extent[4] = {cache->head_dim, cache->page_size, cache->heads, cache->pages};
    for (int i = 1; i < 4; ++i) {
        LAVA_ARG(st[i] >= 0 && st[i] <= ((int64_t)1 << 40), "%s: cache stride %d is %lld", fn, i, (long long)st[i]);
        LAVA_ARG(extent[i] <= 1 || st[i] >= cache->head_dim, "%s: cache stride %d smaller than head_dim", fn, i);
    }
    const int64_t span = (cache->page_size - 1) * st[1] + (cache->heads - 1) * st[2] + cache->head_dim;
    LAVA_REQUIRE(st[1] <= 0x3fffffff && st[2] <= 0x3fffffff && span <= 0x3fffffff, LAVA_HIP_ERR_UNSUPPORTED,
                 "%s: a page spans 2^31 bytes or more", fn);
    *c = {cache->k, cache->v, st[1], st[2], st[3], cache->head_dim, cache->page_size, cache->heads,
          (int)cache->pages, fast_div((uint32_t)cache->page_size)};
    *b = {batch->q_start, batch->kv_len, batch->table, batch->sequences, batch->max_pages, (int)batch->tokens,
          batch->max_pages * cache->page_size};
    if (batch->sequences == 0 || batch->tokens == 0) return LAVA_HIP_OK;
    LAVA_ARG(batch->q_start && batch->kv_len && (batch->table || batch->max_pages == 0), "%s: null pointer in the batch", fn);
    LAVA_ARG((cache->k && cache->v) || cache->pages == 0, "%s: null pointer in the cache", fn);
    LAVA_ARG(aligned(batch->q_start, 4) && aligned(batch->kv_len, 4) && aligned(batch->table, 4) && aligned(cache->k, 2) &&
             aligned(cache->v, 2), "%s: misaligned", fn);
    return LAVA_HIP_OK;
}

int paged_check_strides(const char* fn, const char* what, const int64_t* st, int64_t D, int64_t heads, int64_t tokens) {
    LAVA_ARG(st[0] == 1, "%s: %s: the head dimension (E) must be contiguous", fn, what);
    for (int i = 1; i < 3; ++i) {
        LAVA_ARG(st[i] >= 0 && st[i] <= ((int64_t)1 << 40), "%s: %s: stride %d is %lld", fn, what, i, (long long)st[i]);
        LAVA_ARG((i == 1 ? heads : tokens) <= 1 || st[i] >= D, "%s: %s: stride %d smaller than head_dim", fn, what, i);
    }
    return LAVA_HIP_OK;
}

int paged_check_device(const char* fn, const void* ptr, void* stream) {
    static const int devices = [] {
        int n = 0;
        return hipGetDeviceCount(&n) == hipSuccess ? n : 1;
    }();
    if (devices <= 1) return LAVA_HIP_OK;
    int cur = 0;
    LAVA_HIP_TRY(hipGetDevice(&cur));
    if (stream) {
        hipDevice_t dev = 0;
        LAVA_HIP_TRY(hipStreamGetDevice(as_stream(stream), &dev));
        LAVA_ARG(dev == cur, "%s: the stream belongs to device %d, the current device is %d", fn, (int)dev, cur);
    }
    hipPointerAttribute_t at;
    if (ptr && hipPointerGetAttributes(&at, ptr) == hipSuccess)
        LAVA_ARG(at.device == cur, "%s: the cache is on device %d, the current device is %d", fn, at.device, cur);
    else
        (void)hipGetLastError();
    return LAVA_HIP_OK;
}

// One wavefront a row (query and head): 64 keys at a time, a key a lane for the scores, then the head dimension over
// the lanes for the sums.  Masked keys are not read at all.
template <typename T>
__global__ void __launch_bounds__(64) paged_any_kernel(PaParams p) {
    __shared__ float q[256];
    __shared__ float w[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x;
    const int t = (int)(pg_block() / (unsigned)p.Hq), h = (int)(pg_block() % (unsigned)p.Hq), D = p.c.D;
    const int b = paged_find(p.b, t, lane);
    if (b >= p.b.B) return;
    const PagedSeq s = paged_seq(p.b, b);
    if (t < s.first || t >= s.first + s.n) return;
    const int end = p.P + s.kv, pos = end - s.n + (t - s.first), bid = pa_leading(p, b);
    const PaRange r = pa_range(p, pos, end, bid);
    const float slope = p.slopes ? p.slopes[h] * PA_LOG2E : 0.f;
    const T* qr = (const T*)p.Q + (int64_t)t * p.qst + (int64_t)h * p.qsh;
    for (int e = lane; e < D; e += 64) q[e] = (float)qr[e];
    __syncthreads();
    const int64_t head = (int64_t)(h / p.G) * p.c.sh;
    float acc[4] = {}, m = -INFINITY, l = 0.f;
    for (int j0 = r.lo; j0 <= r.hi; j0 += 64) {
        const int j = j0 + lane;
        bool keep = j <= r.hi;
        int64_t o = 0;
        float x = -INFINITY;
        if (keep) {
            const int k = j < p.P ? j : j - p.P;
            const int page_no = (int)div_of((uint32_t)k, p.c.by_page);
            const int page = j < p.P ? p.ppages[page_no] : p.b.table[(int64_t)b * p.b.max_pages + page_no];
            keep = page >= 0 && page < p.c.pages;
            if (keep) {
                o = (int64_t)page * p.c.sp + (int64_t)(k - page_no * p.c.page) * p.c.sl + head;
                const T* kr = (const T*)p.c.k + o;
                float d = 0.f;
                for (int e = 0; e < D; ++e) d = fmaf(q[e], (float)kr[e], d);
                x = d * p.mul;
                if (p.cap2 != 0.f) x = pa_cap_each(d, pa_cap(x, p.cap2), p.near, p.a);
                x -= slope * fabsf((float)(pos - j));
            }
        }
        uint64_t live = __builtin_amdgcn_ballot_w64(keep);
        float top = x;
        for (int i = 1; i < 64; i *= 2) top = fmaxf(top, __shfl_xor(top, i, 64));
        const float mn = fmaxf(m, top), sub = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - sub);   // m = -inf: 0
        const float e1 = keep ? __builtin_amdgcn_exp2f(x - sub) : 0.f;
        __syncthreads();   // the round before has read w and at
        w[lane] = e1;
        at[lane] = o;
        __syncthreads();
        float sum = e1;
        for (int i = 1; i < 64; i *= 2) sum += __shfl_xor(sum, i, 64);
        l = l * alpha + sum;
        m = mn;
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] *= alpha;
        for (; live; live &= live - 1) {
            const int i = __builtin_ctzll(live);
            const T* vr = (const T*)p.c.v + at[i];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (lane + 64 * u < D) acc[u] = fmaf(w[i], (float)vr[lane + 64 * u], acc[u]);
        }
    }
    T* orow = (T*)p.O + (int64_t)t * p.ost + (int64_t)h * p.osh;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < D) orow[lane + 64 * u] = (T)(acc[u] * inv);
    if (p.lse && lane == 0) p.lse[(int64_t)t * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * PA_LN2;
}

// What both attention entry points check and fill in.  *done: there is nothing to compute.
static int pa_prepare(const char* fn, const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch,
                      const lava_hip_attn_score* score, int64_t q_heads, PaParams* p, bool* done) {
    *done = true;
    int rc = paged_check(fn, cache, batch, &p->c, &p->b);
    if (rc != LAVA_HIP_OK) return rc;
    // a position is at least its sequence's length less 2^30 then, and itself, less a window (shorter than the table and the
    // prefix) or a key's position fits 32 bits
    LAVA_REQUIRE(p->b.T <= 0x40000000, LAVA_HIP_ERR_UNSUPPORTED, "%s: tokens = %d are more than 2^30", fn, p->b.T);
    LAVA_ARG(q_heads >= 0 && q_heads <= 65535, "%s: q_heads = %lld is outside [0, 65535]", fn, (long long)q_heads);
    LAVA_ARG(q_heads % p->c.heads == 0, "%s: %lld query heads are not a multiple of the cache's %d", fn,
             (long long)q_heads, p->c.heads);
    if (score) {
        LAVA_ARG(std::isfinite(score->scale) && std::isfinite(score->cap), "%s: scale or cap is not finite", fn);
        LAVA_ARG(score->cap >= 0.f, "%s: cap = %g is negative", fn, score->cap);
        LAVA_ARG(score->window >= 0, "%s: window = %d is negative", fn, score->window);
        LAVA_ARG(aligned(score->slopes, 4) && aligned(score->bidirectional, 4), "%s: slopes or bidirectional misaligned", fn);
        LAVA_ARG(!score->bidirectional || score->causal, "%s: bidirectional keys need a causal call", fn);
        p->cap2 = std::min(score->cap * PA_LOG2E, 1e38f);   // the exact form's 2 cap2 stays finite
        p->mul = score->cap > 0.f ? (float)(2.0 * score->scale / score->cap * 1.4426950408889634) : (float)(score->scale * 1.4426950408889634);
        LAVA_ARG(std::isfinite(p->mul), "%s: scale / cap overflows", fn);
        if (score->cap > 0.f) {
            // tanh(z) = z (c0 + c1 z^2 + ..) for |z| <= 1/2, z = q.k scale / cap
            const double c[5] = {0.9999999316221511, -0.33332776175690243, 0.13320570647011903, -0.052762128916049526,
                                 0.01673756352440004};
            const double z = (double)score->scale / score->cap;
            double power = (double)score->cap * 1.4426950408889634 * z, reach = 0.5;
            for (int i = 0; i < 5; ++i, power *= z * z) {
                p->a[i] = (float)(c[i] * power);
                // a coefficient that 32 bits do not hold to its last places: only scores that do without its term, below 2^-26 of them
                if (i > 0 && std::fabs(p->a[i]) < 0x1p-126f) reach = std::min(reach, std::pow(0x1p-26 / std::fabs(c[i]), 0.5 / i));
            }
            p->near = (float)std::min(reach / std::fabs(z), 1e15);   // u = s^2 stays in range
            // powers of a large scale / cap leave 32 bits: then the exact form always
            for (int i = 0; i < 5; ++i)
                if (!std::isfinite(p->a[i])) p->near = -1.f;
        }
        p->causal = score->causal != 0;
        p->window = score->window;
        p->slopes = score->slopes;
        p->bidir = score->bidirectional;
    }
    p->Hq = (int)q_heads;
    p->G = (int)(q_heads / p->c.heads);
    if (p->b.T == 0 || p->b.B == 0 || q_heads == 0) return LAVA_HIP_OK;
    p->by_g = fast_div((uint32_t)p->G);
    *done = false;
    return LAVA_HIP_OK;
}

// Rows (queries times heads of a key head) that a sequence has at most, as far as the host knows.
static int64_t pa_max_rows(const PaParams& p, const lava_hip_kv_batch* batch) {
    const int64_t q = batch->max_q > 0 && batch->max_q < p.b.T ? batch->max_q : p.b.T;
    return q * p.G;
}

// Whether the cache allows 16-byte reads of 8 keys in one page (and rows, rounded up to tiles, fit 31 bits).
static bool pa_vectors(const PaParams& p) {
    return (int64_t)p.b.T * p.G <= 0x7fffff00 && p.c.D % 8 == 0 && p.c.page % 8 == 0 && p.c.sl % 8 == 0 && p.c.sh % 8 == 0 && p.c.sp % 8 == 0 &&
           aligned(p.c.k, 16) && aligned(p.c.v, 16);
}

// Sequences of more rows (new tokens times the query heads of a key head) run on the tile kernel, of fewer on the row
// kernel.  (us, row / tile kernel: 16 x 17 tokens of 4 heads over 2000 keys, 68 rows 75 / 44; 8 x 32 over 3000, 128 rows 69 / 48; one of
// 16 over 2000, 64 rows 30 / 33.)
constexpr int PA_TILE_ROWS = 32;
// Behind a shared prefix those of more rows, which fill a tile by themselves, read it by themselves.  (us, together / by
// themselves; 8 sequences, 4 heads a key head, up to 300 keys behind 1024 and behind 8192: 260 rows each 64 / 31 and 129 / 132, 384 78 / 32
// and 164 / 140; 128 rows 56 / 31 and 79 / 81, 252 64 / 32 and 116 / 110: behind a short prefix fewer would do.)
constexpr int PA_SHARE_ROWS = 256;
// Rows of a stacked prefix up to which its tiles have 128 rows: two of 256 would leave CUs without a part and cost more each.  (us
// behind 1024 and 8192, 256 / 128 rows a tile: 40 rows 35 / 29 and 40 / 35, 256 40 / 34 and 51 / 40, 320 48 / 42 and 56 / 58, 384
// 48 / 42 and 56 / 59, 640 59 / 53 and 82 / 80, 1024 73 / 66 and 93 / 99.)
constexpr int PA_PREFIX_ROWS = 320;
constexpr size_t PA_ALIGN = 256;

// Rows a tile of the tile kernel: 128 take 0.6 of the time of 256 (a fragment read feeds one product, not two), so they pay
// where tiles of 256 would be half empty, or too few for the CUs and over short keys (over long keys the split fills them).
// Measured (us, 256 / 128 rows; 32 heads, 8 key heads, D = 128): one prompt of 256 15.9 / 12.0, 1024 32 / 26, 2048 63 / 61, 4096
// 147 / 189; 4 of 512 24 / 30; 64 tokens over 8000 keys 69 / 44, 256 over 16000 102 / 108, 2 x 512 over 20000 340 / 387.
static int pa_tile_width(const PaParams& p, int64_t sequences) {
    const int64_t rows = (int64_t)p.b.T * p.G;
    const bool few = rows / 256 * p.c.heads < 200 && (int64_t)p.b.kv_max + p.P <= 8192;
    return rows <= 160 * sequences || few ? 1 : 2;
}

// Rows that the workspace holds: of parts, of the stacked prefix's parts, whole ones behind it.
struct PaRows {
    size_t parts, pre, whole;
};
static PaRows pa_rows(const PaParams& p, const PaShape& sh) {
    auto launch = [](size_t grid, size_t rows) { return 2 * grid * rows; };
    return {std::max(launch(sh.row_grid, 16 * sh.nr), launch(PT_GRID, 128 * sh.qh)), launch(PT_GRID, 128 * sh.pre_qh),
            p.stack ? 2 * (size_t)p.b.T * p.Hq : 0};
}

// Key heads a pass: the kernels count a launch's blocks of work (row tiles times the keys' blocks, of as many keys as the table
// has room for) and its workgroups in 31 bits.  Whole tiles need no count of blocks: where even one head has too many, the tile
// kernel does not split.  0: the row kernel's launch, or the prefix's, does not fit with one head.
static int pa_heads_a_pass(PaParams* p, const PaShape& sh) {
    const int64_t most = 0x7fffffff - 1024;   // and what rounding up over the workgroups adds
    const int64_t rows = (int64_t)p->b.T * p->G, seqs = std::min(p->b.B, p->b.T);   // (those with rows)
    auto blocks = [](int64_t keys, int64_t size) { return (keys + size - 1) / size; };
    int64_t work = 1;   // a head's, of the launch that has most
    if (sh.nr) {
        const int64_t R = 16 * sh.nr;
        int64_t tiles = rows / R + seqs;
        if (p->row_limit < 0x7fffffff) tiles = std::min(tiles, seqs * blocks(p->row_limit, R));
        int64_t of_keys = tiles * std::max<int64_t>(1, blocks(p->b.kv_max, PR_BK));
        if (p->stack == 1) of_keys += blocks(rows, R) * blocks(p->P, PR_BK);
        work = std::max(work, of_keys);
    }
    if (sh.pre_qh) work = std::max(work, blocks(rows, 128 * sh.pre_qh) * blocks(p->P, PT_BK));
    if (sh.qh) {
        const int64_t tiles = rows / (128 * sh.qh) + seqs;
        const int64_t of_keys = tiles * std::max<int64_t>(1, blocks(p->b.kv_max, PT_BK) + blocks(p->P, PT_BK));
        if (of_keys > most) p->whole = 1;
        work = std::max(work, p->whole ? tiles : of_keys);
    }
    return (int)std::min<int64_t>(p->c.heads, most / work);
}

// What depends on the call's sizes alone: which kernels take which sequences.
static PaShape pa_plan_call(PaParams* p, int64_t max_rows) {
    const int pin = kernel_override(LAVA_HIP_FAMILY_PAGED);
    PaShape sh = {};
    sh.dp = p->c.D <= 64 ? 64 : p->c.D <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)p->b.T * p->G;
    p->row_limit = 0x7fffffff;
    const int limit = p->P > 0 ? PA_SHARE_ROWS : PA_TILE_ROWS;
    if (paged_tile_takes(*p) && (pin >= 3 || (pin == 0 && max_rows > limit))) {
        sh.qh = pin == 4 ? 1 : pin == 3 ? 2 : pa_tile_width(*p, p->b.B);
        // where the sequences' mean is above the limit the tile kernel takes the short ones too (it reads their keys as
        // fast) rather than a launch for them
        p->row_limit = pin >= 3 || rows > limit * (int64_t)p->b.B ? 0 : limit;
        // tiles enough for the CUs over few keys, or keys fewer than a split costs: never split, so no launch to join parts, 2 to
        // 4 us.  (us, never / as the device finds; prompts of 32 heads on 8: 8 of 1344 tokens 153 / 158, one of 1792 51.5 / 54.0, 4 of
        // 2048 158 / 160; past 32 blocks one of 2176 62.7 / 64.7, 8 352 / 358, 4 of 2560 236 / 238, but over few long keys whole
        // tiles leave CUs idle: 64 tokens behind 8000.)
        const int64_t blocks = ((int64_t)p->b.kv_max + p->P + PT_BK - 1) / PT_BK;
        p->whole = blocks <= PT_SPLIT || (blocks <= 32 && rows / (128 * sh.qh) * p->c.heads >= 128);
    }
    if (p->row_limit > 0) {
        if (p->P > 0) {   // the prefix once for all: beside the sequences, or on the tile kernel for many rows
            const bool many = rows > PA_TILE_ROWS && paged_tile_takes(*p) && pin != 2;
            p->stack = many ? 2 : 1;
            sh.pre_qh = many ? (rows <= PA_PREFIX_ROWS ? 1 : 2) : 0;
        }
        const int64_t most = p->stack == 1 ? rows : std::min<int64_t>(max_rows, p->row_limit);
        sh.nr = most <= 16 ? 1 : 2;
        // as many workgroups as fit (LDS: 512 bytes a column of the head)
        sh.row_grid = (unsigned)(PA_CUS * (sh.dp == 64 ? 3 : sh.dp == 128 ? 2 : 1));
    }
    sh.heads = pa_heads_a_pass(p, sh);
    if (sh.heads == 0 && paged_tile_takes(*p) && pin == 0) {   // more rows and wider tables than the row kernel counts: all on tiles
        sh.qh = 2;
        sh.nr = sh.pre_qh = 0;
        sh.row_grid = 0;
        p->row_limit = p->stack = 0;
        sh.heads = pa_heads_a_pass(p, sh);
    }
    p->by_rows = fast_div(std::max(1u, sh.row_grid));
    p->by_tiles = fast_div(PT_GRID);
    const size_t row = sh.dp * sizeof(float) + sizeof(float2);
    const PaRows n = pa_rows(*p, sh);
    sh.count_bytes = STREAM_WS_RESERVED;
    sh.bytes = sh.count_bytes + (n.parts + n.pre + n.whole) * row + PA_MAX_GRID * sizeof(PaOpen) + 8 * PA_ALIGN;
    return sh;
}

static_assert(STREAM_WS_PAGED + PA_MAX_GRID * sizeof(unsigned) <= STREAM_WS_RESERVED, "the arrivals lie in the reserved part");
static_assert(PT_GRID <= PA_MAX_GRID && 3 * PA_CUS <= PA_MAX_GRID, "every launch's workgroups have a place");

// Lays a workspace out: arrivals at `count`, the rest from `at` on.
static void pa_workspace(PaParams* p, const PaShape& sh, void* count, void* rest) {
    uint8_t* at = (uint8_t*)rest;
    auto take = [&](size_t bytes) {
        at = (uint8_t*)(((uintptr_t)at + PA_ALIGN - 1) & ~(uintptr_t)(PA_ALIGN - 1));
        uint8_t* q = at;
        at += bytes;
        return q;
    };
    const PaRows n = pa_rows(*p, sh);
    p->ws_count = (unsigned*)count;
    p->ws_open = (PaOpen*)take(PA_MAX_GRID * sizeof(PaOpen));
    p->ws_o = (float*)take(n.parts * sh.dp * sizeof(float));
    p->ws_ml = (float2*)take(n.parts * sizeof(float2));
    p->pre_o = (float*)take(n.pre * sh.dp * sizeof(float));
    p->pre_ml = (float2*)take(n.pre * sizeof(float2));
    p->row_o = (float*)take(n.whole * sh.dp * sizeof(float));
    p->row_ml = (float2*)take(n.whole * sizeof(float2));
}

static int pa_launch(const PaParams& call, const PaShape& sh, int dtype, hipStream_t s) {
    int rc = LAVA_HIP_OK;
    for (int h0 = 0; h0 < call.c.heads && rc == LAVA_HIP_OK; h0 += sh.heads) {   // (f16 and bf16: 2 bytes an element)
        PaParams p = call;
        const int64_t q0 = (int64_t)h0 * p.G;
        p.c.heads = std::min(sh.heads, call.c.heads - h0);
        p.c.k = (uint16_t*)p.c.k + h0 * p.c.sh;
        p.c.v = (uint16_t*)p.c.v + h0 * p.c.sh;
        p.Q = (const uint16_t*)p.Q + q0 * p.qsh;
        p.O = (uint16_t*)p.O + q0 * p.osh;
        if (p.lse) p.lse += q0;
        if (p.slopes) p.slopes += q0;
        if (sh.qh) rc = paged_tile_launch(p, sh.qh, false, dtype, s);
        if (rc == LAVA_HIP_OK && sh.pre_qh) rc = paged_tile_launch(p, sh.pre_qh, true, dtype, s);
        if (rc == LAVA_HIP_OK && sh.nr) rc = paged_rows_launch(p, sh, dtype, s);
    }
    return rc;
}

static int pa_attn(const char* fn, const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch,
                   const lava_hip_attn_score* score, const int32_t* ppages, int64_t prefix, const void* Q, void* O,
                   int64_t q_heads, const int64_t* q_strides, const int64_t* o_strides, float* lse, void* stream) {
    PaParams p = {};
    bool done;
    LAVA_ARG(score, "%s: null score", fn);
    int rc = pa_prepare(fn, cache, batch, score, q_heads, &p, &done);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG(prefix >= 0, "%s: prefix_len is negative", fn);
    LAVA_REQUIRE(prefix <= 0x3ffffe00, LAVA_HIP_ERR_UNSUPPORTED, "%s: prefix_len = %lld is longer than 2^30 - 512", fn,
                 (long long)prefix);   // positions and the block behind the last fit 31 bits
    if (done) return LAVA_HIP_OK;
    LAVA_ARG(Q && O && q_strides && o_strides && (ppages || prefix == 0), "%s: null pointer", fn);
    LAVA_ARG(aligned(Q, 2) && aligned(O, 2) && aligned(lse, 4) && aligned(ppages, 4), "%s: misaligned", fn);
    rc = paged_check_strides(fn, "q_strides", q_strides, p.c.D, q_heads, p.b.T);
    if (rc == LAVA_HIP_OK) rc = paged_check_strides(fn, "o_strides", o_strides, p.c.D, q_heads, p.b.T);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_REQUIRE((int64_t)p.b.T * q_heads <= 0x7fffffff, LAVA_HIP_ERR_UNSUPPORTED,
                 "%s: %lld rows (tokens * q_heads) are 2^31 or more", fn, (long long)p.b.T * q_heads);
    rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    rc = paged_check_device(fn, p.c.k, stream);
    if (rc != LAVA_HIP_OK) return rc;
    p.Q = Q;
    p.O = O;
    p.lse = lse;
    p.qsh = q_strides[1];
    p.qst = q_strides[2];
    p.osh = o_strides[1];
    p.ost = o_strides[2];
    p.o16 = aligned(O, 16) && p.osh % 8 == 0 && p.ost % 8 == 0;
    p.ppages = ppages;
    p.P = (int)prefix;
    if (p.window >= (int64_t)p.P + p.b.kv_max) p.window = 0;   // hides nothing (and positions less it stay in 32 bits)
    hipStream_t s = as_stream(stream);
    bool fast = kernel_override(LAVA_HIP_FAMILY_PAGED) != 1 && pa_vectors(p) && aligned(Q, 16) && aligned(O, 8);
    for (int i = 1; i < 3; ++i) fast = fast && q_strides[i] % 8 == 0 && o_strides[i] % 4 == 0;
    const PaShape sh = fast ? pa_plan_call(&p, pa_max_rows(p, batch)) : PaShape{};
    if (sh.heads > 0) {
        if (batch->workspace) {
            LAVA_ARG(batch->workspace_bytes >= sh.bytes, "%s: the workspace of %zu bytes is smaller than the %zu this call needs",
                     fn, batch->workspace_bytes, sh.bytes);
            LAVA_ARG(aligned(batch->workspace, 16), "%s: misaligned workspace", fn);
            pa_workspace(&p, sh, batch->workspace, (uint8_t*)batch->workspace + sh.count_bytes);
            return pa_launch(p, sh, cache->dtype, s);
        }
        return with_stream_workspace(sh.bytes, stream, [&](void* ws) {
            pa_workspace(&p, sh, (uint8_t*)ws + STREAM_WS_PAGED, (uint8_t*)ws + sh.count_bytes);
            return pa_launch(p, sh, cache->dtype, s);
        });
    }
    if (cache->dtype == LAVA_HIP_F16)
        hipLaunchKernelGGL((paged_any_kernel<f16>), pg_grid((int64_t)p.b.T * p.Hq), dim3(64), 0, s, p);
    else
        hipLaunchKernelGGL((paged_any_kernel<bf16>), pg_grid((int64_t)p.b.T * p.Hq), dim3(64), 0, s, p);
    LAVA_LAUNCH_CHECK("paged_any_kernel");
    return LAVA_HIP_OK;
}

}  // namespace lava

using namespace lava;

extern "C" int lava_hip_paged_attn(const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch,
                                   const lava_hip_attn_score* score, const void* Q, void* O, int64_t q_heads,
                                   const int64_t* q_strides, const int64_t* o_strides, float* lse, void* stream) {
    return pa_attn("paged_attn", cache, batch, score, nullptr, 0, Q, O, q_heads, q_strides, o_strides, lse, stream);
}

extern "C" int lava_hip_shared_prefix_attn(const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch,
                                           const lava_hip_attn_score* score, const int32_t* prefix_pages,
                                           int64_t prefix_len, const void* Q, void* O, int64_t q_heads,
                                           const int64_t* q_strides, const int64_t* o_strides, float* lse, void* stream) {
    LAVA_REQUIRE(!score || !score->bidirectional, LAVA_HIP_ERR_UNSUPPORTED,
                 "shared_prefix_attn: bidirectional keys are not taken with a shared prefix");
    return pa_attn("shared_prefix_attn", cache, batch, score, prefix_pages, prefix_len, Q, O, q_heads, q_strides,
                   o_strides, lse, stream);
}

extern "C" int lava_hip_paged_workspace_bytes(const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch,
                                              int64_t q_heads, int64_t prefix_len, size_t* bytes) {
    PaParams p = {};
    bool done;
    LAVA_ARG(bytes, "paged_workspace_bytes: null pointer");
    LAVA_ARG(prefix_len >= 0, "paged_workspace_bytes: prefix_len is negative");
    const int rc = pa_prepare("paged_workspace_bytes", cache, batch, nullptr, q_heads, &p, &done);
    if (rc != LAVA_HIP_OK) return rc;
    *bytes = 0;
    if (done) return LAVA_HIP_OK;
    p.P = (int)std::min<int64_t>(prefix_len, 0x3ffffe00);
    if (!pa_vectors(p)) return LAVA_HIP_OK;
    // whatever Q's and O's strides are: with those that the tile kernel takes, and without
    for (const int64_t stride : {(int64_t)0, (int64_t)1 << 40}) {
        PaParams q = p;
        q.qst = stride;
        const PaShape sh = pa_plan_call(&q, pa_max_rows(q, batch));
        if (sh.heads > 0) *bytes = std::max(*bytes, sh.bytes);
    }
    return LAVA_HIP_OK;
}
