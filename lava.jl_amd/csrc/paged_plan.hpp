// paged_plan.hpp -- how the paged attention kernels share out their work, and join its parts (device side, internal).
//
// Work is counted in blocks of BK keys: (sequence, key head, row tile, block), flattened in that order.  A launch of n
// workgroups cuts it into n equal parts; lengths are on the device, so every wavefront finds its workgroup's part
// itself, by one scan over the sequences.  A part is a run of segments, each some blocks of one row tile.  A
// segment of all of its tile's blocks gives the result; another leaves (sums, maximum, weight) in the
// workspace -- of a workgroup's segments only the first can continue a tile and only the last can leave one open,
// so two tiles' rows a workgroup hold them -- and a tile's parts are joined in key order, by the last of its
// workgroups to arrive (16 rows) or by a launch of their own (more rows, which would keep one workgroup for long).
#pragma once
#include <algorithm>

#include "paged_attn.hpp"
#include "paged_types.hpp"

namespace lava {

// The kernel's parameters, its first argument, held in two registers' lanes: loaded once, and read back a lane a dword
// where a phase of the kernel needs them.  Kept in scalar registers throughout they spill, and scalar loads of the kernel's
// arguments at each phase, each of which goes to the host's memory, took 2 to 10 us a workgroup.
struct PaArgs {
    uint32_t a, b;   // lane i: dwords i and 64 + i
    __device__ __forceinline__ void load(int lane) {
        constexpr int N = sizeof(PaParams) / 4;
        static_assert(sizeof(PaParams) % 4 == 0 && N > 64 && N <= 128, "two dwords a lane hold the parameters");
        auto q = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
        a = q[lane];
        b = q[64 + min(lane, N - 65)];
    }
    // as read in this phase: not hoisted from the loops around it
    __device__ __forceinline__ PaParams get() {
        constexpr int N = sizeof(PaParams) / 4;
        struct {
            uint32_t d[N];
        } x;
        asm volatile("" : "+v"(a), "+v"(b));
#pragma unroll
        for (int i = 0; i < N; ++i) x.d[i] = (uint32_t)__builtin_amdgcn_readlane((int)(i < 64 ? a : b), i & 63);
        PaParams p = __builtin_bit_cast(PaParams, x);
        global(p.c.k), global(p.c.v), global(p.b.q_start), global(p.b.kv_len), global(p.b.table), global(p.Q), global(p.O);
        global(p.lse), global(p.slopes), global(p.bidir), global(p.ppages), global(p.ws_o), global(p.ws_ml), global(p.ws_count), global(p.ws_open);
        global(p.pre_o), global(p.pre_ml), global(p.row_o), global(p.row_ml);
        return p;
    }
    // says that a pointer made of register contents is to global memory
    template <typename T>
    __device__ __forceinline__ static void global(T*& q) {
        q = (T*)(__attribute__((address_space(1))) T*)(uintptr_t)q;
    }
};

// x, as if newly computed: addresses made from it in one phase of a segment are not hoisted out of the loop over segments,
// where they would take registers from the others.
__device__ __forceinline__ int pa_again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A sequence's (or the stacked prefix's) share: key blocks [p0, p0 + np) of the prefix, then [o0, o0 + nb - np) of its
// own keys, for every row tile and key head.
struct PaSeq {
    int tiles, nb, p0, np, o0;
};

// BK: keys of a block.  ABOVE: the launch takes the sequences of more than row_limit rows (and reads the prefix for each of
// them), else those of at most that many (whose prefix is stacked).  PRE: the call has a shared prefix.
template <int BK, bool ABOVE, bool PRE>
__device__ __forceinline__ PaSeq pa_seq(const PaParams& p, const PagedSeq& s, int R) {
    PaSeq w = {};
    const int rows = s.n * p.G;   // below 2^31, as all rows of the batch are
    if (rows == 0 || (rows > p.row_limit) != ABOVE) return w;
    w.nb = (s.kv + BK - 1) / BK;
    if (p.window > 0 || PRE) {
        const int P = PRE ? p.P : 0, lo = p.window > 0 ? max(0, P + s.kv - s.n - p.window + 1) : 0;   // first position seen
        if (PRE && ABOVE && lo < P) {
            w.p0 = lo / BK;
            w.np = (P + BK - 1) / BK - w.p0;
        }
        const int own = min(max(0, lo - P), s.kv);
        w.o0 = own / BK;
        w.nb = w.np + w.nb - w.o0;
    }
    w.nb = max(1, w.nb);   // rows without keys are written too
    w.tiles = (rows + R - 1) / R;
    return w;
}
// Blocks that the first row tile sees, about: a causal sequence's tiles see more and more.
template <int BK>
__device__ __forceinline__ int pa_first_nb(const PaParams& p, const PagedSeq& s, const PaSeq& w) {
    return p.causal && !p.bidir ? max(1, w.nb - (s.n + BK - 1) / BK) : w.nb;
}
__device__ __forceinline__ uint32_t pa_work(const PaParams& p, const PaSeq& w) {
    return (uint32_t)w.tiles * (uint32_t)w.nb * (uint32_t)p.c.heads;
}

// Scans and reductions over the wavefront by DPP: shifts within 16 lanes, then the last lane of 16 (of 32) to the
// lanes behind it; lanes that receive nothing combine with `id`.  Some 50 cycles, against 700 for six LDS-pipe shuffles, and a
// workgroup starts with several.
template <typename F>
__device__ __forceinline__ int pa_scan_with(int x, int id, F f) {   // inclusive
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x111, 0xf, 0xf, false));   // row_shr 1, 2, 4, 8
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x112, 0xf, 0xf, false));
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x114, 0xf, 0xf, false));
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x118, 0xf, 0xf, false));
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x142, 0xa, 0xf, false));   // row_bcast 15 into rows 1 and 3
    x = f(x, __builtin_amdgcn_update_dpp(id, x, 0x143, 0xc, 0xf, false));   // row_bcast 31 into rows 2 and 3
    return x;
}
__device__ __forceinline__ uint32_t pa_scan(uint32_t x) {
    return (uint32_t)pa_scan_with((int)x, 0, [](int a, int b) { return (int)((uint32_t)a + (uint32_t)b); });
}
__device__ __forceinline__ int pa_wave_max(int x) {
    return __builtin_amdgcn_readlane(pa_scan_with(x, (int)0x80000000, [](int a, int b) { return max(a, b); }), 63);
}
__device__ __forceinline__ int pa_wave_min(int x) {
    return __builtin_amdgcn_readlane(pa_scan_with(x, 0x7fffffff, [](int a, int b) { return min(a, b); }), 63);
}

// What every wavefront knows of the whole call.  The first 64 sequences stay in its lanes.
struct PaPlan {
    uint32_t total;     // blocks of work
    uint32_t upto;      // lane i: those of sequences 0 .. i
    PagedSeq mine;      // lane i: sequence i
    // a call with a shared prefix: its stacked share, in front of the sequences (no tiles: none)
    PaSeq prefix;
    uint32_t pre_work;
    int t0, t1;         // rows of the batch
    bool plain;         // every row sees the whole prefix
    bool falls;         // q_start does
};

__device__ __forceinline__ PagedSeq pa_lane_seq(const PaParams& p, int b) {
    PagedSeq s = {0, 0, 0};
    if (b < p.b.B) s = paged_seq(p.b, b);
    return s;
}

// seqs: the launch takes sequences; prefix: it takes the stacked prefix.
template <int BK, bool ABOVE, bool PRE>
__device__ __forceinline__ PaPlan pa_plan(const PaParams& p, int R, bool seqs, bool prefix, int lane) {
    PaPlan g = {};
    int lo = 0x7fffffff;
    bool plain = p.window == 0, falls = false;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        const PagedSeq s = pa_lane_seq(p, b0 + lane);
        if (b0 + lane < p.b.B) falls = falls || p.b.q_start[b0 + lane + 1] < p.b.q_start[b0 + lane];
        const uint32_t upto = pa_scan(seqs ? pa_work(p, pa_seq<BK, ABOVE, PRE>(p, s, R)) : 0u);
        if (b0 == 0) {
            g.mine = s;
            g.upto = upto;
        }
        if (PRE && s.n > 0) {
            lo = min(lo, p.window > 0 ? max(0, p.P + s.kv - s.n - p.window + 1) : 0);
            plain = plain && s.n <= s.kv;
        }
        g.total += __builtin_amdgcn_readlane(upto, 63);
    }
    if (PRE && prefix) {
        lo = pa_wave_min(lo);
        g.plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
        g.t0 = min(max(p.b.q_start[0], 0), p.b.T);
        g.t1 = min(max(p.b.q_start[p.b.B], g.t0), p.b.T);
        if (lo < p.P && g.t1 > g.t0) {
            g.prefix.p0 = lo / BK;
            g.prefix.np = g.prefix.nb = (p.P + BK - 1) / BK - g.prefix.p0;
            g.prefix.tiles = ((g.t1 - g.t0) * p.G + R - 1) / R;
            g.pre_work = pa_work(p, g.prefix);
        }
        g.total += g.pre_work;
    }
    // sequences that overlap would be more rows than T, whose blocks the host has counted in 31 bits: no work
    if (__builtin_amdgcn_ballot_w64(falls) != 0) {
        g.total = g.pre_work = 0;
        g.falls = true;
    }
    return g;
}

// The segment at block `at` of the work: its sequence (b = -1: the stacked prefix), the work in front of that, and
// what of it the tile and head are.
struct PaSegment {
    int b;
    PagedSeq seq;
    PaSeq sw;
    uint32_t before;
    int head, tile, blk0;
};
template <int BK, bool ABOVE, bool PRE>
__device__ __forceinline__ PaSegment pa_segment(const PaParams& p, const PaPlan& g, int R, uint32_t at, int lane) {
    PaSegment x = {};
    if (PRE && at < g.pre_work) {
        x.b = -1;
        x.seq = {g.t0, g.t1 - g.t0, 0};
        x.sw = g.prefix;
    } else {
        x.before = PRE ? g.pre_work : 0;
        uint32_t upto = g.upto;
        PagedSeq s = g.mine;
        for (int b0 = 0;;) {
            const uint64_t past = __builtin_amdgcn_ballot_w64(x.before + upto > at);
            if (past != 0) {
                const int i = __builtin_ctzll(past);
                if (i > 0) x.before += __builtin_amdgcn_readlane(upto, i - 1);
                x.b = b0 + i;
                x.seq.first = __builtin_amdgcn_readlane(s.first, i);
                x.seq.n = __builtin_amdgcn_readlane(s.n, i);
                x.seq.kv = __builtin_amdgcn_readlane(s.kv, i);
                break;
            }
            x.before += __builtin_amdgcn_readlane(upto, 63);
            b0 += 64;
            if (b0 >= p.b.B) break;   // not reached for at < total
            s = pa_lane_seq(p, b0 + lane);
            upto = pa_scan(pa_work(p, pa_seq<BK, ABOVE, PRE>(p, s, R)));
        }
        x.sw = pa_seq<BK, ABOVE, PRE>(p, x.seq, R);
    }
    const uint32_t rel = at - x.before, ht = rel / (uint32_t)x.sw.nb;
    x.blk0 = __builtin_amdgcn_readfirstlane((int)(rel - ht * (uint32_t)x.sw.nb));
    x.head = __builtin_amdgcn_readfirstlane((int)(x.sw.tiles == 1 ? ht : ht / (uint32_t)x.sw.tiles));
    x.tile = (int)ht - x.head * x.sw.tiles;
    x.tile = __builtin_amdgcn_readfirstlane(x.tile);
    return x;
}

// The tile kernel's choice: tiles one by one, a workgroup each, or the even split over PT_GRID workgroups.  Whole tiles take
// the longest one's time, or the CUs' share and, at the end, half the longest on some; the split takes the share that counts
// a sequence's every tile as long as its last, and PT_SPLIT blocks more (parts written, a launch that joins them).
// tiles_upto: lane i: row tiles of sequences 0 .. i.
template <bool PRE>
__device__ __forceinline__ bool pa_by_tile(const PaParams& p, const PaPlan& g, int R, int lane, int& tiles_upto) {
    int longest = 0;
    uint32_t seen = 0;   // blocks that rows see, about
    tiles_upto = 0;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        const PagedSeq s = b0 == 0 ? g.mine : pa_lane_seq(p, b0 + lane);
        const PaSeq q = pa_seq<PT_BK, true, PRE>(p, s, R);
        longest = max(longest, q.nb);
        seen += q.tiles > 0 ? (uint32_t)q.tiles * (uint32_t)(q.nb + pa_first_nb<PT_BK>(p, s, q)) / 2u * (uint32_t)p.c.heads : 0u;
        if (b0 == 0) tiles_upto = (int)pa_scan((uint32_t)q.tiles);
    }
    if (p.whole) return true;
    longest = pa_wave_max(longest);
    seen = __builtin_amdgcn_readlane(pa_scan(seen), 63);
    return max(longest, (int)(seen / PA_CUS) + longest / 2) <= (int)(g.total / PA_CUS) + PT_SPLIT;
}

// A workgroup's place among `n` (a multiple of 8): consecutive parts on one XCD, which share keys in its L2.
__device__ __forceinline__ uint32_t pa_place(uint32_t n) { return (blockIdx.x & 7) * (n >> 3) + (blockIdx.x >> 3); }
// Blocks a workgroup, at least `least`.
__device__ __forceinline__ uint32_t pa_per(uint32_t total, const FastDiv& n, uint32_t least) {
    return max(least, div_of(total + n.d - 1, n));
}

// The position of row `t` of the batch behind the stacked prefix: of the sequence whose end is the first behind it.
__device__ __forceinline__ int pa_row_pos(const PaParams& p, int t) {
    int a = 0, z = p.b.B;
    while (a < z) {
        const int mid = (a + z) >> 1;
        if (min(p.b.q_start[mid + 1], p.b.T) <= t) a = mid + 1;
        else z = mid;
    }
    if (a >= p.b.B) return p.P;
    const PagedSeq s = paged_seq(p.b, a);
    return p.P + s.kv - s.n + (t - s.first);
}
// Whether rows [t0, t1] of the batch are all of one sequence of more than row_limit rows (whose prefix
// another launch reads).  By a wavefront together.
__device__ __forceinline__ bool pa_other(const PaParams& p, int t0, int t1, int lane) {
    if (p.row_limit == 0x7fffffff) return false;
    const int b = paged_find(p.b, t0, lane);
    if (b >= p.b.B) return true;
    const PagedSeq s = paged_seq(p.b, b);
    return (int64_t)s.n * p.G > p.row_limit && t1 < s.first + s.n;
}

// Where a wavefront's keys are, 8 at a time: its tiles (GPT eights each) 64 / GPT at a time in one register, an eight a lane,
// and the next as many in another.  One load round trip finds them all, and a lane read each gives them back as
// scalars; page numbers by scalar loads in the loop, which LDS reads then wait for, cost 2 us a workgroup's start and 0.3
// a block in the tile kernel.
template <int GPT, bool PRE>
struct PaPages {
    static constexpr int TPC = 64 / GPT;
    // elements from the cache's begin, head 0, of even chunks and of odd ones; -1: no page, or no key.  (Two members: of an array
    // indexed by the chunk the compiler makes LDS, whose place it finds in the dispatch packet, in the host's memory: 2 to 10 us.)
    int64_t even, odd;
    // chunk c.  where(tile, eight, k, pre): the eight's first key of the prefix (pre) or of the sequence; false: past the end
    template <typename F>
    __device__ __forceinline__ void load(const PaParams& p, int b, int c, int lane, F where) {
        int k;
        bool pre;
        int64_t o = -1;
        if (where(c * TPC + lane / GPT, lane % GPT, k, pre)) {
            const int no = (int)div_of((uint32_t)k, p.c.by_page);
            const int* table = p.b.table + (int64_t)max(b, 0) * p.b.max_pages;
            const int pg = PRE && pre ? p.ppages[no] : table[no];
            if ((uint32_t)pg < (uint32_t)p.c.pages) o = (int64_t)pg * p.c.sp + (int64_t)(k - no * p.c.page) * p.c.sl;
        }
        const bool to_odd = (c & 1) != 0;
        even = to_odd ? even : o;
        odd = to_odd ? o : odd;
    }
    __device__ __forceinline__ static int64_t lane_of(int64_t v, int at) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, at);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), at);
        return (int64_t)((uint64_t)hi << 32 | lo);
    }
    __device__ __forceinline__ int64_t get(int tile, int i) const {
        const int at = (tile % TPC) * GPT + i;
        const bool of_odd = ((tile / TPC) & 1) != 0;
        const int64_t a = lane_of(even, at), b = lane_of(odd, at);
        return of_odd ? b : a;
    }
};

// A tile in parts: those of workgroups i0 .. i0 + n - 1 of its launch.
struct PaParts {
    uint32_t i0;
    int n;
};
// a: the tile's first block of work.
__device__ __forceinline__ PaParts pa_parts(uint32_t a, int nb, uint32_t per) {
    const uint32_t i0 = a / per;
    return {i0, (int)((a + (uint32_t)nb - 1) / per - i0) + 1};
}
// The place of row `row` of part j, tiles of R rows: 2 R rows of place a workgroup, of which the tile has those from the second
// half of i0's to the first half of the last one's.  A row's parts lie one behind the other, in one page (part by part they were
// 128 KB apart, and a round trip to sixteen of them took 4 us).
__device__ __forceinline__ int64_t pa_part(const PaParts& t, int j, int row, int R) {
    return ((int64_t)2 * t.i0 + 1) * R + (int64_t)row * t.n + j;
}

// ---- parts ----------------------------------------------------------------------------
// Parts that are joined in the launch that makes them are written and read as device-wide relaxed atomics of 8 bytes: they
// pass the XCDs' L2 caches without a fence that would write those back, and a wait for the stores before the
// arrival is counted orders them.  Parts for a later launch are plain stores.

__device__ __forceinline__ void pa_put(float* p, float a, float b) {
    const float2 v = make_float2(a, b);
    __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_get(const float* p) {
    return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Rows joined by a wavefront, 256 / DP of them at once: DP / 4 lanes a row, 4 columns a lane.  Part j of the lane's row has its
// (maximum, weight) and sums at part(j, ml, o); n parts (at least one).  Sums are requested beside the weights, one round trip for
// both: those of a part of no weight are not written, and what is read of them is dropped.  LIVE: the parts come from
// workgroups of this launch (device-wide loads).
template <int DP, bool LIVE, typename F>
__device__ __forceinline__ void pa_join_rows(int n, F part, int lane, f32x4& o, float& m, float& l) {
    const int most = pa_wave_max(n), c = lane % (DP / 4);
    m = -INFINITY;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    // parts in flight: a round trip to what other workgroups wrote takes 1 to 2 us; 4 where those are all (of places past
    // the last part the last one is read again: 16 for tiles of 2 parts: 40 us, now 17, on 12 chunks behind 777 to 6000 keys)
    auto some_of = [&](int j0, auto in_flight) __attribute__((always_inline)) {
        constexpr int U = decltype(in_flight)::value;
        float2 x[U];
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float2* ml;
            const float* q;
            part(min(j0 + u, n - 1), ml, q);
            q += 4 * c;
            if constexpr (LIVE) {
                x[u] = pa_get((const float*)ml);
                const float2 a = pa_get(q), b = pa_get(q + 2);
                v[u] = f32x4{a.x, a.y, b.x, b.y};
            } else {
                x[u] = *ml;
                v[u] = *reinterpret_cast<const f32x4*>(q);
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // all requests before the first use
        float top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j0 + u >= n) x[u] = make_float2(-INFINITY, 0.f);
            top = fmaxf(top, x[u].x);
        }
        const float sub = top == -INFINITY ? 0.f : top, a = __builtin_amdgcn_exp2f(m - sub);
        m = top;
        l *= a;
        o *= a;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float f = __builtin_amdgcn_exp2f(x[u].x - sub);
            l = fmaf(f, x[u].y, l);
            const bool some = x[u].y != 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = some ? fmaf(f, v[u][e], o[e]) : o[e];
        }
    };
    if (most <= 4) {
        some_of(0, pg_int<4>{});
    } else {
        for (int j0 = 0; j0 < most; j0 += 16) some_of(j0, pg_int<16>{});
    }
}

template <typename T, int DP>
__device__ __forceinline__ void pa_store_row(const PaParams& p, int t, int h, f32x4 o, float m, float l, int lane) {
    const int d = 4 * (lane % (DP / 4));
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typedef T v4 __attribute__((ext_vector_type(4)));
    if (d < p.c.D) {   // D is a multiple of 8
        const v4 v = {(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
        *reinterpret_cast<v4*>((T*)p.O + (int64_t)t * p.ost + (int64_t)h * p.osh + d) = v;
    }
    if (p.lse && d == 0) p.lse[(int64_t)t * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * PA_LN2;
}

// Rows r .. r + 256 / DP - 1 (below live) of a tile in parts: joined and written.
template <typename T, int DP, bool LIVE>
__device__ __forceinline__ void pa_join_tile_rows(const PaParams& p, const PaParts& t, int R, int r, int live, int row0, int first,
                                                  int head, int lane) {
    const int mine = r + lane / (DP / 4), in = min(mine, live - 1);
    f32x4 o;
    float m, l;
    pa_join_rows<DP, LIVE>(t.n, [&](int j, const float2*& ml, const float*& q) {
        const int64_t at = pa_part(t, j, in, R);
        ml = p.ws_ml + at;
        q = p.ws_o + at * DP;
    }, lane, o, m, l);
    const int i = (int)div_of((uint32_t)(row0 + in), p.by_g);
    if (mine < live) pa_store_row<T, DP>(p, first + i, head * p.G + row0 + in - i * p.G, o, m, l, lane);
}

// The end of a segment that left a part: the last workgroup of the tile to come here joins its parts.  Every wavefront of the
// workgroup calls it, its stores made.
template <typename T, int DP, int WAVES>
__device__ __forceinline__ void pa_arrive(const PaParams& p, const PaParts& t, int R, int live, int row0, int first,
                                          int head, int w, int lane, int* flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned before = __hip_atomic_fetch_add(p.ws_count + t.i0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = before == (unsigned)(t.n - 1);
        if (last) __hip_atomic_store(p.ws_count + t.i0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    constexpr int RPW = 256 / DP;
    for (int r = w * RPW; r < live; r += WAVES * RPW) pa_join_tile_rows<T, DP, true>(p, t, R, r, live, row0, first, head, lane);
}

// The end of a workgroup of a launch whose parts paged_join_tiles_kernel joins: its open tile, if it has one.
__device__ __forceinline__ void pa_leave_open(PaOpen* at, const PaOpen& x) {
    if (threadIdx.x == 0) *at = x;
}

// Joins the parts of tiles of many rows, which one workgroup would be at for long (256 rows in 32 parts: 80 us): block
// i `shares` + y takes share y of the rows of the tile that workgroup i left open, if it did.  A tile's shares lie on
// different XCDs (with the tiles' first workgroups 32 apart and a tile a workgroup column, all were on one, at its 0.9 TB/s).
template <typename T, int DP>
__global__ void __launch_bounds__(256) paged_join_tiles_kernel(PaParams, int R, int shares) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    PaArgs args;
    args.load(lane);
    const PaParams p = args.get();
    const uint32_t i0 = blockIdx.x / (unsigned)shares;
    const int share = (int)(blockIdx.x - i0 * (unsigned)shares);
    const PaOpen x = p.ws_open[i0];
    if (x.parts == 0) return;
    constexpr int RPW = 256 / DP;
    for (int r = (4 * share + w) * RPW; r < x.live; r += 4 * shares * RPW)
        pa_join_tile_rows<T, DP, false>(p, {i0, x.parts}, R, r, x.live, x.row0, x.first, x.head, lane);
}

}  // namespace lava
