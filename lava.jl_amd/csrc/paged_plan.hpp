// paged_plan.hpp -- how the paged attention kernels share out their work, and join its parts (device side, internal).
//
// Work is counted in blocks of BK keys: (sequence, key head, row tile, block), flattened in that order.  A launch of n
// workgroups cuts it into n equal parts; lengths are on the device, so every wavefront finds its workgroup's part
// itself, by one scan over the sequences.  A part is a run of segments, each some blocks of one row tile.  A
// segment of all of its tile's blocks gives the result; another leaves (sums, maximum, weight) in the
// workspace -- of a workgroup's segments only the first can continue a tile and only the last can leave one open,
// so two slots a workgroup hold them -- and the last workgroup of a tile to arrive joins its parts in key order.
#pragma once
#include "paged_attn.hpp"

namespace lava {

// A sequence's (or the stacked prefix's) share: key blocks [p0, p0 + np) of the prefix, then [o0, o0 + nb - np) of its
// own keys, for every row tile and key head.
struct PaSeq {
    uint32_t work;
    int tiles, nb, p0, np, o0;
    int first_nb;   // blocks that the first row tile sees, about (a causal sequence's tiles see more and more)
};

// ABOVE: the launch takes the sequences of more than row_limit rows (and reads the prefix for each of them),
// else those of at most that many.
template <int BK, bool ABOVE>
__device__ __forceinline__ PaSeq pa_seq(const PaParams& p, const PagedSeq& s, int R) {
    PaSeq w = {};
    const int64_t rows = (int64_t)s.n * p.G;
    if (rows == 0 || (rows > p.row_limit) != ABOVE) return w;
    const int first = p.P + s.kv - s.n;
    const int lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
    if (p.P > 0 && (ABOVE || p.stack == 0) && lo < p.P) {
        w.p0 = lo / BK;
        w.np = (p.P + BK - 1) / BK - w.p0;
    }
    const int own = max(0, lo - p.P);
    w.o0 = own / BK;
    w.nb = max(1, w.np + (s.kv > own ? (s.kv + BK - 1) / BK - w.o0 : 0));   // rows without keys are written too
    w.first_nb = p.causal && !p.bidir ? max(1, w.nb - (s.n + BK - 1) / BK) : w.nb;
    w.tiles = ((int)rows + R - 1) / R;
    w.work = (uint32_t)w.tiles * (uint32_t)w.nb * (uint32_t)p.c.heads;
    return w;
}

__device__ __forceinline__ uint32_t pa_scan(uint32_t x, int lane) {   // inclusive, over the wavefront
    for (int i = 1; i < 64; i *= 2) {
        const uint32_t y = __shfl_up(x, i, 64);
        x += lane >= i ? y : 0;
    }
    return x;
}
__device__ __forceinline__ float pa_wave_max(float x) {
    for (int i = 1; i < 64; i *= 2) x = fmaxf(x, __shfl_xor(x, i, 64));
    return x;
}
__device__ __forceinline__ float pa_wave_sum(float x) {
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i, 64);
    return x;
}

// What every wavefront knows of the whole call.
struct PaPlan {
    uint32_t total;
    PaSeq prefix;       // the stacked prefix, in front of the sequences (work 0: none)
    int t0, t1;         // rows of the batch
    bool plain;         // every row sees the whole prefix
    uint32_t upto;      // lane i: the work of sequences 0 .. i (i < 64)
    uint32_t seen;      // ABOVE: blocks that rows see, about (total counts every tile like its sequence's last)
    int longest;        // ABOVE: the most blocks of a tile
};

// The stacked prefix for the rows of all sequences; lo: the first position that one of them sees.
template <int BK>
__device__ __forceinline__ void pa_plan_prefix(const PaParams& p, PaPlan& g, int R, int lo) {
    g.t0 = min(max(p.b.q_start[0], 0), p.b.T);
    g.t1 = min(max(p.b.q_start[p.b.B], g.t0), p.b.T);
    if (lo < p.P && g.t1 > g.t0) {
        g.prefix.p0 = lo / BK;
        g.prefix.np = g.prefix.nb = (p.P + BK - 1) / BK - g.prefix.p0;
        g.prefix.tiles = ((g.t1 - g.t0) * p.G + R - 1) / R;
        g.prefix.work = (uint32_t)g.prefix.tiles * (uint32_t)g.prefix.nb * (uint32_t)p.c.heads;
    }
}

// SEQS: the launch takes sequences; PREFIX: it takes the stacked prefix.
template <int BK, bool ABOVE>
__device__ __forceinline__ PaPlan pa_plan(const PaParams& p, int R, bool seqs, bool prefix, int lane) {
    PaPlan g = {};
    int lo = 0x7fffffff;
    bool plain = p.window == 0;
    uint32_t seen = 0;
    int longest = 0;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        uint32_t work = 0;
        if (b0 + lane < p.b.B) {
            const PagedSeq s = paged_seq(p.b, b0 + lane);
            if (seqs) {
                const PaSeq q = pa_seq<BK, ABOVE>(p, s, R);
                work = q.work;
                seen += (uint32_t)q.tiles * (uint32_t)(q.nb + q.first_nb) / 2u * (uint32_t)p.c.heads;
                longest = max(longest, q.tiles > 0 ? q.nb : 0);
            }
            if (s.n > 0) {
                lo = min(lo, p.window > 0 ? max(0, p.P + s.kv - s.n - p.window + 1) : 0);
                plain = plain && s.n <= s.kv;
            }
        }
        const uint32_t upto = pa_scan(work, lane);
        if (b0 == 0) g.upto = upto;
        g.total += __builtin_amdgcn_readlane(upto, 63);
    }
    if constexpr (ABOVE) {
        for (int i = 1; i < 64; i *= 2) {
            seen += __shfl_xor(seen, i, 64);
            longest = max(longest, __shfl_xor(longest, i, 64));
        }
        g.seen = __builtin_amdgcn_readfirstlane(seen);
        g.longest = __builtin_amdgcn_readfirstlane(longest);
    }
    if (prefix) {
        for (int i = 1; i < 64; i *= 2) lo = min(lo, __shfl_xor(lo, i, 64));
        g.plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
        pa_plan_prefix<BK>(p, g, R, __builtin_amdgcn_readfirstlane(lo));
        g.total += g.prefix.work;
    }
    return g;
}

// The sequence that holds block `w` of the work, and the work in front of it; -1: the stacked prefix.
template <int BK, bool ABOVE>
__device__ __forceinline__ int pa_locate(const PaParams& p, const PaPlan& g, int R, uint32_t w, int lane, uint32_t& before) {
    before = 0;
    if (w < g.prefix.work) return -1;
    before = g.prefix.work;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        uint32_t upto = g.upto;
        if (b0 > 0) {
            uint32_t work = 0;
            if (b0 + lane < p.b.B) work = pa_seq<BK, ABOVE>(p, paged_seq(p.b, b0 + lane), R).work;
            upto = pa_scan(work, lane);
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > w);
        if (past != 0) {
            const int i = __builtin_ctzll(past);
            if (i > 0) before += __builtin_amdgcn_readlane(upto, i - 1);
            return b0 + i;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return p.b.B;   // not reached for w < total
}

// A workgroup's place among `n` (a multiple of 8): consecutive parts on one XCD, which share keys in its L2.
__device__ __forceinline__ uint32_t pa_place(uint32_t n) { return (blockIdx.x & 7) * (n >> 3) + (blockIdx.x >> 3); }
__device__ __forceinline__ uint32_t pa_per(uint32_t total, uint32_t n) { return max(1u, (total + n - 1) / n); }

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

// ---- parts ----------------------------------------------------------------------------
// Partial results are written and read as device-wide relaxed atomics of 8 bytes: they pass the XCDs' L2 caches
// without a fence that would write those back, and a wait for the stores before the arrival is counted orders them.

__device__ __forceinline__ void pa_put(float* p, float a, float b) {
    const float2 v = make_float2(a, b);
    __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_get(const float* p) {
    return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// A row's parts joined by a wavefront: part j's (maximum, weight) at ml(j), its sums at o(j); DP columns, DP / 64 a lane.
// Parts of no weight have no sums.
template <int DP, typename ML, typename OF>
__device__ __forceinline__ void pa_join_row(int n, ML ml, OF of, int lane, float (&o)[DP / 64], float& m, float& l) {
    constexpr int NC = DP / 64;
    m = -INFINITY;
    for (int j0 = 0; j0 < n; j0 += 64)
        if (j0 + lane < n) m = fmaxf(m, pa_get((const float*)ml(j0 + lane)).x);
    m = pa_wave_max(m);
    const float sub = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 64) {
        float f = 0.f;
        if (j0 + lane < n) {
            const float2 x = pa_get((const float*)ml(j0 + lane));
            f = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - sub);
            l += x.y * f;
        }
        const int k = min(n - j0, 64);
        constexpr int U = NC == 4 ? 4 : 8;   // loads in flight
        for (int j = 0; j < k; j += U) {
            float2 v[U][(NC + 1) / 2];
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                w[u] = j + u < k ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(j + u, 63))) : 0.f;
#pragma unroll
                for (int c = 0; c < (NC + 1) / 2; ++c) {
                    v[u][c] = make_float2(0.f, 0.f);
                    if (w[u] != 0.f) {
                        const float* q = of(j0 + j + u);
                        if constexpr (NC == 1)
                            v[u][c].x = __hip_atomic_load(q + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        else
                            v[u][c] = pa_get(q + NC * lane + 2 * c);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < NC; ++c) o[c] = fmaf(w[u], c & 1 ? v[u][c / 2].y : v[u][c / 2].x, o[c]);
        }
    }
    l = pa_wave_sum(l);
}

template <typename T, int DP>
__device__ __forceinline__ void pa_store_row(const PaParams& p, int t, int h, const float (&o)[DP / 64], float m, float l, int lane) {
    constexpr int NC = DP / 64;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* orow = (T*)p.O + (int64_t)t * p.ost + (int64_t)h * p.osh + NC * lane;
    typedef T vt __attribute__((ext_vector_type(NC)));
    if (NC * lane < p.c.D) {   // D is a multiple of 8
        vt v;
#pragma unroll
        for (int c = 0; c < NC; ++c) v[c] = (T)(o[c] * inv);
        *reinterpret_cast<vt*>(orow) = v;
    }
    if (p.lse && lane == 0) p.lse[(int64_t)t * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * PA_LN2;
}

// The end of a segment that left a part: the last workgroup of the tile to come here joins its parts, those of
// workgroups i0 .. i1.  Every wavefront of the workgroup calls it, its stores made.
template <typename T, int DP, int WAVES>
__device__ __forceinline__ void pa_arrive(const PaParams& p, uint32_t i0, uint32_t i1, int R, int live, int row0, int first,
                                          int head, int w, int lane, int* flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned before = __hip_atomic_fetch_add(p.ws_count + i0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = before == i1 - i0;
        if (last) __hip_atomic_store(p.ws_count + i0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
    for (int r = w; r < live; r += WAVES) {
        auto at = [&](int j) { return (int64_t)(2 * (i0 + (uint32_t)j) + (j == 0 ? 1u : 0u)) * R + r; };
        float o[DP / 64], m, l;
        pa_join_row<DP>((int)(i1 - i0 + 1), [&](int j) { return p.ws_ml + at(j); }, [&](int j) { return p.ws_o + at(j) * DP; }, lane, o,
                        m, l);
        const int i = (int)div_of((uint32_t)(row0 + r), p.by_g);
        pa_store_row<T, DP>(p, first + i, head * p.G + row0 + r - i * p.G, o, m, l, lane);
    }
}

}  // namespace lava
