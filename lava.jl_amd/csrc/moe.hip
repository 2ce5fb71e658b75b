// moe.hip -- tokens routed to experts, sorted by them, and the experts' results summed.
//
// Routing: L lanes of a wavefront (16 up to 128 experts, 32 up to 256, then 64) have a token, lane l the logits of experts
// V l .. V l + V - 1, and take the highest one top_k times: a maximum over the lanes by rotations within 16 lanes, then the
// lowest expert that has it.  (A token a wavefront costs more: of 64 lanes' reductions each is half as long again and serves one token instead of
// four: 16384 tokens of 64 experts 20.0 us against 13.7.)  Without a bias the order of p is that of the logits, by which
// experts, and groups counted by their best, are then compared: p of two may be equal in 64 bits (sigmoids of 38 and 39).  With one,
// and for groups counted by two, c = p + bias is taken in 32 bits first; where two that the choice tells apart lie nearer to each
// other than c's rounding may move them, the wavefront's tokens are done again in 64.
// Bound by issue: 8 ranks of 256 experts in 8 groups with a bias take 29 to 33 us for 16384 tokens (0.5 TB/s of logits), of which
// the few that are done again are the last 7; a decode step's 64 tokens of 64 experts with their plan 8.8, one token 8.2.
//
// Sorting: workgroup b has tokens [b * span, (b + 1) * span), counts its assignments per expert, and in a second launch
// (in the same one where a workgroup has all tokens) adds the counts of the lower workgroups and places its own in
// order: a stable counting sort without global atomics, the same in every run.  Every workgroup looks at all the others' counts, which
// are bytes where they fit: 16384 tokens, 8 of 256, the second launch 6.8 us, with counts of 32 bits, which given ids need as one may
// come any number of times, 10.8 (and 2.5 for the counts; 64 tokens 3.9).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_common.hpp"
#include "lava_hip_internal.hpp"
#include "w8a8.hpp"

namespace lava {

namespace {

constexpr int MOE_THREADS = 1024, MOE_WAVES = MOE_THREADS / 64;
constexpr int MOE_EXPERTS = 1024, MOE_TOP_K = 32;
constexpr int MOE_BLOCKS = 256;    // workgroups that share a sort, at most
constexpr int MOE_SPAN = 64;       // tokens a workgroup, at least
constexpr int MOE_COLUMNS = 8;     // of a row that a thread sums

struct Plan {   // what a kernel needs of a plan
    int32_t* offsets;   // null: none is written
    int32_t* order;
    int32_t* counts;    // [workgroup][expert], or bytes, rows of whole words
    int tokens, experts, top_k, span;
    int bytes;          // no count is above 255
};

// tokens a workgroup has
int span_of(int64_t tokens) {
    const int64_t per = (tokens + MOE_BLOCKS - 1) / MOE_BLOCKS;
    return (int)((per + MOE_SPAN - 1) / MOE_SPAN * MOE_SPAN);
}
int blocks_of(int64_t tokens) {
    if (tokens == 0) return 1;
    const int span = span_of(tokens);
    return (int)((tokens + span - 1) / span);
}

struct Router {
    const float* bias;
    int experts, top_k, softmax, groups, top_groups, group_best, renormalize;
    int by_logit;   // nothing is compared by p: there is no bias, and groups are counted by their best or all stay
    float scale;
};

constexpr float NONE = -__builtin_inff();

// ---- over the L lanes of a token, the result the same in all of them, bit for bit (each step is symmetric) ----
// Two wait states lie between a result and its use by another lane.
#define LAVA_ROW_ALL(OP)                                                       \
    "s_nop 1\n\t" OP " %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"   \
    "s_nop 1\n\t" OP " %0, %0, %0 row_ror:4 row_mask:0xf bank_mask:0xf\n\t"   \
    "s_nop 1\n\t" OP " %0, %0, %0 row_ror:2 row_mask:0xf bank_mask:0xf\n\t"   \
    "s_nop 1\n\t" OP " %0, %0, %0 row_ror:1 row_mask:0xf bank_mask:0xf"
// f(x, the other's x) of lane l and lane l ^ 16, or l ^ 32: v_permlane16_swap exchanges one copy's odd rows of 16 lanes with the
// other's even ones.
template <int D, typename F>
__device__ __forceinline__ uint32_t across(uint32_t x, F f) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 both;
    if constexpr (D == 16) both = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x, x, false, false));
    else both = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(x, x, false, false));
    return f(both[0], both[1]);
}
template <int L, typename F>
__device__ __forceinline__ uint32_t rows(uint32_t x, F f) {
    if constexpr (L > 16) x = across<16>(x, f);
    if constexpr (L > 32) x = across<32>(x, f);
    return x;
}
template <int L>
__device__ __forceinline__ float all_max(float x) {
    asm(LAVA_ROW_ALL("v_max_f32_dpp") : "+v"(x));
    return __uint_as_float(rows<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int L>
__device__ __forceinline__ float all_sum(float x) {
    asm(LAVA_ROW_ALL("v_add_f32_dpp") : "+v"(x));
    return __uint_as_float(rows<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
template <int L>
__device__ __forceinline__ int all_min(int x) {
    asm(LAVA_ROW_ALL("v_min_i32_dpp") : "+v"(x));
    return (int)rows<L>((uint32_t)x, [](uint32_t a, uint32_t b) { return (uint32_t)min((int)a, (int)b); });
}
template <int L>
__device__ __forceinline__ uint32_t all_max(uint32_t x) {
    asm(LAVA_ROW_ALL("v_max_u32_dpp") : "+v"(x));
    return rows<L>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
#undef LAVA_ROW_ALL
// The upper halves of bits that order as the numbers do, then the lower ones of those that have the highest.
template <int L>
__device__ __forceinline__ double all_max(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x), sign = 1ull << 63;
    const uint64_t key = b & sign ? ~b : b | sign;
    const uint32_t hi = (uint32_t)(key >> 32), top = all_max<L>(hi);
    const uint64_t best = (uint64_t)top << 32 | all_max<L>(hi == top ? (uint32_t)key : 0u);
    return __builtin_bit_cast(double, best & sign ? best ^ sign : ~best);
}
template <int L>
__device__ __forceinline__ double all_sum(double x) {
#pragma unroll
    for (int d = 1; d < L; d <<= 1) x += __shfl_xor(x, d, 64);
    return x;
}

// p of a logit: in 32 bits by v_exp_f32 and v_rcp_f32 (1 ulp each; the exponent's rounding is below |x| 2^-24, of p (1 - p) |x| <
// 0.3 in all), enough to choose by where `apart` says so
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float quotient(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double quotient(double x) { return 1.0 / x; }

// The experts of the token that these L lanes have, highest first, rank r in lane r % L's sel[r / L] (and, where there is no bias,
// their logits in xs); true unless 32 bits do not settle the order.  most: the largest finite |bias|.
template <int L, int V, typename Real>
__device__ __forceinline__ bool choose(const Router& r, const float (&x)[V], const float (&bias)[V], float most, int lane,
                                       int (&sel)[2], float (&xs)[2]) {
    constexpr bool SINGLE = sizeof(Real) == 4;
    constexpr Real LEAST = (Real)NONE;
    bool by_logit = r.by_logit;
    Real c[V];
    Real near = 0;   // how near two c may be that 32 bits cannot tell apart, without the part that grows with c
    if (by_logit) {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = (Real)x[v];
    } else {
        Real top = 0, norm = 1;
        if (r.softmax) {
            float m = x[0];
#pragma unroll
            for (int v = 1; v < V; ++v) m = fmaxf(m, x[v]);
            m = all_max<L>(m);
            top = m == NONE ? (Real)0 : (Real)m;
            Real sum = 0;
#pragma unroll
            for (int v = 0; v < V; ++v) sum += exp_of((Real)x[v] - top);
            sum = all_sum<L>(sum);
            norm = sum > 0 ? 1 / sum : (Real)0;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Real p = r.softmax ? exp_of((Real)x[v] - top) * norm : quotient(1 + exp_of(-(Real)x[v]));
            c[v] = x[v] == NONE ? LEAST : p + (Real)bias[v];
        }
        // Each p is off by, in units of 2^-24: a sigmoid 2 p (1 - p) |x| < 0.5 of the exponent and log2 e, 2 p (1 - p) <= 0.5 of
        // exp, the sum 1, the quotient 2, below 4; a softmax, of the largest p, the exponent 1.1, exp 2, the sum V + 6 <= 22
        // additions of terms off by 3 ln 1024 + 2 on average, the quotient and the product 2, below 52.
        if (SINGLE) near = r.softmax ? norm * (Real)0x1p-17f : (Real)0x1p-21f;
    }
    auto apart = [&](Real hi, Real lo, int terms) {
        if (!SINGLE || by_logit || lo == LEAST) return true;
        // the sum of two c may be far below them: their own roundings
        const Real more = terms == 2 ? (Real)0x1p-21f * (1 + (Real)most) : (Real)0;
        return hi - lo > terms * (near + (Real)0x1p-22f * fmax((Real)fabs(hi), (Real)fabs(lo))) + more;
    };
    bool sure = true;
    if (r.top_groups < r.groups) {
        // a group's best two: of a lane's experts, then over the lanes
        const int size = r.experts / r.groups, base = (threadIdx.x & 63) - lane;
        auto join = [&](Real& b1, Real& b2, int d) __attribute__((always_inline)) {
            const Real o1 = __shfl_xor(b1, d, 64), o2 = __shfl_xor(b2, d, 64);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        };
        constexpr int GV = 64 / L;
        Real count[GV], b1, b2;   // group g's in lane g % L's count[g / L]
#pragma unroll
        for (int i = 0; i < GV; ++i) count[i] = LEAST;
        const int span = size / V;
        if (size % V == 0 && (span & (span - 1)) == 0) {   // whole lanes, a power of two of them: all groups at once
            b1 = b2 = LEAST;
#pragma unroll
            for (int v = 0; v < V; ++v) {   // beyond the experts c is the least
                b2 = fmax(b2, fmin(b1, c[v]));
                b1 = fmax(b1, c[v]);
            }
            for (int d = 1; d < span; d <<= 1) join(b1, b2, d);
            // at most L / span groups, so one a lane
            const Real o = __shfl(r.group_best == 2 ? b1 + b2 : b1, base + min(lane * span, L - 1), 64);
            count[0] = lane < r.groups ? o : LEAST;
        } else {   // one group after another: its highest, then its highest without that one
            for (int g = 0; g < r.groups; ++g) {
                const int lo = g * size, hi = lo + size;
                auto highest = [&](int but) __attribute__((always_inline)) {
                    Real m = LEAST;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const int e = lane * V + v;
                        m = fmax(m, e >= lo && e < hi && e != but ? c[v] : LEAST);
                    }
                    return all_max<L>(m);
                };
                Real o = highest(-1);
                if (r.group_best == 2) {
                    int at = L * V;
#pragma unroll
                    for (int v = V - 1; v >= 0; --v) {
                        const int e = lane * V + v;
                        at = e >= lo && e < hi && c[v] == o ? e : at;
                    }
                    o += highest(all_min<L>(at));
                }
#pragma unroll
                for (int i = 0; i < GV; ++i) count[i] = g == i * L + lane ? o : count[i];
            }
        }
        int rank[GV];   // the groups in front of this one
#pragma unroll
        for (int i = 0; i < GV; ++i) rank[i] = 0;
        for (int g = 0; g < r.groups; ++g) {
            Real mine = count[0];
#pragma unroll
            for (int i = 1; i < GV; ++i) mine = g / L == i ? count[i] : mine;
            const Real o = __shfl(mine, base + g % L, 64);
#pragma unroll
            for (int i = 0; i < GV; ++i) rank[i] += o > count[i] || (o == count[i] && g < i * L + lane);
        }
        Real worst = LEAST, next = LEAST;   // -(the least that stays), the highest that does not
        uint64_t kept = 0;
#pragma unroll
        for (int i = 0; i < GV; ++i) {
            const bool in = i * L + lane < r.groups, stays = in && rank[i] < r.top_groups;
            worst = fmax(worst, stays ? -count[i] : LEAST);
            next = fmax(next, in && !stays ? count[i] : LEAST);
            const uint64_t all = __ballot(stays) >> base;   // the token's lanes on
            kept |= (L == 64 ? all : all & ((1ull << (L & 63)) - 1)) << (i * (L & 63));
        }
        sure = apart(-all_max<L>(worst), all_max<L>(next), r.group_best);
        const float inv = 1.f / (float)size;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int g = (int)(((float)(lane * V + v) + 0.5f) * inv);
            if (!(kept >> (g & 63) & 1)) c[v] = LEAST;
            else if (r.bias == nullptr) c[v] = (Real)x[v];
        }
        by_logit = r.bias == nullptr;   // from here on: single experts
    }
    sel[0] = sel[1] = -1;
    xs[0] = xs[1] = NONE;
    Real last = 0;
    for (int i = 0; i < r.top_k + (SINGLE && !by_logit); ++i) {
        Real top = c[0];
#pragma unroll
        for (int v = 1; v < V; ++v) top = fmax(top, c[v]);
        top = all_max<L>(top);
        if (i > 0) sure = sure && apart(last, top, 1);
        last = top;
        if (i == r.top_k) break;
        int at = L * V;   // the lowest expert that has it
#pragma unroll
        for (int v = V - 1; v >= 0; --v) at = c[v] == top ? lane * V + v : at;
        at = all_min<L>(at);
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = lane * V + v == at ? LEAST : c[v];
        at = top == LEAST ? -1 : at;   // none left
        sel[0] = i == lane ? at : sel[0];
        xs[0] = i == lane ? (float)top : xs[0];
        if (L < 32) {
            sel[1] = i == L + lane ? at : sel[1];
            xs[1] = i == L + lane ? (float)top : xs[1];
        }
    }
    return sure;
}

// Places the tokens' assignments: base[e] is the next free place of expert e's run.
// Stable: 1024 assignments at a time, a thread each; its place is base + those of lower wavefronts + those of lower lanes.
__device__ void place(const Plan& p, const int32_t* ids, int64_t first, int64_t last, int32_t* base, uint16_t* below) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, E = p.experts;
    const int bits = 32 - __clz(E - 1 > 0 ? E - 1 : 1);
    for (int64_t i0 = first; i0 < last; i0 += MOE_THREADS) {
        for (int i = threadIdx.x; i < MOE_WAVES * E; i += MOE_THREADS) below[i] = 0;
        __syncthreads();
        const int64_t i = i0 + threadIdx.x;
        const int e = i < last ? ids[i] : -1;
        const bool ok = e >= 0 && e < E;
        uint64_t same = __ballot(ok);   // lanes of the same expert
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(ok && (e >> b & 1));
            same &= (e >> b & 1) ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (ok && rank == 0) below[w * E + e] = (uint16_t)__popcll(same);
        __syncthreads();
        if (ok) {
            int at = base[e] + rank;
            for (int v = 0; v < w; ++v) at += below[v * E + e];
            p.order[at] = (int32_t)i;
        }
        __syncthreads();
        for (int j = threadIdx.x; j < E; j += MOE_THREADS) {
            int sum = 0;
            for (int v = 0; v < MOE_WAVES; ++v) sum += below[v * E + j];
            base[j] += sum;
        }
        __syncthreads();
    }
}

// Exclusive scan of v over the workgroup's threads; total: of all.
__device__ __forceinline__ int scan(int v, int32_t* tmp, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d, 64);
        if (lane >= d) sum += o;
    }
    if (lane == 63) tmp[w] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < MOE_WAVES; ++i) {
        if (i < w) before += tmp[i];
        total += tmp[i];
    }
    __syncthreads();
    return before + sum - v;
}

// Of workgroup b, whose own and the others' counts are known: writes its part of the plan.
__device__ void finish_plan(const Plan& p, const int32_t* ids, int b, int blocks, int before, int all, int32_t* base,
                            uint16_t* below, int32_t* tmp) {
    int total;
    const int start = scan(all, tmp, total);   // of expert threadIdx.x
    if (threadIdx.x < (unsigned)p.experts) {
        base[threadIdx.x] = start + before;
        if (b == 0) p.offsets[threadIdx.x] = start;
    }
    if (b == 0 && threadIdx.x == 0) p.offsets[p.experts] = total;
    const int rows = p.tokens * p.top_k;
    for (int64_t i = (int64_t)total + b * MOE_THREADS + threadIdx.x; i < rows; i += (int64_t)blocks * MOE_THREADS) p.order[i] = -1;
    __syncthreads();
    const int64_t last = min((int64_t)(b + 1) * p.span, (int64_t)p.tokens);
    place(p, ids, (int64_t)b * p.span * p.top_k, last * p.top_k, base, below);
}

struct SortShared {
    int32_t base[MOE_EXPERTS];
    int32_t tmp[MOE_WAVES];
};
static_assert(MOE_THREADS == MOE_EXPERTS, "a thread an expert");

__host__ __device__ constexpr int byte_row(int experts) { return (experts + 3) & ~3; }

}  // namespace

// VEC: rows of logits aligned to V of them (or 16 bytes), experts a multiple of V.
template <typename T, int L, int V, bool VEC>
__global__ void __launch_bounds__(MOE_THREADS) moe_route_kernel(Router r, const T* __restrict__ logits, int64_t ldl,
                                                                int32_t* ids, float* weights, Plan p) {
    extern __shared__ uint16_t below[];   // MOE_WAVES * experts where one workgroup has all tokens and writes the plan
    __shared__ SortShared sh;
    constexpr int PER = MOE_THREADS / L, S = L < 32 ? 2 : 1;   // tokens at once; ranks a lane
    const int lane = threadIdx.x & (L - 1), b = blockIdx.x;
    if (p.offsets) {
        sh.base[threadIdx.x] = 0;
        __syncthreads();
    }
    float bias[V], most = 0.f;
    bool bad_bias = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = r.bias && lane * V + v < r.experts ? r.bias[lane * V + v] : 0.f;
        bad_bias |= !(bias[v] < __builtin_inff());
        most = fmaxf(most, bias[v] == NONE ? 0.f : fabsf(bias[v]));
    }
    if (r.group_best == 2) most = all_max<L>(most);   // only those counts need it
    const int64_t last = min((int64_t)(b + 1) * p.span, (int64_t)p.tokens);
    for (int64_t t0 = (int64_t)b * p.span; t0 < last; t0 += PER) {
        const int64_t t = t0 + threadIdx.x / L;
        const bool live = t < last;
        const T* row = logits + (live ? t : 0) * ldl;
        float x[V];
        if constexpr (VEC) {
            constexpr int C = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
            typedef T Tv __attribute__((ext_vector_type(C)));
            const bool in = live && lane * V < r.experts;
#pragma unroll
            for (int v = 0; v < V; v += C) {
                const Tv q = *reinterpret_cast<const Tv*>(row + (in ? lane * V + v : 0));
#pragma unroll
                for (int i = 0; i < C; ++i) x[v + i] = in ? (float)q[i] : NONE;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = live && lane * V + v < r.experts ? (float)row[lane * V + v] : NONE;
        }
        bool bad = bad_bias;
#pragma unroll
        for (int v = 0; v < V; ++v) bad |= !(x[v] < __builtin_inff());
        bad = all_min<L>(bad ? 0 : 1) == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = bad ? NONE : x[v];
        int sel[2];
        float xs[2];
        const bool sure = choose<L, V, float>(r, x, bias, most, lane, sel, xs);
        if (__ballot(!sure) != 0) choose<L, V, double>(r, x, bias, most, lane, sel, xs);

        // the weights, from the chosen logits; divided by their sum they are taken relative to the highest logit among them,
        // so that p of far masked or shut out experts, below the least float, does not make 0 / 0.  In 32 bits, the type of the weights,
        // whose last bit that costs (measured 6e-8 off, rounded once from 64 bits 3e-8)
        float weight[S], top = NONE, all = 0.f;
        if (r.bias) {
#pragma unroll
            for (int i = 0; i < S; ++i) xs[i] = sel[i] >= 0 ? (float)row[sel[i]] : NONE;
        }
#pragma unroll
        for (int i = 0; i < S; ++i) top = fmaxf(top, xs[i]);
        if (r.softmax && !r.renormalize) {
#pragma unroll
            for (int v = 0; v < V; ++v) top = fmaxf(top, x[v]);
        }
        top = all_max<L>(top);
        if (!r.softmax) top = r.renormalize ? fminf(top, 0.f) : 0.f;
        if (top == NONE) top = 0.f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            // softmax: exp(x - top); sigmoid: exp(-top) / (1 + exp(-x)), where top is 0 unless every x is below it
            weight[i] = sel[i] < 0    ? 0.f
                        : r.softmax   ? expf(xs[i] - top)
                        : xs[i] > 0.f ? 1.f / (1.f + expf(-xs[i]))
                                      : expf(xs[i] - top) / (1.f + expf(xs[i]));
            all += weight[i];
        }
        if (!r.renormalize) {
            all = r.softmax ? 0.f : lane == 0 ? 1.f : 0.f;
            if (r.softmax) {
#pragma unroll
                for (int v = 0; v < V; ++v) all += expf(x[v] - top);
            }
        }
        all = all_sum<L>(all);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int rank = i * L + lane;
            if (!live || rank >= r.top_k) continue;
            float o = weight[i] / all * r.scale;
            if (sel[i] < 0) o = bad ? __builtin_nanf("") : 0.f;
            ids[t * r.top_k + rank] = sel[i];
            weights[t * r.top_k + rank] = o;
            if (p.offsets && sel[i] >= 0) atomicAdd(&sh.base[sel[i]], 1);
        }
    }
    if (!p.offsets) return;
    __syncthreads();   // the counts, and this workgroup's ids in memory
    const int all = threadIdx.x < (unsigned)p.experts ? sh.base[threadIdx.x] : 0;
    if (gridDim.x > 1) {
        if (p.bytes) {
            if (threadIdx.x < (unsigned)byte_row(p.experts))
                reinterpret_cast<uint8_t*>(p.counts)[b * byte_row(p.experts) + threadIdx.x] = (uint8_t)all;
        } else if (threadIdx.x < (unsigned)p.experts) {
            p.counts[b * p.experts + threadIdx.x] = all;
        }
        return;
    }
    __syncthreads();
    finish_plan(p, ids, 0, 1, 0, all, sh.base, below, sh.tmp);
}

// Counts given ids; a workgroup that has all tokens places them too.
__global__ void __launch_bounds__(MOE_THREADS) moe_count_kernel(const int32_t* __restrict__ ids, Plan p) {
    extern __shared__ uint16_t below[];
    __shared__ SortShared sh;
    const int b = blockIdx.x;
    sh.base[threadIdx.x] = 0;
    __syncthreads();
    const int64_t last = min((int64_t)(b + 1) * p.span, (int64_t)p.tokens) * p.top_k;
    for (int64_t i = (int64_t)b * p.span * p.top_k + threadIdx.x; i < last; i += MOE_THREADS) {
        const int e = ids[i];
        if (e >= 0 && e < p.experts) atomicAdd(&sh.base[e], 1);
    }
    __syncthreads();
    const int all = threadIdx.x < (unsigned)p.experts ? sh.base[threadIdx.x] : 0;
    if (gridDim.x > 1) {
        if (threadIdx.x < (unsigned)p.experts) p.counts[b * p.experts + threadIdx.x] = all;
        return;
    }
    __syncthreads();
    finish_plan(p, ids, 0, 1, 0, all, sh.base, below, sh.tmp);
}

// Adds the workgroups' counts, in front of this one's and all.  BYTES: four experts a load, both sums in one word (at most 256 * 255).
template <bool BYTES>
__global__ void __launch_bounds__(MOE_THREADS) moe_place_kernel(const int32_t* __restrict__ ids, Plan p) {
    extern __shared__ uint16_t below[];
    __shared__ SortShared sh;
    constexpr int C = BYTES ? 4 : 1, MOST = 16;   // experts a thread; parts of the workgroups' rows that are read side by side
    __shared__ uint32_t part[BYTES ? 1 : 2][C * MOE_THREADS];
    const int mine = blockIdx.x, blocks = gridDim.x, words = BYTES ? byte_row(p.experts) / 4 : p.experts;
    int width = 64 / C;
    while (width < words) width <<= 1;
    const int parts = min(MOST, MOE_THREADS / width), at = threadIdx.x & (width - 1), row = threadIdx.x / width;
    uint32_t before[C] = {}, all[C] = {};
    if (at < words && row < parts) {
        for (int b0 = row; b0 < blocks; b0 += 16 * parts) {
            uint32_t n[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int b = b0 + i * parts;
                n[i] = b < blocks ? reinterpret_cast<const uint32_t*>(p.counts)[b * words + at] : 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool lower = b0 + i * parts < mine;
                if constexpr (BYTES) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) all[c] += (n[i] >> 8 * c & 255u) * (lower ? 0x10001u : 0x10000u);
                } else {
                    all[0] += n[i];
                    before[0] += lower ? n[i] : 0u;
                }
            }
        }
    }
    if (row < parts) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            part[0][C * (row * width + at) + c] = all[c];
            if constexpr (!BYTES) part[1][row * width + at] = before[c];
        }
    }
    __syncthreads();
    uint32_t sum = 0, lower = 0;
    if (threadIdx.x < (unsigned)p.experts) {
        for (int i = 0; i < parts; ++i) {
            sum += part[0][i * C * width + threadIdx.x];
            if constexpr (!BYTES) lower += part[1][i * width + threadIdx.x];
        }
        if constexpr (BYTES) {
            lower = sum & 0xffffu;
            sum >>= 16;
        }
    }
    finish_plan(p, ids, mine, blocks, (int)lower, (int)sum, sh.base, below, sh.tmp);
}

// A thread 8 columns of a token, of any alignment.  Bound by the bytes: 8 rows of 2048 bf16 for 8192 tokens 48.2 us, 6.3 TB/s (with 4
// columns a thread 57.6, with 2 94.5); rows of 2047 54.2.
template <typename T>
__global__ void __launch_bounds__(256) moe_combine_kernel(const T* __restrict__ Y, int64_t ldy, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ weights, int top_k, int64_t n,
                                                          const T* base, int64_t ldb, T* out, int64_t ldo, int per_row) {
    constexpr int C = MOE_COLUMNS;
    typedef T Tv __attribute__((ext_vector_type(C)));
    typedef Tv Tvu __attribute__((aligned(sizeof(T))));
    const int64_t t = blockIdx.x / per_row;
    const int64_t col = ((int64_t)(blockIdx.x % per_row) * 256 + threadIdx.x) * C;
    if (col >= n) return;
    const bool whole = col + C <= n;
    auto load = [&](const T* p) __attribute__((always_inline)) {
        if (whole) return (Tv)*reinterpret_cast<const Tvu*>(p);
        Tv v;
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] = col + i < n ? p[i] : (T)0.f;
        return v;
    };
    float sum[C];
#pragma unroll
    for (int i = 0; i < C; ++i) sum[i] = 0.f;
    if (base) {
        const Tv v = load(base + t * ldb + col);
#pragma unroll
        for (int i = 0; i < C; ++i) sum[i] = (float)v[i];
    }
    for (int j = 0; j < top_k; ++j) {
        const int64_t a = t * top_k + j;
        const float w = weights[a];
        if (ids && ids[a] < 0) {
#pragma unroll
            for (int i = 0; i < C; ++i) sum[i] += w * 0.f;
            continue;
        }
        const Tv v = load(Y + a * ldy + col);
#pragma unroll
        for (int i = 0; i < C; ++i) sum[i] = __builtin_fmaf(w, (float)v[i], sum[i]);
    }
    T* o = out + t * ldo + col;
    Tv r;
#pragma unroll
    for (int i = 0; i < C; ++i) r[i] = narrow<T>(sum[i]);
    if (whole) {
        *reinterpret_cast<Tvu*>(o) = r;
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (col + i < n) o[i] = r[i];
    }
}

namespace {

int check_router(const lava_hip_moe_router* r) {
    LAVA_ARG(r != nullptr, "moe_route: null router");
    LAVA_ARG(r->experts >= 1 && r->top_k >= 1, "moe_route: %d of %d experts", r->top_k, r->experts);
    LAVA_REQUIRE(r->experts <= MOE_EXPERTS && r->top_k <= MOE_TOP_K, LAVA_HIP_ERR_UNSUPPORTED,
                 "moe_route: %d of %d experts (at most %d of %d)", r->top_k, r->experts, MOE_TOP_K, MOE_EXPERTS);
    LAVA_ARG(r->top_k <= r->experts, "moe_route: top_k = %d of %d experts", r->top_k, r->experts);
    LAVA_ARG(r->score == LAVA_HIP_SCORE_SOFTMAX || r->score == LAVA_HIP_SCORE_SIGMOID, "moe_route: unknown score %d", r->score);
    LAVA_ARG(r->groups >= 1 && r->experts % r->groups == 0, "moe_route: %d experts in %d groups", r->experts, r->groups);
    LAVA_REQUIRE(r->groups <= 64, LAVA_HIP_ERR_UNSUPPORTED, "moe_route: %d groups (at most 64)", r->groups);
    LAVA_ARG(r->top_groups >= 1 && r->top_groups <= r->groups, "moe_route: top_groups = %d of %d", r->top_groups, r->groups);
    LAVA_ARG((r->group_best == 1 || r->group_best == 2) && r->group_best <= r->experts / r->groups,
             "moe_route: group_best = %d of groups of %d", r->group_best, r->experts / r->groups);
    LAVA_ARG(r->scale - r->scale == 0.f, "moe_route: scale is not finite");
    LAVA_ARG(aligned(r->bias, 4), "moe_route: misaligned bias");
    return LAVA_HIP_OK;
}

size_t plan_bytes(int64_t tokens, int experts) {
    const int blocks = blocks_of(tokens);
    return blocks > 1 ? (size_t)blocks * experts * sizeof(int32_t) : 0;
}

int check_sizes(const char* name, int64_t tokens, int experts, int top_k) {
    LAVA_ARG(tokens >= 0, "%s: negative tokens (%lld)", name, (long long)tokens);
    LAVA_ARG(experts >= 1 && top_k >= 1, "%s: a plan of %d of %d experts", name, top_k, experts);
    LAVA_REQUIRE(experts <= MOE_EXPERTS && top_k <= MOE_TOP_K, LAVA_HIP_ERR_UNSUPPORTED,
                 "%s: a plan of %d of %d experts (at most %d of %d)", name, top_k, experts, MOE_TOP_K, MOE_EXPERTS);
    LAVA_REQUIRE(tokens <= W8_MOST / top_k, LAVA_HIP_ERR_UNSUPPORTED, "%s: %lld tokens of %d experts are too many", name,
                 (long long)tokens, top_k);
    return LAVA_HIP_OK;
}

Plan plan_of(const lava_hip_moe_plan* plan) {
    Plan p = {};
    p.offsets = plan->offsets;
    p.order = plan->order;
    p.counts = static_cast<int32_t*>(plan->workspace);
    p.tokens = (int)plan->tokens;
    p.experts = plan->experts;
    p.top_k = plan->top_k;
    p.span = plan->tokens ? span_of(plan->tokens) : MOE_SPAN;
    return p;
}

size_t below_bytes(int experts) { return (size_t)MOE_WAVES * experts * sizeof(uint16_t); }

int launch_place(const int32_t* ids, const Plan& p, int blocks, hipStream_t s) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(MOE_THREADS), below_bytes(p.experts), s, ids, p);
    };
    p.bytes ? go(moe_place_kernel<true>) : go(moe_place_kernel<false>);
    LAVA_LAUNCH_CHECK("moe_place_kernel");
    return LAVA_HIP_OK;
}

template <typename T>
int launch_route(const Router& r, const void* logits, int64_t ldl, int32_t* ids, float* weights, const Plan& p, int blocks,
                 hipStream_t s) {
    const size_t lds = p.offsets && blocks == 1 ? below_bytes(p.experts) : 0;
    const T* x = static_cast<const T*>(logits);
    auto by_v = [&](auto ltag, auto vtag) {
        constexpr int V = decltype(vtag)::value;
        constexpr int L = decltype(ltag)::value;
        constexpr size_t al = V * sizeof(T) < 16 ? V * sizeof(T) : 16;
        const bool vec = r.experts % V == 0 && ldl * (int64_t)sizeof(T) % al == 0 && aligned(logits, al);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(MOE_THREADS), lds, s, r, x, ldl, ids, weights, p);
        };
        vec ? go(moe_route_kernel<T, L, V, true>) : go(moe_route_kernel<T, L, V, false>);
    };
    std::integral_constant<int, 16> few;
    if (r.experts <= 64) by_v(few, std::integral_constant<int, 4>{});
    else if (r.experts <= 128) by_v(few, std::integral_constant<int, 8>{});
    else if (r.experts <= 256) by_v(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
    else if (r.experts <= 512) by_v(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    else by_v(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
    LAVA_LAUNCH_CHECK("moe_route_kernel");
    return p.offsets && blocks > 1 ? launch_place(ids, p, blocks, s) : LAVA_HIP_OK;
}

template <typename T>
int launch_combine(const void* Y, int64_t ldy, const int32_t* ids, const float* weights, int64_t tokens, int top_k, int64_t n,
                   const void* base, int64_t ldb, void* out, int64_t ldo, hipStream_t s) {
    const int64_t per_row = (n + 256 * MOE_COLUMNS - 1) / (256 * MOE_COLUMNS);
    LAVA_REQUIRE(per_row <= 0x7fffffff && tokens <= 0xffffff / per_row, LAVA_HIP_ERR_UNSUPPORTED,
                 "moe_combine: %lld tokens of %lld values are too many", (long long)tokens, (long long)n);
    hipLaunchKernelGGL(moe_combine_kernel<T>, dim3((unsigned)(tokens * per_row)), dim3(256), 0, s, static_cast<const T*>(Y), ldy, ids,
                       weights, top_k, n, static_cast<const T*>(base), ldb, static_cast<T*>(out), ldo, (int)per_row);
    LAVA_LAUNCH_CHECK("moe_combine_kernel");
    return LAVA_HIP_OK;
}

bool float_type(int dtype) { return dtype == LAVA_HIP_F32 || dtype == LAVA_HIP_F16 || dtype == LAVA_HIP_BF16; }

}  // namespace

int check_plan(const char* name, const lava_hip_moe_plan* plan, bool write) {
    LAVA_ARG(plan != nullptr, "%s: null plan", name);
    const int rc = check_sizes(name, plan->tokens, plan->experts, plan->top_k);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG((plan->offsets != nullptr && plan->order != nullptr) || (plan->tokens == 0 && !(write && !plan->offsets)),
             "%s: null offsets or order", name);
    LAVA_ARG(aligned(plan->offsets, 4) && aligned(plan->order, 4) && aligned(plan->workspace, 4), "%s: misaligned plan", name);
    if (write) {
        const size_t need = plan_bytes(plan->tokens, plan->experts);
        LAVA_ARG(need == 0 || (plan->workspace != nullptr && plan->workspace_bytes >= need),
                 "%s: the plan's workspace of %zu bytes is smaller than %zu", name, plan->workspace_bytes, need);
    }
    return LAVA_HIP_OK;
}

}  // namespace lava

using namespace lava;

extern "C" {

int lava_hip_moe_plan_workspace_bytes(int64_t tokens, int32_t experts, int32_t top_k, size_t* bytes) {
    LAVA_ARG(bytes != nullptr, "moe_plan_workspace_bytes: null output pointer");
    const int rc = check_sizes("moe_plan_workspace_bytes", tokens, experts, top_k);
    if (rc != LAVA_HIP_OK) return rc;
    *bytes = plan_bytes(tokens, experts);
    return LAVA_HIP_OK;
}

int lava_hip_moe_route(const lava_hip_moe_router* router, int dtype, const void* logits, int64_t ldl, int64_t tokens,
                       int32_t* ids, float* weights, const lava_hip_moe_plan* plan, void* stream) {
    int rc = check_router(router);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG(float_type(dtype), "moe_route: dtype %d is not f32, f16 or bf16", dtype);
    rc = check_sizes("moe_route", tokens, router->experts, router->top_k);
    if (rc != LAVA_HIP_OK) return rc;
    if (plan != nullptr) {
        rc = check_plan("moe_route", plan, true);
        if (rc != LAVA_HIP_OK) return rc;
        LAVA_ARG(plan->tokens == tokens && plan->experts == router->experts && plan->top_k == router->top_k,
                 "moe_route: a plan of %lld tokens and %d of %d experts", (long long)plan->tokens, plan->top_k, plan->experts);
    }
    if (tokens == 0 && plan == nullptr) return LAVA_HIP_OK;
    LAVA_ARG(tokens == 0 || (logits != nullptr && ids != nullptr && weights != nullptr), "moe_route: null pointer");
    LAVA_ARG(ldl >= router->experts, "moe_route: ldl = %lld is smaller than the experts", (long long)ldl);
    LAVA_ARG(aligned(logits, dtype == LAVA_HIP_F32 ? 4 : 2) && aligned(ids, 4) && aligned(weights, 4),
             "moe_route: operands not aligned to their element size");
    rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    Router r = {router->bias, router->experts, router->top_k, router->score == LAVA_HIP_SCORE_SOFTMAX, router->groups,
                router->top_groups, router->group_best, router->renormalize,
                router->bias == nullptr && (router->top_groups == router->groups || router->group_best == 1), router->scale};
    Plan p = {};
    if (plan != nullptr) p = plan_of(plan);
    p.tokens = (int)tokens;
    p.span = tokens ? span_of(tokens) : MOE_SPAN;
    p.bytes = p.span <= 255;   // a token has an expert once
    const int blocks = blocks_of(tokens);
    hipStream_t s = as_stream(stream);
    if (dtype == LAVA_HIP_F32) return launch_route<float>(r, logits, ldl, ids, weights, p, blocks, s);
    if (dtype == LAVA_HIP_F16) return launch_route<f16>(r, logits, ldl, ids, weights, p, blocks, s);
    return launch_route<bf16>(r, logits, ldl, ids, weights, p, blocks, s);
}

int lava_hip_moe_sort(const int32_t* ids, const lava_hip_moe_plan* plan, void* stream) {
    int rc = check_plan("moe_sort", plan, true);
    if (rc != LAVA_HIP_OK) return rc;
    LAVA_ARG(plan->tokens == 0 || ids != nullptr, "moe_sort: null ids");
    LAVA_ARG(aligned(ids, 4), "moe_sort: misaligned ids");
    rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    const Plan p = plan_of(plan);
    const int blocks = blocks_of(plan->tokens);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(moe_count_kernel, dim3((unsigned)blocks), dim3(MOE_THREADS), blocks > 1 ? 0 : below_bytes(p.experts), s,
                       ids, p);
    LAVA_LAUNCH_CHECK("moe_count_kernel");
    return blocks > 1 ? launch_place(ids, p, blocks, s) : LAVA_HIP_OK;
}

int lava_hip_moe_combine(int dtype, const void* Y, int64_t ldy, const int32_t* ids, const float* weights, int64_t tokens,
                         int32_t top_k, int64_t n, const void* base, int64_t ldb, void* out, int64_t ldo, void* stream) {
    LAVA_ARG(float_type(dtype), "moe_combine: dtype %d is not f32, f16 or bf16", dtype);
    LAVA_ARG(tokens >= 0 && n >= 0 && top_k >= 0, "moe_combine: negative extent (tokens=%lld top_k=%d n=%lld)",
             (long long)tokens, top_k, (long long)n);
    if (tokens == 0 || n == 0) return LAVA_HIP_OK;
    LAVA_ARG(out != nullptr && (top_k == 0 || (Y != nullptr && weights != nullptr)), "moe_combine: null pointer");
    LAVA_ARG((top_k == 0 || ldy >= n) && ldo >= n && (base == nullptr || ldb >= n),
             "moe_combine: a stride (%lld, %lld, %lld) is smaller than n", (long long)ldy, (long long)ldb, (long long)ldo);
    const size_t sz = dtype == LAVA_HIP_F32 ? 4 : 2;
    LAVA_ARG(aligned(Y, sz) && aligned(base, sz) && aligned(out, sz) && aligned(ids, 4) && aligned(weights, 4),
             "moe_combine: operands not aligned to their element size");
    LAVA_ARG(base != out || ldb == ldo, "moe_combine: base in place of out with another stride");
    const int rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    hipStream_t s = as_stream(stream);
    if (dtype == LAVA_HIP_F32)
        return launch_combine<float>(Y, ldy, ids, weights, tokens, top_k, n, base, ldb, out, ldo, s);
    if (dtype == LAVA_HIP_F16)
        return launch_combine<f16>(Y, ldy, ids, weights, tokens, top_k, n, base, ldb, out, ldo, s);
    return launch_combine<bf16>(Y, ldy, ids, weights, tokens, top_k, n, base, ldb, out, ldo, s);
}

}  // extern "C"
