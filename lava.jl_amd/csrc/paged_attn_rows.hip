// paged_attn_rows.hip -- attention over the paged cache by rows, split evenly along the keys.
//
// The rows of one key head are its queries times its G query heads: row r of a sequence is query r / G, head r % G, and
// all of them read the same keys.  A decode step has 1 to 16 such rows and reads every key and value once: it is bound
// by HBM, 4 D bytes a key and key head.  So
//  * the work of a call -- (sequence, key head, row tile, block of 128 keys), flattened -- is cut into as many equal parts
//    as workgroups fit the chip, whatever the lengths are: long sequences are split, short ones share a workgroup.
//    Lengths are on the device, so every workgroup finds its part itself from one scan over the sequences;
//  * a workgroup's four wavefronts take 32 keys of a block each and do not wait for each other: K and V come by
//    LDS-DMA (bytes in flight without registers), one tile of each per wavefront, K's next tile requested when
//    the scores are done and V's when the sums are, so one of the two is always on its way;
//  * S^T = K Q^T and O^T = V^T P^T on 16x16x32 MFMAs: a lane owns one row, the score accumulator converts in place to the
//    second product's operand (k-slot (g, i) is key 4 g + i of the first 16 keys or, from i = 4 on, of the second; V^T comes
//    in that order from transposing LDS reads);
//  * a part that does not cover all keys of its rows leaves (sum, max, weight) in the workspace, and a second small
//    kernel joins the parts in key order, so results do not depend on timing.
// K and V pages are found 8 keys at a time (page sizes are multiples of 8); a page number that is none reads as zeros
// and is masked, as are rows at and past the sequence's end.
#include "paged_attn.hpp"

#include <algorithm>

#include "lds_dma.hpp"
#include "paged_types.hpp"

namespace lava {

constexpr int PR_BK = 128;      // keys of a block, 32 a wavefront
constexpr float PR_RESCALE = 8.f;   // the maximum moves when a score exceeds it by more than this: P <= 2^8

// ---- the plan -------------------------------------------------------------------------

// A sequence's (or the stacked prefix's) share of the work: key blocks [p0, p0 + np) of the prefix, then
// [o0, o0 + nb - np) of its own keys, for every row tile and key head.
struct PrSeq {
    uint32_t work;
    int tiles, nb, p0, np, o0;
};

__device__ __forceinline__ PrSeq pr_seq(const PaParams& p, const PagedSeq& s, int R) {
    PrSeq w = {};
    const int64_t rows = (int64_t)s.n * p.G;
    if (rows == 0 || rows > p.row_limit) return w;
    const int first = p.P + s.kv - s.n;
    const int lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
    if (p.P > 0 && !p.stack && lo < p.P) {
        w.p0 = lo / PR_BK;
        w.np = (p.P + PR_BK - 1) / PR_BK - w.p0;
    }
    const int own = max(0, lo - p.P);
    w.o0 = own / PR_BK;
    w.nb = max(1, w.np + (s.kv > own ? (s.kv + PR_BK - 1) / PR_BK - w.o0 : 0));   // rows without keys are written too
    w.tiles = ((int)rows + R - 1) / R;
    w.work = (uint32_t)w.tiles * (uint32_t)w.nb * (uint32_t)p.c.heads;
    return w;
}

__device__ __forceinline__ uint32_t pr_sum(uint32_t x) {
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i, 64);
    return x;
}
__device__ __forceinline__ uint32_t pr_scan(uint32_t x, int lane) {   // inclusive
    for (int i = 1; i < 64; i *= 2) {
        const uint32_t y = __shfl_up(x, i, 64);
        x += lane >= i ? y : 0;
    }
    return x;
}

// What every wavefront knows of the whole call.
struct PrPlan {
    uint32_t total, per;    // blocks of work, and of a workgroup
    PrSeq prefix;           // stack: the prefix for all rows together, in front of the sequences
    int t0, t1;             // rows of the batch
    bool plain;             // stack: every row sees the whole prefix
    uint32_t upto;          // lane i: the work of sequences 0 .. i (i < 64)
};

__device__ __forceinline__ PrPlan pr_plan(const PaParams& p, int R, int lane) {
    PrPlan g = {};
    uint32_t total = 0;
    int lo = 0x7fffffff;
    bool plain = p.window == 0;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        uint32_t work = 0;
        if (b0 + lane < p.b.B) {
            const PagedSeq s = paged_seq(p.b, b0 + lane);
            work = pr_seq(p, s, R).work;
            if (s.n > 0) {
                const int first = p.P + s.kv - s.n;
                lo = min(lo, p.window > 0 ? max(0, first - p.window + 1) : 0);
                plain = plain && s.n <= s.kv;
            }
        }
        const uint32_t upto = pr_scan(work, lane);
        if (b0 == 0) g.upto = upto;
        total += __builtin_amdgcn_readlane(upto, 63);
    }
    if (p.stack) {
        for (int i = 1; i < 64; i *= 2) lo = min(lo, __shfl_xor(lo, i, 64));
        lo = __builtin_amdgcn_readfirstlane(lo);
        g.plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
        g.t0 = min(max(p.b.q_start[0], 0), p.b.T);
        g.t1 = min(max(p.b.q_start[p.b.B], g.t0), p.b.T);
        if (lo < p.P && g.t1 > g.t0) {
            g.prefix.p0 = lo / PR_BK;
            g.prefix.np = g.prefix.nb = (p.P + PR_BK - 1) / PR_BK - g.prefix.p0;
            g.prefix.tiles = ((g.t1 - g.t0) * p.G + R - 1) / R;
            g.prefix.work = (uint32_t)g.prefix.tiles * (uint32_t)g.prefix.nb * (uint32_t)p.c.heads;
        }
    }
    g.total = total + g.prefix.work;
    return g;
}

// The sequence that holds block `w` of the work, and the work in front of it; -1: the stacked prefix.
__device__ __forceinline__ int pr_locate(const PaParams& p, const PrPlan& g, int R, uint32_t w, int lane, uint32_t& before) {
    before = 0;
    if (w < g.prefix.work) return -1;
    before = g.prefix.work;
    for (int b0 = 0; b0 < p.b.B; b0 += 64) {
        uint32_t upto = g.upto;
        if (b0 > 0) {
            uint32_t work = 0;
            if (b0 + lane < p.b.B) work = pr_seq(p, paged_seq(p.b, b0 + lane), R).work;
            upto = pr_scan(work, lane);
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

__device__ __forceinline__ uint32_t pr_per(uint32_t total) { return max(1u, (total + gridDim.x - 1) / gridDim.x); }

// ---- the kernel -----------------------------------------------------------------------

template <int N>
__device__ __forceinline__ void pr_wait() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ float pr_max4(float x) {   // over the four lanes of a row
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}

// DP: the head dimension rounded up to 64, 128 or 256; a tile is 16 NR rows.
template <typename T, int DP, int NR>
__global__ void __launch_bounds__(256, (DP <= 128 && NR <= 2) ? 2 : 1) paged_rows_kernel(PaParams p) {
    typedef PgType<T> TT;
    typedef typename TT::v8 v8;
    typedef typename TT::v4 v4;
    typedef __attribute__((address_space(3))) v8 lds_v8;
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    typedef __attribute__((address_space(3))) pg_s16x4 lds_s16x4;
    constexpr int R = 16 * NR;
    constexpr int CH = DP / 8, RB = DP * 2;        // 16-byte chunks and bytes of a staged row
    constexpr int RPI = 64 / CH;                   // rows a DMA instruction
    constexpr int NI = 32 / RPI;                   // DMA instructions a tile
    constexpr int IPG = 8 / RPI;                   // of those, per 8 keys
    constexpr int TILE = 32 * RB;
    constexpr int NKS = DP / 32, NDT = DP / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[4][2][TILE];   // per wavefront: K, V
    __shared__ float2 stat[4][R];
    auto kswz = [](int row) { return CH == 8 ? ((row & 7) ^ ((row >> 3) & 1)) : (row & 15); };
    auto vswz = [](int row) { return CH == 8 ? 2 * ((row >> 1) & 3) : 2 * (row & 7); };

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;

    const PrPlan plan = pr_plan(p, R, lane);
    const uint32_t total = __builtin_amdgcn_readfirstlane(plan.total);
    const uint32_t per = pr_per(total);
    const uint32_t begin = min(total, blockIdx.x * per), stop = min(total, begin + per);
    if (begin >= stop) return;

    // LDS-DMA: lane offsets within 8 keys, by the parity of the 8 and the instruction
    const uint32_t row_bytes = (uint32_t)(p.c.sl * 2);
    uint32_t ofs_k[2][IPG], ofs_v[IPG];
#pragma unroll
    for (int i = 0; i < IPG; ++i) {
        const int row = RPI * i + lane / CH;
#pragma unroll
        for (int par = 0; par < 2; ++par) {
            const int c = (lane % CH) ^ kswz(8 * par + row);
            ofs_k[par][i] = 8 * c < p.c.D ? (uint32_t)row * row_bytes + 16u * (uint32_t)c : OOB_OFS;
        }
        const int c = (lane % CH) ^ vswz(row);
        ofs_v[i] = 8 * c < p.c.D ? (uint32_t)row * row_bytes + 16u * (uint32_t)c : OOB_OFS;
    }
    const uint32_t lds_k = lds_addr(&ring[w][0][0]), lds_v = lds_addr(&ring[w][1][0]);
    uint32_t k_rd[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) k_rd[ks] = lds_k + (uint32_t)(r16 * RB + (((4 * ks + g) ^ kswz(r16)) << 4));
    // V^T: source lane (jj, q) of a 16-lane group addresses V[key 4 g + jj][16 dt + 4 q .. + 3]
    uint32_t v_rd[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
        const int jj = r16 >> 2, q = r16 & 3, row = 4 * g + jj;
        v_rd[dt] = lds_v + (uint32_t)(row * RB + (((2 * dt + (q >> 1)) ^ vswz(row)) << 4) + ((q & 1) << 3));
    }

    for (uint32_t at = begin; at < stop;) {
        // ---- the segment: a row tile of a sequence (or of the stacked prefix), some of its blocks
        uint32_t before;
        const int b = __builtin_amdgcn_readfirstlane(pr_locate(p, plan, R, at, lane, before));
        before = __builtin_amdgcn_readfirstlane(before);
        PagedSeq seq = {plan.t0, plan.t1 - plan.t0, 0};
        PrSeq sw = plan.prefix;
        if (b >= 0) {
            seq = paged_seq(p.b, b);
            sw = pr_seq(p, seq, R);
        }
        const int nb = __builtin_amdgcn_readfirstlane(sw.nb), np = __builtin_amdgcn_readfirstlane(sw.np);
        const int p0 = __builtin_amdgcn_readfirstlane(sw.p0), o0 = __builtin_amdgcn_readfirstlane(sw.o0);
        const uint32_t tiles = __builtin_amdgcn_readfirstlane(sw.tiles);
        const uint32_t rel = at - before, ht = rel / (uint32_t)nb;
        const int blk0 = (int)(rel - ht * (uint32_t)nb);
        const int head = (int)(ht / tiles), tile = (int)(ht - (uint32_t)head * tiles);
        const int nblk = min(nb - blk0, (int)(stop - at));
        const int kv = __builtin_amdgcn_readfirstlane(seq.kv);

        // ---- the rows of this lane
        v8 qf[NR][NKS];
        int row_t[NR], row_h[NR], lo[NR], hi[NR];
        float pos[NR], slope[NR];
        bool live[NR];
        int lo_max = 0, hi_min = 0x7fffffff;
        const int bid = (b >= 0 && p.bidir) ? p.bidir[b] : 0;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const uint32_t row = (uint32_t)(tile * R + 16 * nr + r16);
            const int i = (int)div_of(row, p.by_g);
            live[nr] = i < seq.n;
            row_t[nr] = seq.first + i;
            row_h[nr] = head * p.G + (int)(row - (uint32_t)(i * p.G));
            int end = p.P + kv, at_pos = end - seq.n + i;
            lo[nr] = 0;
            hi[nr] = 0x7fffffff;
            if (b < 0) {
                end = p.P;
                at_pos = p.P;
                if ((!plan.plain || p.slopes) && live[nr]) {
                    // the row's sequence: the first whose end lies behind it
                    int a = 0, z = p.b.B;
                    while (a < z) {
                        const int mid = (a + z) >> 1;
                        if (min(p.b.q_start[mid + 1], p.b.T) <= row_t[nr]) a = mid + 1;
                        else z = mid;
                    }
                    if (a < p.b.B) {
                        const PagedSeq s = paged_seq(p.b, a);
                        at_pos = p.P + s.kv - s.n + (row_t[nr] - s.first);
                    }
                }
            }
            if (live[nr]) {
                const PaRange rg = pa_range(p, at_pos, end, bid);
                lo[nr] = rg.lo;
                hi[nr] = rg.hi;
            }
            pos[nr] = (float)at_pos;
            slope[nr] = (p.slopes && live[nr]) ? p.slopes[row_h[nr]] * PA_LOG2E : 0.f;
            lo_max = max(lo_max, lo[nr]);
            hi_min = min(hi_min, hi[nr]);
            const T* qr = (const T*)p.Q + (int64_t)row_t[nr] * p.qst + (int64_t)row_h[nr] * p.qsh + 8 * g;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                qf[nr][ks] = v8{};
                if (live[nr] && 32 * ks + 8 * g < p.c.D) qf[nr][ks] = *reinterpret_cast<const v8*>(qr + 32 * ks);
            }
        }
        for (int i = 1; i < 16; i *= 2) {
            lo_max = max(lo_max, __shfl_xor(lo_max, i, 64));
            hi_min = min(hi_min, __shfl_xor(hi_min, i, 64));
        }
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
        hi_min = __builtin_amdgcn_readfirstlane(hi_min);

        // ---- this wavefront's tile of block j: where its keys are
        struct Tile {
            int page[4], row[4], n[4];   // per 8 keys: the page (-1: none), the row in it, keys below the end
            int pos;                     // position of the first key
            int last;                    // of the source's last key
        };
        const pg_table own = (pg_table)(uintptr_t)(p.b.table + (int64_t)max(b, 0) * p.b.max_pages);
        const pg_table shared = (pg_table)(uintptr_t)p.ppages;
        auto lookup = [&](int j) __attribute__((always_inline)) {
            Tile t;
            const int blk = blk0 + j;
            const bool pre = blk < np;
            const int key0 = (pre ? p0 + blk : o0 + blk - np) * PR_BK + 32 * w;
            const int len = j < nblk ? (pre ? p.P : kv) : 0;
            t.pos = key0 + (pre ? 0 : p.P);
            t.last = pre ? p.P - 1 : p.P + kv - 1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = key0 + 8 * i;
                t.n[i] = min(max(len - k, 0), 8);
                t.page[i] = 0;
                t.row[i] = 0;
                if (t.n[i] > 0) {
                    const int no = (int)div_of((uint32_t)k, p.c.by_page);
                    t.row[i] = k - no * p.c.page;
                    const int pg = pre ? shared[no] : own[no];
                    t.page[i] = (uint32_t)pg < (uint32_t)p.c.pages ? pg : -1;
                }
            }
            return t;
        };
        auto request = [&](const Tile& t, bool is_k) __attribute__((always_inline)) {
            const T* base = (const T*)(is_k ? p.c.k : p.c.v) + (int64_t)head * p.c.sh;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool none = t.page[i] < 0 || t.n[i] == 0;
                const T* at8 = base + (none ? 0 : (int64_t)t.page[i] * p.c.sp + (int64_t)t.row[i] * p.c.sl);
                const uint32_t bytes = none ? 0u : (uint32_t)(t.n[i] - 1) * row_bytes + 2u * (uint32_t)p.c.D;
                const v4i rs = make_rsrc(at8, bytes);
#pragma unroll
                for (int u = 0; u < IPG; ++u)
                    dma16(rs, is_k ? ofs_k[i & 1][u] : ofs_v[u], 0u,
                          __builtin_amdgcn_readfirstlane((is_k ? lds_k : lds_v) + 1024u * (uint32_t)(i * IPG + u)));
            }
        };

        // Q and the slopes are used here, so that the compiler waits for their loads now and not in the loop, where its
        // wait (it does not count the DMAs) would be for everything in flight
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const uint4 u = __builtin_bit_cast(uint4, qf[nr][ks]);
                asm volatile("" ::"v"(u.x), "v"(u.y), "v"(u.z), "v"(u.w));
            }
            asm volatile("" ::"v"(slope[nr]));
        }
        f32x4 o[NDT][NR];
        float m[NR], l[NR];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            m[nr] = -INFINITY;
            l[nr] = 0.f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt][nr] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        __syncthreads();   // the segment before has left the ring and the statistics
        Tile now = lookup(0), next = lookup(1);
        request(now, true);
        request(now, false);
        for (int j = 0; j < nblk; ++j) {
            pr_wait<NI>();   // K is here, V may not be
            f32x4 st[2][NR];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) st[kt][nr] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const v8 a = *(const lds_v8*)(uintptr_t)(k_rd[ks] + (uint32_t)(16 * kt * RB));
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) st[kt][nr] = TT::mma16(a, qf[nr][ks], st[kt][nr]);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K's place is read
            request(next, true);

            const int first = now.pos, none = (now.page[0] < 0) | (now.page[1] < 0) << 1 | (now.page[2] < 0) << 2 | (now.page[3] < 0) << 3;
            const bool cut = none != 0 || first < lo_max || first + 31 > min(hi_min, now.last);
            float up[NR];
            bool move = false;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float top = -INFINITY;
                const int last = min(hi[nr], now.last);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = first + 16 * kt + 4 * g + r;
                        float x = pa_score(st[kt][nr][r], p.mul, p.cap2);
                        if (p.slopes) x = fmaf(-slope[nr], fabsf(pos[nr] - (float)key), x);
                        if (cut) {
                            const bool keep = key >= lo[nr] && key <= last && !((none >> (2 * kt + (g >> 1))) & 1);
                            x = keep ? x : -INFINITY;
                        }
                        st[kt][nr][r] = x;
                        top = fmaxf(top, x);
                    }
                up[nr] = top;
                move = move || top > m[nr] + PR_RESCALE;
            }
            if (__builtin_amdgcn_ballot_w64(move) != 0) {
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    const float mn = fmaxf(m[nr], pr_max4(up[nr]));
                    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[nr] - mn);
                    m[nr] = mn;
                    l[nr] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt) o[dt][nr] *= alpha;
                }
            }
            v8 pf[NR];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                const float sub = m[nr] == -INFINITY ? 0.f : m[nr];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const T q = (T)__builtin_amdgcn_exp2f(st[e >> 2][nr][e & 3] - sub);
                    pf[nr][e] = q;
                    l[nr] += (float)q;   // the sum is of what is multiplied
                }
            }
            pr_wait<NI>();   // V is here
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const pg_s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)v_rd[dt]);
                const pg_s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(v_rd[dt] + (uint32_t)(16 * RB)));
                const v8 a = __builtin_bit_cast(v8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) o[dt][nr] = TT::mma16(a, pf[nr], o[dt][nr]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V's place is read
            request(next, false);
            now = next;
            next = lookup(j + 2);
        }

        // ---- the four wavefronts' parts together, two row sixteens at a time through the ring
        pr_wait<0>();
        float f[NR], ml[NR], ll[NR];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            l[nr] += __shfl_xor(l[nr], 16, 64);
            l[nr] += __shfl_xor(l[nr], 32, 64);
            if (g == 0) stat[w][16 * nr + r16] = make_float2(m[nr], l[nr]);
        }
        __syncthreads();
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            ml[nr] = -INFINITY;
            ll[nr] = 0.f;
            float2 s4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s4[i] = stat[i][16 * nr + r16];
                ml[nr] = fmaxf(ml[nr], s4[i].x);
            }
            const float sub = ml[nr] == -INFINITY ? 0.f : ml[nr];
#pragma unroll
            for (int i = 0; i < 4; ++i) ll[nr] += s4[i].y * __builtin_amdgcn_exp2f(s4[i].x - sub);
            f[nr] = __builtin_amdgcn_exp2f(m[nr] - sub);
        }
        const bool whole = nblk == nb, direct = whole && !p.stack;
        constexpr int NH = NR < 2 ? 1 : 2;
        const uint32_t box = lds_addr(&ring[0][0][0]) + 16u * (uint32_t)lane;
#pragma unroll
        for (int n0 = 0; n0 < NR; n0 += NH) {
            if (n0 > 0) __syncthreads();
#pragma unroll
            for (int u = 0; u < NH; ++u)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
                    *(lds_f32x4*)(uintptr_t)(box + 1024u * (uint32_t)((w * NH + u) * NDT + dt)) = o[dt][n0 + u] * f[n0 + u];
            __syncthreads();
#pragma unroll
            for (int u = 0; u < NH; ++u) {
                const int nr = n0 + u;
                const int64_t out_row = (int64_t)row_t[nr] * p.Hq + row_h[nr];
                const float inv = ll[nr] == 0.f ? 0.f : 1.f / ll[nr];
                T* orow = (T*)p.O + (int64_t)row_t[nr] * p.ost + (int64_t)row_h[nr] * p.osh + 4 * g;
                float* prow;
                float2* pml;
                if (whole) {
                    const int64_t i = (b < 0 ? 0 : (int64_t)p.b.T * p.Hq) + out_row;
                    prow = p.row_o + i * DP;
                    pml = p.row_ml + i;
                } else {
                    const int64_t i = (int64_t)(2 * blockIdx.x + (blk0 == 0 ? 1 : 0)) * R + 16 * nr + r16;
                    prow = p.ws_o + i * DP;
                    pml = p.ws_ml + i;
                }
#pragma unroll
                for (int d4 = 0; d4 < NDT / 4; ++d4) {
                    const int dt = 4 * d4 + w;
                    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 4; ++i) x += *(const lds_f32x4*)(uintptr_t)(box + 1024u * (uint32_t)((i * NH + u) * NDT + dt));
                    if (!live[nr]) continue;
                    if (direct) {
                        const v4 y = {(T)(x[0] * inv), (T)(x[1] * inv), (T)(x[2] * inv), (T)(x[3] * inv)};
                        if (16 * dt + 4 * g < p.c.D) *reinterpret_cast<v4*>(orow + 16 * dt) = y;
                    } else {
                        *reinterpret_cast<f32x4*>(prow + 16 * dt + 4 * g) = x;
                    }
                }
                if (live[nr] && w == 0 && g == 0) {
                    if (direct) {
                        if (p.lse) p.lse[out_row] = ll[nr] == 0.f ? -INFINITY : (ml[nr] + log2f(ll[nr])) * PA_LN2;
                    } else {
                        *pml = make_float2(ml[nr], ll[nr]);
                    }
                }
            }
        }
        at += (uint32_t)nblk;
    }
}

// Joins the parts of every row that has more than one: the prefix's (stacked) and its sequence's, each in the order of
// its keys.  One wavefront a row; a lane holds DP / 64 columns.
template <typename T, int DP>
__global__ void __launch_bounds__(256) paged_join_kernel(PaParams p, int R, uint32_t parts) {
    constexpr int NC = DP / 64;
    typedef float vf __attribute__((ext_vector_type(NC)));
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)p.b.T * p.Hq) return;
    const int t = __builtin_amdgcn_readfirstlane((int)(row / p.Hq)), h = __builtin_amdgcn_readfirstlane((int)(row % p.Hq));
    const int b = paged_find(p.b, t, lane);
    if (b >= p.b.B) return;
    const PagedSeq s = paged_seq(p.b, b);
    if (t < s.first || t >= s.first + s.n || (int64_t)s.n * p.G > p.row_limit) return;
    const PrPlan plan = pr_plan(p, R, lane);
    const uint32_t per = max(1u, (plan.total + parts - 1) / parts);
    const int head = h / p.G;
    uint32_t before = plan.prefix.work;
    for (int b0 = 0; b0 < b; b0 += 64) {
        uint32_t upto = plan.upto;
        if (b0 > 0) {
            uint32_t work = 0;
            if (b0 + lane < p.b.B) work = pr_seq(p, paged_seq(p.b, b0 + lane), R).work;
            upto = pr_scan(work, lane);
        }
        before += __builtin_amdgcn_readlane(upto, min(b - b0, 64) - 1);
    }
    float m = -INFINITY, l = 0.f;
    vf o = {};
    auto take = [&](const float* po, float2 ml) {
        const float mn = fmaxf(m, ml.x), sub = mn == -INFINITY ? 0.f : mn;
        const float a = __builtin_amdgcn_exp2f(m - sub), c = __builtin_amdgcn_exp2f(ml.x - sub);
        o = o * a + *reinterpret_cast<const vf*>(po + NC * lane) * c;
        l = l * a + ml.y * c;
        m = mn;
    };
    // one row tile's parts: false if its one part has written O already
    auto source = [&](const PrSeq& sw, uint32_t w0, uint32_t r, int which) {
        const uint32_t tile = r / (uint32_t)R, in = r - tile * (uint32_t)R;
        const uint32_t a = w0 + ((uint32_t)head * (uint32_t)sw.tiles + tile) * (uint32_t)sw.nb, z = a + (uint32_t)sw.nb - 1;
        const uint32_t i0 = a / per, i1 = z / per;
        if (i0 == i1) {
            if (!p.stack) return false;
            const int64_t i = (int64_t)which * p.b.T * p.Hq + row;
            take(p.row_o + i * DP, p.row_ml[i]);
            return true;
        }
        for (uint32_t i = i0; i <= i1; ++i) {
            const int64_t k = (int64_t)(2 * i + (a >= i * per ? 1 : 0)) * R + in;
            take(p.ws_o + k * DP, p.ws_ml[k]);
        }
        return true;
    };
    bool any = false;
    if (plan.prefix.work > 0) any = source(plan.prefix, 0, (uint32_t)((t - plan.t0) * p.G + h % p.G), 0);
    any = source(pr_seq(p, s, R), before, (uint32_t)((t - s.first) * p.G + h % p.G), 1) || any;
    if (!any) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* orow = (T*)p.O + (int64_t)t * p.ost + (int64_t)h * p.osh + NC * lane;
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (NC * lane + i < p.c.D) orow[i] = (T)(o[i] * inv);
    if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * PA_LN2;
}

// ---- host -----------------------------------------------------------------------------

constexpr int PR_CUS = 256;

struct PrShape {
    int dp, nr;
    unsigned grid;
    size_t slots, rows;    // partial results, whole ones
};

static PrShape pr_shape(const PaParams& p, int64_t max_rows) {
    PrShape s;
    s.dp = p.c.D <= 64 ? 64 : p.c.D <= 128 ? 128 : 256;
    if (p.stack) max_rows = std::max<int64_t>(max_rows, (int64_t)p.b.T * p.G);
    s.nr = max_rows <= 16 ? 1 : max_rows <= 32 || s.dp == 256 ? 2 : 4;
    const int wgs = s.dp == 64 && s.nr <= 2 ? 4 : s.dp <= 128 && s.nr <= 2 ? 2 : 1;
    s.grid = (unsigned)(PR_CUS * wgs);
    s.slots = (size_t)s.grid * 2 * 16 * s.nr;
    s.rows = p.stack ? (size_t)2 * p.b.T * p.Hq : 0;
    return s;
}

size_t paged_rows_workspace(const PaParams& p, int64_t max_rows) {
    const PrShape s = pr_shape(p, max_rows);
    return (s.slots + s.rows) * (s.dp * sizeof(float) + sizeof(float2)) + 512;
}

// Whether the call's blocks of work can be counted in 31 bits.
bool paged_rows_fits(const PaParams& p) {
    const double tiles = (double)p.b.T * p.G / 16 + 2.0 * p.b.B + 1;
    const double blocks = ((double)p.b.kv_max + p.P) / PR_BK + 4;
    return tiles * blocks * p.c.heads < 2147483647.0 && (int64_t)p.b.T * p.G <= 0x7fffff00;
}

int paged_rows_launch(PaParams& p, int dtype, int64_t max_rows, void* ws, hipStream_t s) {
    const PrShape sh = pr_shape(p, max_rows);
    uint8_t* at = (uint8_t*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    auto take = [&](size_t bytes) {
        uint8_t* q = at;
        at += bytes;
        return q;
    };
    p.ws_o = (float*)take(sh.slots * sh.dp * sizeof(float));
    p.row_o = (float*)take(sh.rows * sh.dp * sizeof(float));
    p.ws_ml = (float2*)take(sh.slots * sizeof(float2));
    p.row_ml = (float2*)take(sh.rows * sizeof(float2));
    auto by_type = [&](auto tag) {
        typedef decltype(tag) T;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(sh.grid), dim3(256), 0, s, p); };
        if (sh.dp == 64)
            sh.nr == 1 ? go(paged_rows_kernel<T, 64, 1>) : sh.nr == 2 ? go(paged_rows_kernel<T, 64, 2>) : go(paged_rows_kernel<T, 64, 4>);
        else if (sh.dp == 128)
            sh.nr == 1 ? go(paged_rows_kernel<T, 128, 1>) : sh.nr == 2 ? go(paged_rows_kernel<T, 128, 2>) : go(paged_rows_kernel<T, 128, 4>);
        else
            sh.nr == 1 ? go(paged_rows_kernel<T, 256, 1>) : go(paged_rows_kernel<T, 256, 2>);
        const int rc = check_launch("paged_rows_kernel");
        if (rc != LAVA_HIP_OK) return rc;
        const unsigned rows = (unsigned)(((int64_t)p.b.T * p.Hq + 3) / 4);
        auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(rows), dim3(256), 0, s, p, 16 * sh.nr, sh.grid); };
        sh.dp == 64 ? join(paged_join_kernel<T, 64>) : sh.dp == 128 ? join(paged_join_kernel<T, 128>) : join(paged_join_kernel<T, 256>);
        return check_launch("paged_join_kernel");
    };
    return dtype == LAVA_HIP_F16 ? by_type(f16{}) : by_type(bf16{});
}

}  // namespace lava
