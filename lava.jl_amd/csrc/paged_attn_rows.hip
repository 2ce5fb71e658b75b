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
//  * parts that do not cover all keys of their rows are joined in key order by the last workgroup of a row tile to
//    arrive (paged_plan.hpp), so results do not depend on timing; behind a stacked prefix by a second small kernel.
// K and V pages are found 8 keys at a time (page sizes are multiples of 8); a page number that is none reads as zeros
// and is masked, as are rows at and past the sequence's end.

#include <algorithm>

#include "lds_dma.hpp"
#include "paged_plan.hpp"
#include "paged_types.hpp"

namespace lava {

constexpr float PR_RESCALE = 8.f;   // the maximum moves when a score exceeds it by more than this: P <= 2^8

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
    __shared__ int arrived;
    auto kswz = [](int row) { return CH == 8 ? ((row & 7) ^ ((row >> 3) & 1)) : (row & 15); };
    auto vswz = [](int row) { return CH == 8 ? 2 * ((row >> 1) & 3) : 2 * (row & 7); };

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;

    const PaPlan plan = pa_plan<PR_BK, false>(p, R, true, p.stack == 1, lane);
    const uint32_t total = __builtin_amdgcn_readfirstlane(plan.total);
    const uint32_t per = pa_per(total, gridDim.x), wg = pa_place(gridDim.x);
    const uint32_t begin = min(total, wg * per), stop = min(total, begin + per);
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
        const int b = __builtin_amdgcn_readfirstlane(pa_locate<PR_BK, false>(p, plan, R, at, lane, before));
        before = __builtin_amdgcn_readfirstlane(before);
        PagedSeq seq = {plan.t0, plan.t1 - plan.t0, 0};
        PaSeq sw = plan.prefix;
        if (b >= 0) {
            seq = paged_seq(p.b, b);
            sw = pa_seq<PR_BK, false>(p, seq, R);
        }
        const int nb = __builtin_amdgcn_readfirstlane(sw.nb), np = __builtin_amdgcn_readfirstlane(sw.np);
        const int p0 = __builtin_amdgcn_readfirstlane(sw.p0), o0 = __builtin_amdgcn_readfirstlane(sw.o0);
        const uint32_t tiles = __builtin_amdgcn_readfirstlane(sw.tiles);
        const uint32_t rel = at - before, ht = rel / (uint32_t)nb;
        const int blk0 = (int)(rel - ht * (uint32_t)nb);
        const int head = (int)(ht / tiles), tile = (int)(ht - (uint32_t)head * tiles);
        const int nblk = min(nb - blk0, (int)(stop - at));
        const int kv = __builtin_amdgcn_readfirstlane(seq.kv);

        // rows of a sequence that another launch takes, prefix and all
        if (b < 0 && pa_other(p, seq.first + tile * R / p.G, seq.first + min(seq.n - 1, (tile * R + R - 1) / p.G), lane)) {
            at += (uint32_t)nblk;
            continue;
        }

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
                if ((!plan.plain || p.slopes) && live[nr]) at_pos = pa_row_pos(p, row_t[nr]);
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
                const int64_t part = whole ? (b < 0 ? 0 : (int64_t)p.b.T * p.Hq) + out_row
                                           : (int64_t)(2 * wg + (blk0 == 0 ? 1 : 0)) * R + 16 * nr + r16;
                float* prow = (whole ? p.row_o : p.ws_o) + part * DP + 4 * g;
                float2* pml = (whole ? p.row_ml : p.ws_ml) + part;
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
                        pa_put(prow + 16 * dt, x[0], x[1]);
                        pa_put(prow + 16 * dt + 2, x[2], x[3]);
                    }
                }
                if (live[nr] && w == 0 && g == 0) {
                    if (direct) {
                        if (p.lse) p.lse[out_row] = ll[nr] == 0.f ? -INFINITY : (ml[nr] + log2f(ll[nr])) * PA_LN2;
                    } else {
                        pa_put((float*)pml, ml[nr], ll[nr]);
                    }
                }
            }
        }
        if (!whole && p.stack == 0) {
            const uint32_t a = before + ht * (uint32_t)nb;   // the tile's first block
            pa_arrive<T, DP, 4>(p, a / per, (a + (uint32_t)nb - 1) / per, R, min(R, seq.n * p.G - tile * R), tile * R, seq.first,
                                head, w, lane, &arrived);
        }
        at += (uint32_t)nblk;
    }
}

// Behind a stacked prefix: a row's parts, the prefix's and its sequence's, each in the order of its keys.  One
// wavefront a row.
template <typename T, int DP>
__global__ void __launch_bounds__(256) paged_join_kernel(PaParams p, int R, uint32_t row_grid, int pre_R) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)p.b.T * p.Hq) return;
    const int t = __builtin_amdgcn_readfirstlane((int)(row / p.Hq)), h = __builtin_amdgcn_readfirstlane((int)(row % p.Hq));
    const int b = paged_find(p.b, t, lane);
    if (b >= p.b.B) return;
    const PagedSeq s = paged_seq(p.b, b);
    if (t < s.first || t >= s.first + s.n || (int64_t)s.n * p.G > p.row_limit) return;
    // a tile's parts: whole (one, by row), or those of workgroups i0 .. i0 + n - 1
    struct Source {
        const float* o;
        const float2* ml;
        uint32_t i0;
        int n, R, in;
        __device__ int64_t at(int j) const { return n == 1 ? in : (int64_t)(2 * (i0 + (uint32_t)j) + (j == 0 ? 1u : 0u)) * R + in; }
    };
    const int head = h / p.G, g = h - head * p.G;
    auto source = [&](const PaSeq& sw, uint32_t before, uint32_t per, int tile_rows, uint32_t r, const float* o, const float2* ml,
                      int which) {
        const uint32_t tile = r / (uint32_t)tile_rows;
        const uint32_t a = before + ((uint32_t)head * (uint32_t)sw.tiles + tile) * (uint32_t)sw.nb, z = a + (uint32_t)sw.nb - 1;
        Source x;
        x.i0 = a / per;
        x.n = (int)(z / per - x.i0) + 1;
        x.R = tile_rows;
        const bool whole = x.n == 1;
        x.in = whole ? 0 : (int)(r - tile * (uint32_t)tile_rows);
        const int64_t i = (int64_t)which * p.b.T * p.Hq + row;
        x.o = whole ? p.row_o + i * DP : o;
        x.ml = whole ? p.row_ml + i : ml;
        return x;
    };
    const PaPlan plan = pa_plan<PR_BK, false>(p, R, true, p.stack == 1, lane);
    uint32_t before = plan.prefix.work;
    for (int b0 = 0; b0 < b; b0 += 64) {
        uint32_t upto = plan.upto;
        if (b0 > 0) {
            uint32_t work = 0;
            if (b0 + lane < p.b.B) work = pa_seq<PR_BK, false>(p, paged_seq(p.b, b0 + lane), R).work;
            upto = pa_scan(work, lane);
        }
        before += __builtin_amdgcn_readlane(upto, min(b - b0, 64) - 1);
    }
    const uint32_t per = pa_per(plan.total, row_grid);
    const Source own = source(pa_seq<PR_BK, false>(p, s, R), before, per, R, (uint32_t)((t - s.first) * p.G + g), p.ws_o, p.ws_ml, 1);
    Source pre = own;
    pre.n = 0;
    if (p.stack == 1) {
        if (plan.prefix.work > 0) pre = source(plan.prefix, 0, per, R, (uint32_t)((t - plan.t0) * p.G + g), p.ws_o, p.ws_ml, 0);
    } else {
        const PaPlan pp = pa_plan<PT_BK, true>(p, pre_R, false, true, lane);
        if (pp.prefix.work > 0)
            pre = source(pp.prefix, 0, pa_per(pp.total, PT_GRID), pre_R, (uint32_t)((t - pp.t0) * p.G + g), p.pre_o, p.pre_ml, 0);
    }
    float o[DP / 64], m, l;
    pa_join_row<DP>(pre.n + own.n, [&](int j) { return j < pre.n ? pre.ml + pre.at(j) : own.ml + own.at(j - pre.n); },
                    [&](int j) { return j < pre.n ? pre.o + pre.at(j) * DP : own.o + own.at(j - pre.n) * DP; }, lane, o, m, l);
    pa_store_row<T, DP>(p, t, h, o, m, l, lane);
}

int paged_rows_launch(const PaParams& p, const PaShape& sh, int dtype, hipStream_t s) {
    auto by_type = [&](auto tag) {
        typedef decltype(tag) T;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(sh.row_grid), dim3(256), 0, s, p); };
        if (sh.dp == 64)
            sh.nr == 1 ? go(paged_rows_kernel<T, 64, 1>) : sh.nr == 2 ? go(paged_rows_kernel<T, 64, 2>) : go(paged_rows_kernel<T, 64, 4>);
        else if (sh.dp == 128)
            sh.nr == 1 ? go(paged_rows_kernel<T, 128, 1>) : sh.nr == 2 ? go(paged_rows_kernel<T, 128, 2>) : go(paged_rows_kernel<T, 128, 4>);
        else
            sh.nr == 1 ? go(paged_rows_kernel<T, 256, 1>) : go(paged_rows_kernel<T, 256, 2>);
        int rc = check_launch("paged_rows_kernel");
        if (rc != LAVA_HIP_OK || p.stack == 0) return rc;
        const unsigned rows = (unsigned)(((int64_t)p.b.T * p.Hq + 3) / 4);
        auto join = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(rows), dim3(256), 0, s, p, 16 * sh.nr, sh.row_grid, 128 * sh.pre_qh);
        };
        sh.dp == 64 ? join(paged_join_kernel<T, 64>) : sh.dp == 128 ? join(paged_join_kernel<T, 128>) : join(paged_join_kernel<T, 256>);
        return check_launch("paged_join_kernel");
    };
    return dtype == LAVA_HIP_F16 ? by_type(f16{}) : by_type(bf16{});
}

}  // namespace lava
