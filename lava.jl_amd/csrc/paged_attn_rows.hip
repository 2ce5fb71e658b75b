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
//  * parts that do not cover all keys of their rows are joined in key order (paged_plan.hpp), so results do not depend on
//    timing: those of tiles of 16 rows by the last workgroup of a tile to arrive, others by a second small kernel.
// K and V pages are found 8 keys at a time (page sizes are multiples of 8); a page number that is none reads as zeros
// and is masked, as are rows at and past the sequence's end.
// Measured (calls in a row): 64 decoded tokens, 32 heads on 8, D = 128, 100 to 8192 keys each 217 us, 5.5 TB/s of the cache read; one
// of 777 keys 9.6 us, a chain of five dependent reads; 3 of 30000 to 131071 keys on 2 key heads, capped, 55 (60 over changing inputs,
// which no cache holds); 32 sequences of 1 to 4 drafted tokens, 12 heads of D = 64, windows of 1024 and slopes, 24.

#include <algorithm>

#include "lds_dma.hpp"
#include "paged_plan.hpp"

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

// DP: the head dimension rounded up to 64, 128 or 256; a tile is 16 NR rows, NR 1 or 2.
template <typename T, int DP, int NR, bool PRE>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) paged_rows_kernel(PaParams) {
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
    // parts are joined in this launch, by paged_join_tiles_kernel, or (behind a stacked prefix) by paged_join_kernel
    constexpr bool LIVE = NR == 1 && !PRE, LATER = NR == 2 && !PRE;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[4][2][TILE];   // per wavefront: K, V
    __shared__ float2 stat[4][R];
    __shared__ int arrived;
    auto kswz = [](int row) { return CH == 8 ? ((row & 7) ^ ((row >> 3) & 1)) : (row & 15); };
    auto vswz = [](int row) { return CH == 8 ? 2 * ((row >> 1) & 3) : 2 * (row & 7); };

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;

    PaArgs args;
    args.load(lane);
    const PaParams p = args.get();
    const PaPlan plan = pa_plan<PR_BK, false, PRE>(p, R, true, PRE && p.stack == 1, lane);
    const uint32_t per = pa_per(plan.total, p.by_rows, 1), wg = blockIdx.x;
    const uint32_t begin = min(plan.total, wg * per), stop = min(plan.total, begin + per);
    PaOpen open = {};
    if (begin >= stop) {
        if (LATER) pa_leave_open(p.ws_open + wg, open);
        return;
    }

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
        const PaParams p = args.get();
        const PaSegment sg = pa_segment<PR_BK, false, PRE>(p, plan, R, at, lane);
        const int b = sg.b, nb = sg.sw.nb, np = PRE ? sg.sw.np : 0, p0 = sg.sw.p0, o0 = sg.sw.o0;
        const int head = sg.head, tile = sg.tile, blk0 = sg.blk0, kv = sg.seq.kv, rows = sg.seq.n * p.G;
        const int nblk = min(nb - blk0, (int)(stop - at));

        // ---- the rows of this lane; the last position that the first row sees and the first that the last one does
        // bound what needs comparing (rows are in order of their positions)
        v8 qf[NR][NKS];
        int row_t[NR], row_h[NR], lo[NR], hi[NR];
        int pos[NR];
        float slope[NR];
        bool live[NR];
        const int bid = pa_leading(p, b);
        const int end = PRE ? p.P + kv : kv, pos0 = end - sg.seq.n;   // of a prefix tile: P
        int lo_max = pa_range(p, pos0 + (int)div_of((uint32_t)min(tile * R + R - 1, rows - 1), p.by_g), end, bid).lo;
        int hi_min = pa_range(p, pos0 + (int)div_of((uint32_t)(tile * R), p.by_g), end, bid).hi;
        if (PRE && b < 0) {
            lo_max = plan.plain ? 0 : 0x7fffffff;
            hi_min = p.P - 1;
        }
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
        hi_min = __builtin_amdgcn_readfirstlane(hi_min);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const uint32_t row = (uint32_t)(tile * R + 16 * nr + r16);
            const int i = (int)div_of(row, p.by_g);
            live[nr] = (int)row < rows;
            row_t[nr] = sg.seq.first + i;
            row_h[nr] = head * p.G + (int)row - i * p.G;
            int at_pos = pos0 + i;
            if (PRE && b < 0) {
                at_pos = p.P;
                if ((!plan.plain || p.slopes) && live[nr]) at_pos = pa_row_pos(p, row_t[nr]);
            }
            const PaRange rg = pa_range(p, at_pos, end, bid);
            lo[nr] = rg.lo;
            hi[nr] = rg.hi;
            pos[nr] = at_pos;
            slope[nr] = 0.f;
            if (p.slopes && live[nr]) slope[nr] = p.slopes[row_h[nr]] * PA_LOG2E;
            const T* qr = (const T*)p.Q + (int64_t)row_t[nr] * p.qst + (int64_t)row_h[nr] * p.qsh + 8 * g;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                qf[nr][ks] = v8{};
                if (live[nr] && 32 * ks + 8 * g < p.c.D) qf[nr][ks] = *reinterpret_cast<const v8*>(qr + 32 * ks);
            }
        }

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
        {
        const PaParams p = args.get();
        // ---- this wavefront's tiles, 32 keys of a block
        PaPages<4, PRE> pages = {-1, -1};
        auto where = [&](int j, int i, int& k, bool& pre) {
            const int blk = blk0 + j;
            pre = PRE && blk < np;
            k = (pre ? p0 + blk : o0 + blk - np) * PR_BK + 32 * w + 8 * i;
            return j < nblk && k < (pre ? p.P : kv);
        };
        pages.load(p, b, 0, lane, where);
        if (nblk + 1 >= decltype(pages)::TPC) pages.load(p, b, 1, lane, where);   // lookups run two tiles ahead
        struct Tile {
            int64_t at[4];   // per 8 keys, -1: none
            int left;        // keys from the first to the end of the source
            int pos;         // position of the first key
        };
        auto lookup = [&](int j) __attribute__((always_inline)) {
            Tile t;
            const int blk = blk0 + j;
            const bool pre = PRE && blk < np;
            const int key0 = (pre ? p0 + blk : o0 + blk - np) * PR_BK + 32 * w;
            t.pos = key0 + (pre || !PRE ? 0 : p.P);
            t.left = (pre ? p.P : kv) - key0;
#pragma unroll
            for (int i = 0; i < 4; ++i) t.at[i] = pages.get(j, i);
            return t;
        };
        auto request = [&](const Tile& t, bool is_k) __attribute__((always_inline)) {
            const T* base = (const T*)(is_k ? p.c.k : p.c.v) + (int64_t)head * p.c.sh;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t o = t.at[i];
                const uint32_t bytes = o < 0 ? 0u : (uint32_t)(min(t.left - 8 * i, 8) - 1) * row_bytes + 2u * (uint32_t)p.c.D;
                const v4i rs = make_rsrc(base + o, bytes);   // none: nothing in range
#pragma unroll
                for (int u = 0; u < IPG; ++u)
                    dma16(rs, is_k ? ofs_k[i & 1][u] : ofs_v[u], 0u,
                          __builtin_amdgcn_readfirstlane((is_k ? lds_k : lds_v) + 1024u * (uint32_t)(i * IPG + u)));
            }
        };

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

            const int first = now.pos, none = (now.at[0] < 0) | (now.at[1] < 0) << 1 | (now.at[2] < 0) << 2 | (now.at[3] < 0) << 3;
            const int end_pos = first + now.left - 1;   // the source's last key
            // keys that some row does not see and that have values (those past the end read as zeros)
            const bool part_seen = first < lo_max || min(first + 31, end_pos) > hi_min;
            const bool cut = part_seen || none != 0 || first + 31 > end_pos;
            bool near = false;   // with a cap: every score in the polynomial's range
            if (p.cap2 != 0.f) {
                float far = 0.f;
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int e = 0; e < 8; ++e) far = fmaxf(far, fabsf(st[e >> 2][nr][e & 3]));
                near = __builtin_amdgcn_ballot_w64(far > p.near) == 0;
            }
            float up[NR];
            bool move = false;
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float top = -INFINITY;
                const int last = min(hi[nr], end_pos);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = first + 16 * kt + 4 * g + r;
                        const float s = st[kt][nr][r];
                        float x = s * p.mul;
                        if (p.cap2 != 0.f) x = near ? pa_cap_near(s, p.a) : pa_cap_each(s, pa_cap(x, p.cap2), p.near, p.a);
                        if (p.slopes) x = fmaf(-slope[nr], fabsf((float)(pos[nr] - key)), x);
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
            auto vread = [&](int dt) __attribute__((always_inline)) -> v8 {
                const pg_s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)v_rd[dt]);
                const pg_s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(v_rd[dt] + (uint32_t)(16 * RB)));
                return __builtin_bit_cast(v8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            if (__builtin_expect(part_seen, 0) && __builtin_expect(pg_not_finite<T, TILE>(lds_v, lane), 0)) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    v8 up, down;
                    pg_split<T>(vread(dt), up, down);
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        // 1 for the keys that the row sees, made anew for every dt: kept, they make others spill (D = 256: a quarter of the time)
                        int from = lo[nr], to = min(hi[nr], end_pos), at = first;
                        asm volatile("" : "+v"(from), "+v"(to), "+s"(at));
                        from -= at + 4 * g;
                        to -= at + 4 * g;
                        v8 seen;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int key = 16 * (e >> 2) + (e & 3);
                            seen[e] = key >= from && key <= to ? (T)1.f : (T)0.f;
                        }
                        pg_add_not_finite(o[dt][nr], TT::mma16(up, seen, f32x4{0.f, 0.f, 0.f, 0.f}), 1.f);
                        pg_add_not_finite(o[dt][nr], TT::mma16(down, seen, f32x4{0.f, 0.f, 0.f, 0.f}), -1.f);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                pg_drop_not_finite<T, TILE>(lds_v, lane);
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const v8 a = vread(dt);
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) o[dt][nr] = TT::mma16(a, pf[nr], o[dt][nr]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V's place is read
            request(next, false);
            now = next;
            if ((j + 2) % decltype(pages)::TPC == 0 && j + 2 >= decltype(pages)::TPC)
                pages.load(p, b, (j + 2) / decltype(pages)::TPC + 1, lane, where);   // into the place of the chunk just left
            next = lookup(j + 2);
        }

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
        const PaParams e = args.get();
        const bool whole = nblk == nb, direct = whole && !PRE;
        const PaParts parts = pa_parts(at - (uint32_t)blk0, nb, per);
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
                const int64_t out_row = (int64_t)row_t[nr] * e.Hq + row_h[nr];
                const float inv = ll[nr] == 0.f ? 0.f : 1.f / ll[nr];
                T* orow = (T*)e.O + (int64_t)row_t[nr] * e.ost + (int64_t)row_h[nr] * e.osh + 4 * g;
                const int64_t part = whole ? (b < 0 ? 0 : (int64_t)e.b.T * e.Hq) + out_row
                                           : pa_part(parts, (int)(wg - parts.i0), 16 * nr + r16, R);
                float* prow = (whole ? e.row_o : e.ws_o) + part * DP + 4 * g;
                float2* pml = (whole ? e.row_ml : e.ws_ml) + part;
#pragma unroll
                for (int d4 = 0; d4 < NDT / 4; ++d4) {
                    const int dt = 4 * d4 + w;
                    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 4; ++i) x += *(const lds_f32x4*)(uintptr_t)(box + 1024u * (uint32_t)((i * NH + u) * NDT + dt));
                    if (!live[nr]) continue;
                    if (direct) {
                        const v4 y = {(T)(x[0] * inv), (T)(x[1] * inv), (T)(x[2] * inv), (T)(x[3] * inv)};
                        if (16 * dt + 4 * g < e.c.D) *reinterpret_cast<v4*>(orow + 16 * dt) = y;
                    } else {
                        if constexpr (LIVE) {
                            pa_put(prow + 16 * dt, x[0], x[1]);
                            pa_put(prow + 16 * dt + 2, x[2], x[3]);
                        } else {
                            *reinterpret_cast<f32x4*>(prow + 16 * dt) = x;
                        }
                    }
                }
                if (live[nr] && w == 0 && g == 0) {
                    if (direct) {
                        if (e.lse) e.lse[out_row] = ll[nr] == 0.f ? -INFINITY : (ml[nr] + log2f(ll[nr])) * PA_LN2;
                    } else {
                        if constexpr (LIVE) pa_put((float*)pml, ml[nr], ll[nr]);
                        else *pml = make_float2(ml[nr], ll[nr]);
                    }
                }
            }
        }
        if (!whole) {
            if constexpr (LIVE)
                pa_arrive<T, DP, 4>(e, parts, R, min(R, rows - tile * R), tile * R, sg.seq.first, head, w, lane, &arrived);
            else if (LATER && blk0 == 0)
                open = {parts.n, min(R, rows - tile * R), tile * R, sg.seq.first, head};
        }
        at += (uint32_t)nblk;
    }
    if (LATER) pa_leave_open(args.get().ws_open + wg, open);
}

// Behind a stacked prefix: a row's parts, the prefix's and its sequence's, each in the order of its keys.  256 / DP rows a
// wavefront, heads of one token.
template <typename T, int DP>
__global__ void __launch_bounds__(256) paged_join_kernel(PaParams, int R, int pre_R) {
    const int lane = threadIdx.x & 63;
    PaArgs args;
    args.load(lane);
    const PaParams p = args.get();
    constexpr int RPW = 256 / DP;
    const int heads = p.c.heads * p.G;   // of the pass
    const uint32_t per_token = (uint32_t)(heads + RPW - 1) / RPW;   // wavefronts a token
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(pg_block() * 4 + (threadIdx.x >> 6)));
    const int t = (int)(wave / per_token), h0 = (int)(wave - (uint32_t)t * per_token) * RPW;
    if (t >= p.b.T) return;
    const int h = min(h0 + lane / (DP / 4), heads - 1);
    const int b = paged_find(p.b, t, lane);
    if (b >= p.b.B) return;
    const PagedSeq s = paged_seq(p.b, b);
    if (t < s.first || t >= s.first + s.n || s.n * p.G > p.row_limit) return;
    // a tile's parts: whole (one, by row), or in the workspace
    struct Source {
        const float* o;
        const float2* ml;
        PaParts parts;
        int R, in;
        __device__ int64_t at(int j) const { return parts.n == 1 ? 0 : pa_part(parts, j, in, R); }
    };
    const int head = h / p.G, g = h - head * p.G;
    const int64_t row = (int64_t)t * p.Hq + h;
    auto source = [&](const PaSeq& sw, uint32_t before, uint32_t per, int tile_rows, uint32_t r, const float* o, const float2* ml,
                      int which) {
        const uint32_t tile = r / (uint32_t)tile_rows;
        Source x;
        x.parts = pa_parts(before + ((uint32_t)head * (uint32_t)sw.tiles + tile) * (uint32_t)sw.nb, sw.nb, per);
        x.R = tile_rows;
        x.in = (int)(r - tile * (uint32_t)tile_rows);
        const bool whole = x.parts.n == 1;
        const int64_t i = (int64_t)which * p.b.T * p.Hq + row;
        x.o = whole ? p.row_o + i * DP : o;
        x.ml = whole ? p.row_ml + i : ml;
        return x;
    };
    const PaPlan plan = pa_plan<PR_BK, false, true>(p, R, true, p.stack == 1, lane);
    if (plan.falls) return;
    uint32_t before = plan.pre_work;
    for (int b0 = 0; b0 < b; b0 += 64) {
        const uint32_t upto =
            b0 == 0 ? plan.upto : pa_scan(pa_work(p, pa_seq<PR_BK, false, true>(p, pa_lane_seq(p, b0 + lane), R)));
        before += __builtin_amdgcn_readlane(upto, min(b - b0, 64) - 1);
    }
    const uint32_t per = pa_per(plan.total, p.by_rows, 1);
    const Source own = source(pa_seq<PR_BK, false, true>(p, s, R), before, per, R, (uint32_t)((t - s.first) * p.G + g), p.ws_o, p.ws_ml, 1);
    Source pre = own;
    pre.parts.n = 0;
    if (p.stack == 1) {
        if (plan.pre_work > 0) pre = source(plan.prefix, 0, per, R, (uint32_t)((t - plan.t0) * p.G + g), p.ws_o, p.ws_ml, 0);
    } else {
        const PaPlan pp = pa_plan<PT_BK, true, true>(p, pre_R, false, true, lane);
        if (pp.pre_work > 0)
            pre = source(pp.prefix, 0, pa_per(pp.total, p.by_tiles, PT_LEAST), pre_R, (uint32_t)((t - pp.t0) * p.G + g), p.pre_o, p.pre_ml, 0);
    }
    // a row's parts lie one behind the other.  (Values, not the two structures: chosen between by j those went to scratch memory.)
    const int pre_n = pre.parts.n, own_n = own.parts.n;
    const int64_t pre_at = pre.at(0), own_at = own.at(0);
    const float *const pre_o = pre.o, *const own_o = own.o;
    const float2 *const pre_ml = pre.ml, *const own_ml = own.ml;
    f32x4 o;
    float m, l;
    pa_join_rows<DP, false>(pre_n + own_n, [&](int j, const float2*& ml, const float*& q) {
        const bool first = j < pre_n;
        const int64_t at = (first ? pre_at : own_at) + (first ? j : j - pre_n);
        ml = (first ? pre_ml : own_ml) + at;
        q = (first ? pre_o : own_o) + at * DP;
    }, lane, o, m, l);
    if (h0 + lane / (DP / 4) < heads) pa_store_row<T, DP>(p, t, h, o, m, l, lane);
}

int paged_rows_launch(const PaParams& p, const PaShape& sh, int dtype, hipStream_t s) {
    auto by_type = [&](auto tag) {
        typedef decltype(tag) T;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(sh.row_grid), dim3(256), 0, s, p); };
        auto by_shape = [&](auto pre) {
            constexpr bool PRE = decltype(pre)::value;
            if (sh.dp == 64)
                sh.nr == 1 ? go(paged_rows_kernel<T, 64, 1, PRE>) : go(paged_rows_kernel<T, 64, 2, PRE>);
            else if (sh.dp == 128)
                sh.nr == 1 ? go(paged_rows_kernel<T, 128, 1, PRE>) : go(paged_rows_kernel<T, 128, 2, PRE>);
            else
                sh.nr == 1 ? go(paged_rows_kernel<T, 256, 1, PRE>) : go(paged_rows_kernel<T, 256, 2, PRE>);
        };
        p.P > 0 ? by_shape(pg_tag<true>{}) : by_shape(pg_tag<false>{});
        int rc = check_launch("paged_rows_kernel");
        if (rc != LAVA_HIP_OK) return rc;
        if (p.P == 0) {   // (behind a prefix it is always stacked)
            if (sh.nr == 1) return rc;   // joined by the last workgroup of a tile to arrive
            auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(sh.row_grid * 4), dim3(256), 0, s, p, 16 * sh.nr, 4); };
            sh.dp == 64    ? join(paged_join_tiles_kernel<T, 64>)
            : sh.dp == 128 ? join(paged_join_tiles_kernel<T, 128>)
                           : join(paged_join_tiles_kernel<T, 256>);
            return check_launch("paged_join_tiles_kernel");
        }
        const int per_wave = 256 / sh.dp;
        const dim3 rows = pg_grid(((int64_t)p.b.T * ((p.c.heads * p.G + per_wave - 1) / per_wave) + 3) / 4);
        auto join = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, rows, dim3(256), 0, s, p, 16 * sh.nr, 128 * sh.pre_qh);
        };
        sh.dp == 64 ? join(paged_join_kernel<T, 64>) : sh.dp == 128 ? join(paged_join_kernel<T, 128>) : join(paged_join_kernel<T, 256>);
        return check_launch("paged_join_kernel");
    };
    return dtype == LAVA_HIP_F16 ? by_type(f16{}) : by_type(bf16{});
}

}  // namespace lava
