// paged_attn_tile.hip -- attention over the paged cache for prompts: tiles of many rows.
//
// With hundreds of rows that read the same keys the matrix cores bound the call, 4 D flops a row and key.  The form is
// flash_fwd5_kernel's: a workgroup takes 256 rows (QH = 2) or 128, row r being query r / G and head r % G of a key head,
// so that grouped heads fill tiles together; of each SIMD's two wavefronts one computes the scores and the softmax
// of 64 (32) rows, the other their sums, P passing through LDS; K in three and V in two LDS stages of 64 keys by
// LDS-DMA.  What the paged cache and its masks change:
//  * 8 keys at a time are found through the page table, a block ahead of their request;
//  * every row has its own interval of visible positions: only blocks that some row of a pair does not see whole
//    compare, blocks that none sees are skipped, and a pair whose rows see nothing yet has no maximum (unset, -inf);
//  * the scale and the maximum are one fma a score, P = exp2(fma(S, c, -m)); ANY: caps (a polynomial where a block's scores
//    are small, pa_cap_near), slopes, a scale that is not positive.  Folding the scale into Q and the maximum into the
//    product, as flash_fwd5_kernel does for f16, is 3.5 % faster on f16 prompts (4 of 4096 tokens, early calls: 655 against 679 us)
//    and rounds each q once more: 3.8e-4 off against 2.9e-4, of which the results' own rounding is 2.1e-4.

// Measured (calls in a row; the first 40 after a pause, until the clock has settled, in brackets): 4 prompts of 4096 tokens, 32 heads on
// 8, D = 128, 565 us (720), 970 TFLOP/s; 12 sequences' chunks and decode steps behind 777 to 6000 keys, capped, 300 (366); 8 prompts of
// 301 to 1537 tokens, 12 heads of D = 64, 49; a prompt of 64 tokens 9.

#include <algorithm>

#include "lds_dma.hpp"
#include "paged_plan.hpp"

namespace lava {

constexpr int PT_PAIRS = 4;
constexpr int PT_KST = 3, PT_VST = 2;   // LDS stages
constexpr int PT_PF = 4;                // fragments read ahead of their MFMA
constexpr float PT_RESCALE = 8.f;

template <typename T, int DE, int QH, bool ANY, bool PRE>
__global__ void __launch_bounds__(128 * PT_PAIRS, 1) paged_tile_kernel(PaParams, int stacked) {
    typedef PgType<T> TT;
    typedef typename TT::v8 v8;
    typedef typename TT::v4 v4;
    typedef typename TT::v2 v2;
    typedef __attribute__((address_space(3))) v8 lds_v8;
    typedef __attribute__((address_space(3))) pg_s16x4 lds_s16x4;
    typedef int i4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i4 lds_i4;
    constexpr int PQ = 32 * QH, BQ = PQ * PT_PAIRS;
    constexpr int RB = 256, CH = 16, TILE = PT_BK * RB;
    constexpr int NKS = DE / 16, NDT = DE / 32, NSF = 2 * NKS, NVF = 4 * NDT;
    constexpr int PBUF = QH * 4 * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t kbuf[PT_KST][TILE];   // chunk ^ key % 16
    __shared__ __attribute__((aligned(1024))) uint8_t vbuf[PT_VST][TILE];   // chunk ^ 4 (key % 4)
    __shared__ __attribute__((aligned(1024))) uint8_t pbuf[2][PT_PAIRS][PBUF];
    __shared__ float abuf[2][PT_PAIRS][PQ];
    __shared__ int fbuf[2][PT_PAIRS];
    __shared__ int nan_sums[PT_PAIRS];
    __shared__ __attribute__((aligned(16))) int nbuf[PT_KST][4];   // keys without a page, 2 bits of 8 keys each
    __shared__ float mbuf[PT_PAIRS][PQ];

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_s = w < PT_PAIRS;
    const int pr = w & (PT_PAIRS - 1);
    const int r32 = lane & 31, h = lane >> 5;

    const bool prefix = PRE && stacked != 0;   // the launch for the stacked prefix
    // ---- which part of the work
    PaArgs args;
    args.load(lane);
    const PaParams p = args.get();
    const PaPlan plan = pa_plan<PT_BK, true, PRE>(p, BQ, !prefix, prefix, lane);
    int tiles_upto = 0;
    const bool by_tile = !prefix && !plan.falls && pa_by_tile<PRE>(p, plan, BQ, lane, tiles_upto);
    PaOpen open = {};
    const uint32_t block = pg_block();
    if (by_tile && block < PT_GRID) pa_leave_open(p.ws_open + block, open);
    uint32_t at = 0, stop = 1, per = 1, wg = 0;
    PaSegment sg = {};
    if (by_tile) {
        // key heads innermost, so that an XCD's workgroups share few heads' keys; a sequence's last tiles, which
        // see the most keys, first
        int idx = (int)(block / (unsigned)p.c.heads);
        sg.head = (int)block - idx * p.c.heads;
        sg.b = -1;
        int upto = tiles_upto;
        PagedSeq s = plan.mine;
        for (int b0 = 0;;) {
            const uint64_t past = __builtin_amdgcn_ballot_w64(upto > idx);
            if (past != 0) {
                const int i = __builtin_ctzll(past);
                sg.b = b0 + i;
                sg.tile = __builtin_amdgcn_readlane(upto, i) - 1 - idx;   // from the last one down
                sg.seq.first = __builtin_amdgcn_readlane(s.first, i);
                sg.seq.n = __builtin_amdgcn_readlane(s.n, i);
                sg.seq.kv = __builtin_amdgcn_readlane(s.kv, i);
                break;
            }
            idx -= __builtin_amdgcn_readlane(upto, 63);
            b0 += 64;
            if (b0 >= p.b.B) break;
            s = pa_lane_seq(p, b0 + lane);
            upto = (int)pa_scan((uint32_t)pa_seq<PT_BK, true, PRE>(p, s, BQ).tiles);
        }
        if (sg.b < 0) return;
        sg.sw = pa_seq<PT_BK, true, PRE>(p, sg.seq, BQ);
    } else {
        if (block >= PT_GRID) return;
        per = pa_per(plan.total, p.by_tiles, PT_LEAST);
        wg = pa_place(PT_GRID);
        at = min(plan.total, wg * per);
        stop = min(plan.total, at + per);
    }

    // 0 times a value that is not finite is NaN, also in rows that do not see its key: a segment with sums that are NaN is done
    // once more with the values' finite parts apart (pg_split).  That costs inputs without such values 1 %; a look at the
    // values of blocks that not all rows see whole, in the loop, cost 5 to 10.
    bool careful = false;
    for (; at < stop;) {
    // ---- the segment: some key blocks of a row tile
    const PaParams p = args.get();
    if (!by_tile) sg = pa_segment<PT_BK, true, PRE>(p, plan, BQ, at, lane);
    const PagedSeq seq = sg.seq;
    const int b = sg.b, nb = sg.sw.nb, np = PRE ? sg.sw.np : 0, p0 = sg.sw.p0, o0 = sg.sw.o0;
    const int head = __builtin_amdgcn_readfirstlane(sg.head), tile = __builtin_amdgcn_readfirstlane(sg.tile), blk0 = sg.blk0;
    const int nseg = by_tile ? nb : min(nb - blk0, (int)(stop - at));
    const bool whole = nseg == nb;
    const int rows = seq.n * p.G;
    // rows of a sequence that another launch takes, prefix and all
    if (PRE && b < 0 && pa_other(p, seq.first + tile * BQ / p.G, seq.first + min(seq.n - 1, (tile * BQ + BQ - 1) / p.G), lane)) {
        at += (uint32_t)nseg;
        continue;
    }
    const int P = PRE ? p.P : 0;
    const int end = P + (b < 0 ? 0 : seq.kv);
    const int bid = pa_leading(p, b);
    auto block_of = [&](int pos) { return PRE && pos < P ? pos / PT_BK - p0 : np + (pos - P) / PT_BK - o0; };
    auto first_pos = [&](int blk) { return PRE && blk < np ? (p0 + blk) * PT_BK : P + (o0 + blk - np) * PT_BK; };
    // of rows [r0, r1], in order of their positions, the blocks that some row sees
    auto sees = [&](int r0, int r1, int& f, int& l) {
        const int a = (int)div_of((uint32_t)r0, p.by_g), z = (int)div_of((uint32_t)min(r1, rows - 1), p.by_g);
        const int lo = pa_range(p, end - seq.n + a, end, bid).lo, hi = pa_range(p, end - seq.n + z, end, bid).hi;
        f = 0;
        l = -1;
        if (r0 < rows && hi >= lo) {
            f = max(0, block_of(lo));
            l = min(nb - 1, block_of(hi));
        }
    };
    int e0 = blk0, e1 = blk0 + nseg - 1;
    if (b >= 0) {
        int f, l;
        sees(tile * BQ, tile * BQ + BQ - 1, f, l);
        e0 = max(e0, f);
        e1 = min(e1, l);
    }
    e0 = __builtin_amdgcn_readfirstlane(e0);
    const int nblk = __builtin_amdgcn_readfirstlane(max(0, e1 - e0 + 1));
    // this pair's rows and blocks, from e0 on
    const int row0 = tile * BQ + pr * PQ;
    int jf = 0, jl = row0 < rows ? nblk - 1 : -1;
    if (b >= 0) {
        sees(row0, row0 + PQ - 1, jf, jl);
        jf = max(0, jf - e0);
        jl = min(nblk - 1, jl - e0);
    }
    jf = __builtin_amdgcn_readfirstlane(jf);
    jl = __builtin_amdgcn_readfirstlane(jl);
    const uint32_t p_lane = lds_addr(&pbuf[0][0][0]) + (uint32_t)pr * PBUF + 16u * lane;
    auto paddr = [&](int buf, int kt, int ks, int qh) __attribute__((always_inline)) -> uint32_t {
        return p_lane + (uint32_t)(buf * PT_PAIRS * PBUF + ((kt * 2 + ks) * QH + qh) * 1024);
    };

    auto again = [&]() {
        careful = !careful && __builtin_amdgcn_readfirstlane(nan_sums[0] | nan_sums[1] | nan_sums[2] | nan_sums[3]) != 0;
        return careful;
    };

    if (is_s) {
        // ================= score wavefront =================
        // The pair's rows of Q by LDS-DMA, 4 whole rows an instruction, into its P buffers (free until the first block's P), in
        // the K tile's layout; 32 rows x 32 bytes a load straight into the fragments took 8 us a tile.  Row offsets from
        // the tile's first token and head fit 31 bits (paged_tile_takes).
        const uint32_t qbuf = lds_addr(&pbuf[0][pr][0]);
        auto q_row = [&](int r) { return qbuf + (uint32_t)(r / (16 * QH) * PT_PAIRS * PBUF + r % (16 * QH) * RB); };
        {
            const PaParams p = args.get();
            const int lane = pa_again(threadIdx.x & 63);
            const int i0 = (int)div_of((uint32_t)row0, p.by_g);
            const T* base = (const T*)p.Q + (int64_t)(seq.first + i0) * p.qst + (int64_t)(head * p.G) * p.qsh;
            const v4i rs = make_rsrc(base, 0x7fffffffu);
            const uint32_t st = (uint32_t)p.qst * 2u, sh = (uint32_t)p.qsh * 2u;
#pragma unroll
            for (int i = 0; i < 8 * QH; ++i) {
                const int r = 4 * i + lane / CH, row = row0 + r, c = (lane % CH) ^ (r & 15);
                const int t = (int)div_of((uint32_t)row, p.by_g);
                const uint32_t o = (uint32_t)(t - i0) * st + (uint32_t)(row - t * p.G) * sh + 16u * (uint32_t)c;
                dma16(rs, row < rows && 8 * c < p.c.D ? o : OOB_OFS, 0u, __builtin_amdgcn_readfirstlane(q_row(4 * i)));
            }
        }
        // this lane's rows: the positions that they see
        int r_lo[QH], r_hi[QH];
        int r_pos[QH];
        float slope[QH];
        {
            const PaParams p = args.get();
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) {
                const int row = row0 + 32 * qh + r32, i = (int)div_of((uint32_t)row, p.by_g);
                int pos = end - seq.n + i;
                if (PRE && b < 0) {
                    pos = P;
                    if ((!plan.plain || p.slopes) && row < rows) pos = pa_row_pos(p, seq.first + i);
                }
                const PaRange rg = pa_range(p, pos, end, bid);
                r_lo[qh] = rg.lo;
                r_hi[qh] = rg.hi;
                r_pos[qh] = pos;
                slope[qh] = 0.f;
                if (ANY && p.slopes && row < rows) slope[qh] = p.slopes[head * p.G + row - i * p.G] * PA_LOG2E;
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        v8 qf[QH][NKS];   // Q^T: row row0 + 32 qh + r32, d = 16 ks + 8 h + [0, 8)
#pragma unroll
        for (int qh = 0; qh < QH; ++qh)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
                qf[qh][ks] = *(const lds_v8*)(uintptr_t)(q_row(32 * qh + (r32 & 16)) + (uint32_t)((r32 & 15) * RB + (((2 * ks + h) ^ (r32 & 15)) << 4)));
#pragma unroll
        for (int qh = 0; qh < QH; ++qh)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const uint4 u = __builtin_bit_cast(uint4, qf[qh][ks]);
                asm volatile("" ::"v"(u.x), "v"(u.y), "v"(u.z), "v"(u.w) : "memory");
            }
        // between the first position that the pair's last row sees and the last that its first one does, no comparison
        int in_lo = pa_range(p, end - seq.n + (int)div_of((uint32_t)min(row0 + PQ - 1, rows - 1), p.by_g), end, bid).lo;
        int in_hi = pa_range(p, end - seq.n + (int)div_of((uint32_t)row0, p.by_g), end, bid).hi;
        if (PRE && b < 0) {
            in_lo = plan.plain ? 0 : 0x7fffffff;
            in_hi = P - 1;
        }
        in_lo = __builtin_amdgcn_readfirstlane(in_lo);
        in_hi = __builtin_amdgcn_readfirstlane(in_hi);

        const PaParams p = args.get();
        // K fragment (kt, ks): row 32 kt + r32, chunk (2 ks + h) ^ (r32 % 16), which is ks in bits 1 and up of the rest
        const uint32_t kb0 = lds_addr(&kbuf[0][0]) + (uint32_t)(r32 * RB + ((h ^ (r32 & 15)) << 4));
        f32x16 st[2][QH];   // register r: key 32 kt + 8 (r / 4) + 4 h + r % 4
        float m[QH];        // the running maximum, -inf: unset
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) m[qh] = -INFINITY;

        auto block = [&](int j, int buf) __attribute__((always_inline)) {
            uint32_t ka = kb0 + (uint32_t)((j % PT_KST) * TILE);
            asm("; lds address" : "+v"(ka));
            auto kread = [&](int f) __attribute__((always_inline)) -> v8 {   // f = 2 ks + kt
                return *(const lds_v8*)(uintptr_t)((ka ^ (uint32_t)(32 * (f >> 1))) + (uint32_t)((f & 1) * 32 * RB));
            };
            v8 fr[PT_PF];
#pragma unroll
            for (int f = 0; f < PT_PF; ++f) fr[f] = kread(f);
            const i4 nn = *(const lds_i4*)(uintptr_t)lds_addr(&nbuf[j % PT_KST][0]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < QH * NSF; ++i) {
                const int f = i / QH, qh = i % QH, ks = f >> 1, kt = f & 1;
                st[kt][qh] = TT::mma32(fr[f % PT_PF], qf[qh][ks], ks == 0 ? f32x16{} : st[kt][qh]);
                if (qh == QH - 1 && f + PT_PF < NSF) fr[f % PT_PF] = kread(f + PT_PF);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int none = __builtin_amdgcn_readfirstlane(nn.x | nn.y << 2 | nn.z << 4 | nn.w << 6);
            const int pos0 = __builtin_amdgcn_readfirstlane(first_pos(e0 + j));
            const int src_hi = PRE && e0 + j < np ? P - 1 : end - 1;
            // scores relative to the maximum, to 0 while it is unset
            float ref[QH];
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) ref[qh] = m[qh] == -INFINITY ? 0.f : m[qh];
            auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                        for (int r = 0; r < 16; ++r) st[kt][qh][r] = f(st[kt][qh][r], qh, 32 * kt + 8 * (r >> 2) + (r & 3));
            };
            if constexpr (!ANY) each([&](float x, int qh, int) { return fmaf(x, p.mul, -ref[qh]); });
            if constexpr (ANY) {
                if (p.cap2 == 0.f) {
                    each([&](float x, int qh, int) { return fmaf(x, p.mul, -ref[qh]); });
                } else {
                    float far = 0.f;   // NaN: the exact form carries it as well as the other
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                            for (int r = 0; r < 16; ++r) far = fmaxf(far, fabsf(st[kt][qh][r]));
                    if (__builtin_amdgcn_ballot_w64(far > p.near) != 0 && p.cap2 > PA_CAP_SMALL)
                        each([&](float x, int qh, int) { return pa_cap_each(x, pa_cap(x * p.mul, p.cap2), p.near, p.a) - ref[qh]; });
                    else if (__builtin_amdgcn_ballot_w64(far > p.near) != 0)
                        each([&](float x, int qh, int) { return pa_cap(x * p.mul, p.cap2) - ref[qh]; });
                    else
                        each([&](float x, int qh, int) {
                            const float u = x * x;
                            return fmaf(x, fmaf(fmaf(fmaf(fmaf(p.a[4], u, p.a[3]), u, p.a[2]), u, p.a[1]), u, p.a[0]), -ref[qh]);
                        });
                }
                if (p.slopes) {
                    float d0[QH];
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh) d0[qh] = (float)(pos0 + 4 * h - r_pos[qh]);
                    each([&](float x, int qh, int k) { return fmaf(-slope[qh], fabsf(d0[qh] + (float)k), x); });
                }
            }
            if (none != 0 || pos0 < in_lo || pos0 + PT_BK - 1 > min(in_hi, src_hi)) {
#pragma unroll
                for (int qh = 0; qh < QH; ++qh) {
                    int lo = r_lo[qh] - pos0 - 4 * h, hi = min(r_hi[qh], src_hi) - pos0 - 4 * h;
                    asm volatile("; mask" : "+v"(lo), "+v"(hi));
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int kr = 32 * kt + 8 * (r >> 2) + (r & 3);
                            const bool off = kr < lo || kr > hi || ((none >> (4 * kt + (r >> 2))) & 1);
                            st[kt][qh][r] = off ? -INFINITY : st[kt][qh][r];
                        }
                }
            }
            float vl[QH];   // how far the largest score lies above the maximum
            bool up = false;
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) {
                float v = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) v = fmaxf(v, st[kt][qh][r]);
                vl[qh] = v;
                up = up || v > (m[qh] == -INFINITY ? -INFINITY : PT_RESCALE);
            }
            const bool rescale = __builtin_amdgcn_ballot_w64(up) != 0;
            float sub[QH] = {};   // what P = exp2(score - sub) takes off
            if (rescale) {
                float mn[QH];
#pragma unroll
                for (int qh = 0; qh < QH; ++qh) {
                    float a, c;
                    pg_xor32_pair(vl[qh], a, c);
                    const float t = fmaxf(a, c);
                    const bool unset = m[qh] == -INFINITY;
                    mn[qh] = unset ? t : m[qh] + fmaxf(t, 0.f);
                }
#pragma unroll
                for (int qh = 0; qh < QH; ++qh) {
                    const bool unset = m[qh] == -INFINITY, still = mn[qh] == -INFINITY;
                    const float alpha = unset ? 1.f : __builtin_amdgcn_exp2f(m[qh] - mn[qh]);
                    const float to = still ? 0.f : mn[qh];
                    sub[qh] = to - ref[qh];
                    m[qh] = mn[qh];
                    if (h == 0) abuf[buf][pr][32 * qh + r32] = alpha;
                }
            }
            if (lane == 0) fbuf[buf][pr] = rescale ? 1 : 0;
            // kind 0: scores against an unmoved maximum; 1: a moved one; 2: either, masked keys as -0
            auto pstore = [&](auto kind) __attribute__((always_inline)) {
                constexpr int KIND = decltype(kind)::value;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                        for (int qh = 0; qh < QH; ++qh) {
                            v8 u;
                            const float msub = -sub[qh];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                float x = st[kt][qh][8 * ks + k];
                                if constexpr (KIND > 0) x += msub;
                                const T q = (T)__builtin_amdgcn_exp2f(x);
                                u[k] = KIND == 2 && x == -INFINITY ? __builtin_bit_cast(T, (uint16_t)0x8000) : q;
                            }
                            *(lds_v8*)(uintptr_t)paddr(buf, kt, ks, qh) = u;
                        }
            };
            if (__builtin_expect(careful, 0))
                pstore(pg_int<2>{});
            else if (!rescale)
                pstore(pg_int<0>{});
            else
                pstore(pg_int<1>{});
        };

        __syncthreads();   // K_0 .. K_2, V_0 in LDS
        if (jf == 0 && jl >= 0) block(0, 0);
        __syncthreads();   // P_0 published
        for (int j = 0; j < nblk; ++j) {
            if (j + 1 >= jf && j + 1 <= jl) block(j + 1, (j + 1) & 1);
            __syncthreads();
        }
        if (h == 0) {
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) mbuf[pr][32 * qh + r32] = m[qh];
        }
        __syncthreads();
        if (again()) continue;
    } else {
        // ================= output wavefront =================
        const PaParams p = args.get();
        const uint32_t row_bytes = (uint32_t)(p.c.sl * 2);
        uint32_t ofs_k[4], ofs_v[2];   // rows 4 i + lane / 16 of this wavefront's 16
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * i + lane / CH, in8 = row & 7;
            const int ck = (lane % CH) ^ row, cv = (lane % CH) ^ (4 * (row & 3));
            ofs_k[i] = 8 * ck < p.c.D ? (uint32_t)in8 * row_bytes + 16u * (uint32_t)ck : OOB_OFS;
            if (i < 2) ofs_v[i] = 8 * cv < p.c.D ? (uint32_t)in8 * row_bytes + 16u * (uint32_t)cv : OOB_OFS;
        }
        // blocks of 16 keys of this wavefront's
        PaPages<2, PRE> pages = {-1, -1};
        auto where = [&](int j, int i, int& k, bool& pre) {
            const int blk = e0 + j;
            pre = PRE && blk < np;
            k = (pre ? p0 + blk : o0 + blk - np) * PT_BK + 16 * pr + 8 * i;
            return j < nblk && k < (pre ? P : seq.kv);
        };
        pages.load(p, b, 0, lane, where);
        if (nblk + 3 > decltype(pages)::TPC) pages.load(p, b, 1, lane, where);   // requests run three blocks ahead
        auto request = [&](bool is_k, int j) __attribute__((always_inline)) {
            const T* base = (const T*)(is_k ? p.c.k : p.c.v) + (int64_t)head * p.c.sh;
            const int blk = e0 + j;
            const bool pre = PRE && blk < np;
            const int left = (pre ? P : seq.kv) - (pre ? p0 + blk : o0 + blk - np) * PT_BK - 16 * pr;   // keys to the end
            const uint32_t dst = lds_addr(is_k ? &kbuf[0][0] : &vbuf[0][0]) + (uint32_t)pr * 16 * RB +
                                 (uint32_t)(j % (is_k ? PT_KST : PT_VST)) * TILE;
            int none = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t o = pages.get(j, i);
                const uint32_t bytes = o < 0 ? 0u : (uint32_t)(min(left - 8 * i, 8) - 1) * row_bytes + 2u * (uint32_t)p.c.D;
                const v4i rs = make_rsrc(base + o, bytes);   // none: nothing in range
                none |= o < 0 ? 1 << i : 0;
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    dma16(rs, is_k ? ofs_k[2 * i + u] : ofs_v[u], 0u,
                          __builtin_amdgcn_readfirstlane(dst + 1024u * (uint32_t)(2 * i + u)));
            }
            if (is_k && lane == 0) nbuf[j % PT_KST][pr] = none;
        };
        request(true, 0);
        request(true, 1);
        request(true, 2);
        request(false, 0);

        // V^T fragment (dt, key step kk): two transposing reads at keys kk + 4 h + jj and + 8; the chunk
        // (4 dt + 2 dh + q / 2) ^ 4 jj is dt in bits 2 and up of the rest
        const int jj = (lane & 15) >> 2, vq = lane & 3, dh = (lane >> 4) & 1;
        const uint32_t vb0 = lds_addr(&vbuf[0][0]) + (uint32_t)((4 * h + jj) * RB + (((2 * dh + (vq >> 1)) ^ (4 * jj)) << 4) + ((vq & 1) << 3));
        f32x16 o[NDT][QH];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][qh][r] = 0.f;
        float l[QH] = {};   // this lane's part of the row sums of P

        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // K_0 .. K_2, V_0 in LDS
        __syncthreads();   // P_0 published
        auto step = [&](int j, auto slow) __attribute__((always_inline)) {
            const int buf = j & 1;
            // K_{j+3} into K_j's stage, V_{j+1} into V_{j-1}'s, both read in iteration j - 1
            request(true, j + 3);
            request(false, j + 1);
            // V of chunk c - 1 is past when K is two blocks into chunk c
            if ((j + 3) % decltype(pages)::TPC == 2 && j + 3 > decltype(pages)::TPC) pages.load(p, b, (j + 3) / decltype(pages)::TPC + 1, lane, where);
            if (j >= jf && j <= jl) {
                if (fbuf[buf][pr] != 0) {   // the maximum moved at block j
                    float al[QH];
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh) al[qh] = abuf[buf][pr][32 * qh + r32];
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
#pragma unroll
                            for (int qh = 0; qh < QH; ++qh) o[dt][qh][r] *= al[qh];
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh) l[qh] *= al[qh];
                }
                uint32_t va = vb0 + (uint32_t)((j % PT_VST) * TILE);
                asm("; lds address" : "+v"(va));
                auto vread = [&](int f) __attribute__((always_inline)) -> v8 {   // f = NDT kk + dt
                    const int kk = 16 * (f / NDT), dt = f % NDT;
                    const uint32_t at = (va ^ (uint32_t)(64 * dt)) + (uint32_t)(kk * RB);
                    const pg_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)at);
                    const pg_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + 8 * RB));
                    return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                auto pread = [&](int kk, int qh) __attribute__((always_inline)) -> v8 {
                    return *(const lds_v8*)(uintptr_t)paddr(buf, kk >> 1, kk & 1, qh);
                };
                if constexpr (decltype(slow)::value) {
#pragma unroll 1
                    for (int kk = 0; kk < 4; ++kk) {
                        v8 x[QH], seen[QH];
#pragma unroll
                        for (int qh = 0; qh < QH; ++qh) {
                            x[qh] = pread(kk, qh);
                            seen[qh] = pg_seen<T>(x[qh]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) l[qh] = TT::dot2(v2{x[qh][2 * e], x[qh][2 * e + 1]}, l[qh]);
                        }
#pragma unroll
                        for (int dt = 0; dt < NDT; ++dt) {
                            v8 up, down;
                            const v8 a = pg_split<T>(vread(NDT * kk + dt), up, down);
#pragma unroll
                            for (int qh = 0; qh < QH; ++qh) {
                                o[dt][qh] = TT::mma32(a, x[qh], o[dt][qh]);
                                pg_add_not_finite(o[dt][qh], TT::mma32(up, seen[qh], f32x16{}), 1.f);
                                pg_add_not_finite(o[dt][qh], TT::mma32(down, seen[qh], f32x16{}), -1.f);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                } else {
                    v8 fr[PT_PF + 1], pp[2][QH];
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh) pp[0][qh] = pread(0, qh);
#pragma unroll
                    for (int f = 0; f < PT_PF + 1; ++f) fr[f] = vread(f);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < QH * NVF; ++i) {
                        const int f = i / QH, qh = i % QH, kk = f / NDT, dt = f % NDT;
                        if (i % (QH * NDT) == 0 && kk < 3) {
#pragma unroll
                            for (int qq = 0; qq < QH; ++qq) pp[(kk + 1) & 1][qq] = pread(kk + 1, qq);
                        }
                        if (i % (QH * NDT) == QH * NDT / 2) {   // row sums of what is multiplied
#pragma unroll
                            for (int qq = 0; qq < QH; ++qq)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    l[qq] = TT::dot2(v2{pp[kk & 1][qq][2 * e], pp[kk & 1][qq][2 * e + 1]}, l[qq]);
                        }
                        o[dt][qh] = TT::mma32(fr[f % (PT_PF + 1)], pp[kk & 1][qh], o[dt][qh]);
                        if (qh == QH - 1 && f + PT_PF + 1 < NVF) fr[f % (PT_PF + 1)] = vread(f + PT_PF + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // K_{j+3}, V_{j+1} are here
            __syncthreads();
        };
        if (__builtin_expect(!careful, 1)) {
            for (int j = 0; j < nblk; ++j) step(j, pg_tag<false>{});
            float zero[4] = {};
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                    for (int r = 0; r < 16; ++r) zero[r & 3] = fmaf(o[dt][qh][r], 0.f, zero[r & 3]);
            const bool some = __builtin_amdgcn_ballot_w64(!(zero[0] + zero[1] + zero[2] + zero[3] == 0.f)) != 0;
            if (lane == 0) nan_sums[pr] = some;
        } else {
            for (int j = 0; j < nblk; ++j) step(j, pg_tag<true>{});
        }
        __syncthreads();   // the maxima and whether sums are NaN are published
        if (again()) continue;
        const PaParams e = args.get();
        const int lane = pa_again(threadIdx.x & 63), r32 = lane & 31, h = lane >> 5;
        // Rows leave through LDS, so that stores are of whole rows: 16 rows of 256 bytes at a time in each of this wavefront's
        // parts of the K stages and the first V stage, which only it requests into again
        auto o_row = [&](int r) {   // of 64 (32) rows in 16 bits; r / 16: the part
            return (r < 48 ? lds_addr(&kbuf[0][0]) + (uint32_t)(r / 16 * TILE) : lds_addr(&vbuf[0][0])) + (uint32_t)((16 * pr + r % 16) * RB);
        };
        auto live = [&](int qh) { return row0 + 32 * qh + r32 < rows; };
        auto out_row = [&](int row) {   // token * Hq + head
            const int t = (int)div_of((uint32_t)row, e.by_g);
            return (int64_t)(seq.first + t) * e.Hq + head * e.G + row - t * e.G;
        };
        float sum[QH];
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) {
            float a, c;
            pg_xor32_pair(l[qh], a, c);
            sum[qh] = a + c;
        }
        typedef __attribute__((address_space(3))) v4 lds_v4;
        typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
        if (whole && b >= 0) {
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) {
                const float inv = sum[qh] == 0.f ? 0.f : 1.f / sum[qh];
                const uint32_t to = o_row(32 * qh + (r32 & 16)) + (uint32_t)((r32 & 15) * RB + 8 * h);
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const v4 v = {(T)(o[dt][qh][4 * g4] * inv), (T)(o[dt][qh][4 * g4 + 1] * inv), (T)(o[dt][qh][4 * g4 + 2] * inv),
                                      (T)(o[dt][qh][4 * g4 + 3] * inv)};
                        *(lds_v4*)(uintptr_t)(to + (uint32_t)(((4 * dt + g4) ^ (r32 & 15)) << 4)) = v;
                    }
                if (e.lse && live(qh) && h == 0)
                    e.lse[out_row(row0 + 32 * qh + r32)] =
                        sum[qh] == 0.f ? -INFINITY : (mbuf[pr][32 * qh + r32] + log2f(sum[qh])) * PA_LN2;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int cc = lane % CH;
            const bool o16 = e.o16;   // rows of 16-byte pieces, else of 8
            const int i0 = (int)div_of((uint32_t)row0, e.by_g);
            uint8_t* const obase = (uint8_t*)((T*)e.O + (int64_t)(seq.first + i0) * e.ost + (int64_t)(head * e.G) * e.osh);
            const uint32_t ost = (uint32_t)e.ost * 2u, osh = (uint32_t)e.osh * 2u;   // offsets fit 31 bits, as Q's
#pragma unroll
            for (int i = 0; i < 8 * QH; ++i) {
                const int r = 4 * i + lane / CH, row = row0 + r;
                const v8 v = *(const lds_v8*)(uintptr_t)(o_row(4 * i) + (uint32_t)((lane / CH) * RB + ((cc ^ (r & 15)) << 4)));
                if (row < rows && 8 * cc < e.c.D) {
                    const int t = (int)div_of((uint32_t)row, e.by_g);
                    T* orow = (T*)(obase + ((uint32_t)(t - i0) * ost + (uint32_t)(row - t * e.G) * osh + 16u * (uint32_t)cc));
                    if (o16) {
                        *reinterpret_cast<v8*>(orow) = v;
                    } else {
                        *reinterpret_cast<v4*>(orow) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
                        *reinterpret_cast<v4*>(orow + 4) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
                    }
                }
            }
        } else {
            float* po = whole ? e.row_o : prefix ? e.pre_o : e.ws_o;
            float2* pml = whole ? e.row_ml : prefix ? e.pre_ml : e.ws_ml;
            const PaParts parts = pa_parts(at - (uint32_t)blk0, nb, per);
            const int mine = (int)(wg - parts.i0);
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) {
                // 32 rows of sums, DE x 4 bytes: two rows' worth of LDS a row (8 rows a part at DE = 128)
                constexpr int RF = DE * 4, RPP = 16 * RB / RF;
                auto f_row = [&](int r) { return o_row(r / RPP * 16) + (uint32_t)(r % RPP * RF); };
                constexpr int GO = RPP * 4 < 32 ? RPP * 4 : 32;   // rows the four parts hold
                static_assert(GO == 32, "32 rows of sums fit the four parts");
                const uint32_t to = f_row(r32) + 16u * (uint32_t)h;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4)   // 32-byte pieces, ^ row % 8 against bank conflicts
                        *(lds_f32x4*)(uintptr_t)(to + (uint32_t)(((4 * dt + g4) ^ (r32 & 7)) << 5)) =
                            f32x4{o[dt][qh][4 * g4], o[dt][qh][4 * g4 + 1], o[dt][qh][4 * g4 + 2], o[dt][qh][4 * g4 + 3]};
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                // two rows (DE = 128) or four (64) an instruction; rows of no weight are not read again
                constexpr int LPR = DE / 4, RPS = 64 / LPR;
                const uint64_t some = __builtin_amdgcn_ballot_w64(sum[qh] != 0.f && live(qh));
#pragma unroll 8
                for (int r0 = 0; r0 < 32; r0 += RPS) {
                    const int r = r0 + lane / LPR, x = lane % LPR;
                    const f32x4 v = *(const lds_f32x4*)(uintptr_t)(f_row(r) + (uint32_t)(((x >> 1) ^ (r & 7)) << 5) + 16u * (uint32_t)(x & 1));
                    const int row = row0 + 32 * qh + r;
                    if ((some >> r) & 1) {
                        const int64_t part = whole ? out_row(row) : pa_part(parts, mine, pr * PQ + 32 * qh + r, BQ);
                        *reinterpret_cast<f32x4*>(po + part * DE + 4 * x) = v;
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (live(qh) && h == 0)
                    pml[whole ? out_row(row0 + 32 * qh + r32) : pa_part(parts, mine, pr * PQ + 32 * qh + r32, BQ)] = make_float2(mbuf[pr][32 * qh + r32], sum[qh]);
            }
        }
    }
    if (!whole && blk0 == 0 && !prefix)
        open = {pa_parts(at, nb, per).n, min(BQ, rows - tile * BQ), tile * BQ, seq.first, head};
    at += (uint32_t)nseg;
    }
    if (!by_tile && !prefix) pa_leave_open(args.get().ws_open + wg, open);
}

// ---- host -----------------------------------------------------------------------------

// Whether Q's and O's offsets within a tile fit 31 bits.
bool paged_tile_takes(const PaParams& p) {
    auto fits = [&](int64_t st, int64_t sh) { return (256.0 / p.G + 2) * st * 2.0 + (double)p.G * sh * 2.0 + 512 < 2147483647.0; };
    return p.c.D <= 128 && fits(p.qst, p.qsh) && fits(p.ost, p.osh);
}

int paged_tile_launch(const PaParams& p, int qh, bool prefix, int dtype, hipStream_t s) {
    const bool plain = p.cap2 == 0.f && !p.slopes && p.mul > 0.f;
    const int64_t tiles = ((int64_t)p.b.T * p.G / (128 * qh) + std::min(p.b.B, p.b.T)) * p.c.heads;   // no fewer than there are
    const dim3 grid = pg_grid(prefix ? PT_GRID : std::max<int64_t>(tiles, PT_GRID));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(128 * PT_PAIRS), 0, s, p, prefix ? 1 : 0); };
    auto by_d = [&](auto type, auto q, auto any) {
        typedef decltype(type) T;
        constexpr int QH = decltype(q)::value;
        constexpr bool ANY = decltype(any)::value;
        if (p.P > 0)
            p.c.D <= 64 ? go(paged_tile_kernel<T, 64, QH, ANY, true>) : go(paged_tile_kernel<T, 128, QH, ANY, true>);
        else
            p.c.D <= 64 ? go(paged_tile_kernel<T, 64, QH, ANY, false>) : go(paged_tile_kernel<T, 128, QH, ANY, false>);
    };
    auto by_score = [&](auto type, auto q) { plain ? by_d(type, q, pg_tag<false>{}) : by_d(type, q, pg_tag<true>{}); };
    auto by_rows = [&](auto type) { qh == 1 ? by_score(type, pg_int<1>{}) : by_score(type, pg_int<2>{}); };
    dtype == LAVA_HIP_F16 ? by_rows(f16{}) : by_rows(bf16{});
    const int rc = check_launch(qh == 1 ? "paged_tile_kernel+paged_tile_kernel<32>" : "paged_tile_kernel");
    if (rc != LAVA_HIP_OK || prefix || p.whole) return rc;
    auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(PT_GRID * 8), dim3(256), 0, s, p, 128 * qh, 8); };
    auto join_type = [&](auto type) {
        typedef decltype(type) T;
        p.c.D <= 64 ? join(paged_join_tiles_kernel<T, 64>) : join(paged_join_tiles_kernel<T, 128>);
    };
    dtype == LAVA_HIP_F16 ? join_type(f16{}) : join_type(bf16{});
    return check_launch("paged_join_tiles_kernel");
}

}  // namespace lava
