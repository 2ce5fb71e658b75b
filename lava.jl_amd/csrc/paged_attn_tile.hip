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
//  * MODE 0 (f16, 0 < scale log2 e <= 1, no cap or slopes): the scale is folded into Q (one rounding) and the maximum
//    enters the product as a bias k-step, so that P = exp2 of the accumulator; 1 (bf16, positive scale): P = exp2(fma(S, c,
//    -m)), since bf16 would lose 2^-8 of q c; 2: caps, slopes, any scale.

#include <algorithm>

#include "lds_dma.hpp"
#include "paged_plan.hpp"
#include "paged_types.hpp"

namespace lava {

constexpr int PT_PAIRS = 4;
constexpr int PT_KST = 3, PT_VST = 2;   // LDS stages
constexpr int PT_PF = 4;                // fragments read ahead of their MFMA
constexpr float PT_RESCALE = 8.f;

template <typename T, int DE, int QH, int MODE>
__global__ void __launch_bounds__(128 * PT_PAIRS, 1) paged_tile_kernel(PaParams p, int prefix) {
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
    __shared__ __attribute__((aligned(16))) int nbuf[PT_KST][4];   // keys without a page, 2 bits of 8 keys each
    __shared__ float mbuf[PT_PAIRS][PQ];
    __shared__ int arrived;

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool is_s = w < PT_PAIRS;
    const int pr = w & (PT_PAIRS - 1);
    const int r32 = lane & 31, h = lane >> 5;

    // ---- which part of the work.  Tiles one by one, a workgroup each, where the longest does not outlast the rest by more
    // than splitting costs (parts written and joined, about 12 blocks' time, and blocks that only a sequence's
    // last tiles see counted for all); else the even split over PT_GRID workgroups.
    const PaPlan plan = pa_plan<PT_BK, true>(p, BQ, !prefix, prefix, lane);
    const bool by_tile = !prefix && plan.longest / 2 <= 12 + (int)((plan.total - min(plan.total, plan.seen)) / PA_CUS);
    uint32_t at = 0, stop = 1, per = 1, wg = 0, before = 0;
    int tb = -1, t_head = 0, t_tile = 0;
    if (by_tile) {
        // key heads innermost, so that an XCD's workgroups share few heads' keys; a sequence's last tiles, which
        // see the most keys, first
        t_head = (int)(blockIdx.x % (unsigned)p.c.heads);
        int idx = (int)(blockIdx.x / (unsigned)p.c.heads);
        for (int b0 = 0; b0 < p.b.B; b0 += 64) {
            int tiles = 0;
            if (b0 + lane < p.b.B) tiles = pa_seq<PT_BK, true>(p, paged_seq(p.b, b0 + lane), BQ).tiles;
            const int upto = (int)pa_scan((uint32_t)tiles, lane);
            const uint64_t past = __builtin_amdgcn_ballot_w64(upto > idx);
            if (past != 0) {
                const int i = __builtin_ctzll(past);
                const int lower = i > 0 ? __builtin_amdgcn_readlane(upto, i - 1) : 0;
                tb = b0 + i;
                t_tile = __builtin_amdgcn_readlane(upto, i) - 1 - (idx - lower) - lower;   // from the last one down
                break;
            }
            idx -= __builtin_amdgcn_readlane(upto, 63);
        }
        if (tb < 0) return;
    } else {
        if (blockIdx.x >= PT_GRID) return;
        per = pa_per(plan.total, PT_GRID);
        wg = pa_place(PT_GRID);
        at = min(plan.total, wg * per);
        stop = min(plan.total, at + per);
    }

    for (; at < stop;) {
    // ---- the segment: some key blocks of a row tile
    int b = tb;
    PagedSeq seq = {plan.t0, plan.t1 - plan.t0, 0};
    PaSeq sw = plan.prefix;
    if (!by_tile) b = pa_locate<PT_BK, true>(p, plan, BQ, at, lane, before);
    b = __builtin_amdgcn_readfirstlane(b);
    if (b >= 0) {
        seq = paged_seq(p.b, b);
        sw = pa_seq<PT_BK, true>(p, seq, BQ);
    }
    seq.first = __builtin_amdgcn_readfirstlane(seq.first);
    seq.n = __builtin_amdgcn_readfirstlane(seq.n);
    seq.kv = __builtin_amdgcn_readfirstlane(seq.kv);
    const int nb = __builtin_amdgcn_readfirstlane(sw.nb), np = __builtin_amdgcn_readfirstlane(sw.np);
    const int p0 = __builtin_amdgcn_readfirstlane(sw.p0), o0 = __builtin_amdgcn_readfirstlane(sw.o0);
    int head = t_head, tile = t_tile, blk0 = 0, nseg = nb;
    if (!by_tile) {
        const uint32_t rel = at - before, ht = rel / (uint32_t)nb;
        blk0 = (int)(rel - ht * (uint32_t)nb);
        head = (int)(ht / (uint32_t)sw.tiles);
        tile = (int)(ht - (uint32_t)head * (uint32_t)sw.tiles);
        nseg = min(nb - blk0, (int)(stop - at));
    }
    head = __builtin_amdgcn_readfirstlane(head);
    tile = __builtin_amdgcn_readfirstlane(tile);
    blk0 = __builtin_amdgcn_readfirstlane(blk0);
    nseg = __builtin_amdgcn_readfirstlane(nseg);
    const bool whole = nseg == nb;
    const int rows = seq.n * p.G;
    // rows of a sequence that another launch takes, prefix and all
    if (b < 0 && pa_other(p, seq.first + tile * BQ / p.G, seq.first + min(seq.n - 1, (tile * BQ + BQ - 1) / p.G), lane)) {
        at += (uint32_t)nseg;
        continue;
    }
    const int end = b < 0 ? p.P : p.P + seq.kv;
    const int bid = b >= 0 && p.bidir ? p.bidir[b] : 0;
    auto block_of = [&](int pos) { return pos < p.P ? pos / PT_BK - p0 : np + (pos - p.P) / PT_BK - o0; };
    auto first_pos = [&](int blk) { return blk < np ? (p0 + blk) * PT_BK : p.P + (o0 + blk - np) * PT_BK; };
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
    // this lane's rows
    int row_t[QH], row_h[QH], r_lo[QH], r_hi[QH];
    float r_pos[QH];
    bool live[QH];
#pragma unroll
    for (int qh = 0; qh < QH; ++qh) {
        const int row = row0 + 32 * qh + r32;
        const int i = (int)div_of((uint32_t)row, p.by_g);
        live[qh] = row < rows;
        row_t[qh] = seq.first + i;
        row_h[qh] = head * p.G + row - i * p.G;
        int pos = end - seq.n + i;
        if (b < 0) {
            pos = p.P;
            if ((!plan.plain || p.slopes) && live[qh]) pos = pa_row_pos(p, row_t[qh]);
        }
        const PaRange rg = pa_range(p, pos, end, bid);
        r_lo[qh] = live[qh] ? rg.lo : 0;
        r_hi[qh] = live[qh] ? rg.hi : 0x7fffffff;
        r_pos[qh] = (float)pos;
    }

    const uint32_t p_lane = lds_addr(&pbuf[0][0][0]) + (uint32_t)pr * PBUF + 16u * lane;
    auto paddr = [&](int buf, int kt, int ks, int qh) __attribute__((always_inline)) -> uint32_t {
        return p_lane + (uint32_t)(buf * PT_PAIRS * PBUF + ((kt * 2 + ks) * QH + qh) * 1024);
    };

    if (is_s) {
        // ================= score wavefront =================
        v8 qf[QH][NKS];
        float slope[QH] = {};
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) {
            const T* qr = (const T*)p.Q + (int64_t)row_t[qh] * p.qst + (int64_t)row_h[qh] * p.qsh + 8 * h;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                qf[qh][ks] = v8{};
                if (live[qh] && 16 * ks + 8 * h < p.c.D) qf[qh][ks] = *reinterpret_cast<const v8*>(qr + 16 * ks);
            }
            if (MODE == 2 && p.slopes && live[qh]) slope[qh] = p.slopes[row_h[qh]] * PA_LOG2E;
        }
        if constexpr (MODE == 0) {
#pragma unroll
            for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) pg_scale_f16(qf[qh][ks], p.mul);
        }
        // bounds that every row of the pair shares: inside them no comparison
        int in_lo = 0, in_hi = 0x7fffffff;
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) {
            in_lo = max(in_lo, r_lo[qh]);
            in_hi = min(in_hi, r_hi[qh]);
        }
        for (int i = 1; i < 32; i *= 2) {
            in_lo = max(in_lo, __shfl_xor(in_lo, i, 64));
            in_hi = min(in_hi, __shfl_xor(in_hi, i, 64));
        }
        in_lo = __builtin_amdgcn_readfirstlane(in_lo);
        in_hi = __builtin_amdgcn_readfirstlane(in_hi);

        bool fast = MODE == 0;   // the maximum comes in through the product (wavefront-uniform)
        v8 ones{};
        ones[0] = h == 0 ? (T)1.f : (T)0.f;
        v8 qm[QH];
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) qm[qh] = v8{};
        uint32_t kb0[NKS];
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
            kb0[ks] = lds_addr(&kbuf[0][0]) + (uint32_t)(r32 * RB + (((2 * ks + h) ^ (r32 & 15)) << 4));
        f32x16 st[2][QH];   // register r: key 32 kt + 8 (r / 4) + 4 h + r % 4
        float m[QH];        // the running maximum, -inf: unset
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) m[qh] = -INFINITY;

        auto block = [&](int j, int buf) __attribute__((always_inline)) {
            uint32_t ka[NKS];
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                ka[ks] = kb0[ks] + (uint32_t)((j % PT_KST) * TILE);
                asm("; lds address" : "+v"(ka[ks]));
            }
            auto kread = [&](int f) __attribute__((always_inline)) -> v8 {   // f = 2 ks + kt
                return *(const lds_v8*)(uintptr_t)(ka[f >> 1] + (uint32_t)((f & 1) * 32 * RB));
            };
            v8 fr[PT_PF];
#pragma unroll
            for (int f = 0; f < PT_PF; ++f) fr[f] = kread(f);
            const i4 nn = *(const lds_i4*)(uintptr_t)lds_addr(&nbuf[j % PT_KST][0]);
            if constexpr (MODE == 0) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh) st[kt][qh] = TT::mma32(ones, qm[qh], f32x16{});
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < QH * NSF; ++i) {
                const int f = i / QH, qh = i % QH, ks = f >> 1, kt = f & 1;
                st[kt][qh] = TT::mma32(fr[f % PT_PF], qf[qh][ks], MODE != 0 && ks == 0 ? f32x16{} : st[kt][qh]);
                if (qh == QH - 1 && f + PT_PF < NSF) fr[f % PT_PF] = kread(f + PT_PF);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int none = __builtin_amdgcn_readfirstlane(nn.x | nn.y << 2 | nn.z << 4 | nn.w << 6);
            const int pos0 = __builtin_amdgcn_readfirstlane(first_pos(e0 + j));
            const int src_hi = e0 + j < np ? p.P - 1 : end - 1;
            if constexpr (MODE == 2) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int qh = 0; qh < QH; ++qh)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            float x = pa_score(st[kt][qh][r], p.mul, p.cap2);
                            if (p.slopes) {
                                const float key = (float)(pos0 + 4 * h) + (float)(32 * kt + 8 * (r >> 2) + (r & 3));
                                x = fmaf(-slope[qh], fabsf(r_pos[qh] - key), x);
                            }
                            st[kt][qh][r] = x;
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
            // how far the largest score lies above the maximum (above 0 while it is unset)
            const bool fast_blk = fast;
            const float cm = MODE == 1 ? p.mul : 1.f;
            float vl[QH], ref[QH];
            bool up = false;
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) {
                float v = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) v = fmaxf(v, st[kt][qh][r]);
                const bool unset = m[qh] == -INFINITY;
                ref[qh] = unset ? 0.f : m[qh];
                vl[qh] = MODE == 0 && fast_blk ? v : fmaf(v, cm, -ref[qh]);
                up = up || vl[qh] > (unset ? -INFINITY : PT_RESCALE);
            }
            const bool rescale = __builtin_amdgcn_ballot_w64(up) != 0;
            float sub[QH];   // what P = exp2(score - sub) takes off
#pragma unroll
            for (int qh = 0; qh < QH; ++qh) sub[qh] = MODE == 0 && fast_blk ? 0.f : ref[qh];
            if (rescale) {
                float mn[QH];
                bool far = false;
#pragma unroll
                for (int qh = 0; qh < QH; ++qh) {
                    float a, c;
                    pg_xor32_pair(vl[qh], a, c);
                    const float t = fmaxf(a, c);
                    const bool unset = m[qh] == -INFINITY;
                    mn[qh] = unset ? t : m[qh] + fmaxf(t, 0.f);
                    far = far || (mn[qh] != -INFINITY && !(fabsf(mn[qh]) <= 32768.f));
                }
                // m is kept f16-representable while it enters the product; beyond +-32768 it would be too coarse
                if (MODE == 0 && fast && __builtin_amdgcn_ballot_w64(far) != 0) fast = false;
#pragma unroll
                for (int qh = 0; qh < QH; ++qh) {
                    if (MODE == 0 && fast) mn[qh] = (float)(T)mn[qh];
                    const bool unset = m[qh] == -INFINITY, still = mn[qh] == -INFINITY;
                    const float alpha = unset ? 1.f : __builtin_amdgcn_exp2f(m[qh] - mn[qh]);
                    const float to = still ? 0.f : mn[qh];
                    sub[qh] = MODE == 0 && fast_blk ? to - ref[qh] : to;
                    m[qh] = mn[qh];
                    if constexpr (MODE == 0) qm[qh][0] = (fast && h == 0) ? (T)(-to) : (T)0.f;
                    if (h == 0) abuf[buf][pr][32 * qh + r32] = alpha;
                }
            }
            if (lane == 0) fbuf[buf][pr] = rescale ? 1 : 0;
            auto pstore = [&](auto plain) __attribute__((always_inline)) {
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
                                if constexpr (!decltype(plain)::value) x = MODE == 1 ? fmaf(x, cm, msub) : x + msub;
                                u[k] = (T)__builtin_amdgcn_exp2f(x);
                            }
                            *(lds_v8*)(uintptr_t)paddr(buf, kt, ks, qh) = u;
                        }
            };
            if (MODE == 0 && fast_blk && !rescale)
                pstore(pg_tag<true>{});
            else
                pstore(pg_tag<false>{});
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
    } else {
        // ================= output wavefront =================
        const uint32_t row_bytes = (uint32_t)(p.c.sl * 2);
        uint32_t ofs_k[4], ofs_v[2];   // rows 4 i + lane / 16 of this wavefront's 16
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * i + lane / CH, in8 = row & 7;
            const int ck = (lane % CH) ^ row, cv = (lane % CH) ^ (4 * (row & 3));
            ofs_k[i] = 8 * ck < p.c.D ? (uint32_t)in8 * row_bytes + 16u * (uint32_t)ck : OOB_OFS;
            if (i < 2) ofs_v[i] = 8 * cv < p.c.D ? (uint32_t)in8 * row_bytes + 16u * (uint32_t)cv : OOB_OFS;
        }
        struct Src {
            int page[2], row[2], n[2];   // per 8 keys: the page (-1: none), the row in it, keys below the end
        };
        const pg_table own = (pg_table)(uintptr_t)(p.b.table + (int64_t)max(b, 0) * p.b.max_pages);
        const pg_table shared = (pg_table)(uintptr_t)p.ppages;
        auto lookup = [&](int j) __attribute__((always_inline)) {
            Src t;
            const int blk = e0 + j;
            const bool pre = blk < np;
            const int key0 = (pre ? p0 + blk : o0 + blk - np) * PT_BK + 16 * pr;
            const int len = j < nblk ? (pre ? p.P : seq.kv) : 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int k = key0 + 8 * i;
                t.n[i] = min(max(len - k, 0), 8);
                t.page[i] = 0;
                t.row[i] = 0;
                if (t.n[i] > 0) {
                    const int no_ = (int)div_of((uint32_t)k, p.c.by_page);
                    t.row[i] = k - no_ * p.c.page;
                    const int pg = pre ? shared[no_] : own[no_];
                    t.page[i] = (uint32_t)pg < (uint32_t)p.c.pages ? pg : -1;
                }
            }
            return t;
        };
        auto request = [&](const Src& t, bool is_k, int j) __attribute__((always_inline)) {
            const T* base = (const T*)(is_k ? p.c.k : p.c.v) + (int64_t)head * p.c.sh;
            const uint32_t dst = lds_addr(is_k ? &kbuf[0][0] : &vbuf[0][0]) + (uint32_t)pr * 16 * RB +
                                 (uint32_t)(j % (is_k ? PT_KST : PT_VST)) * TILE;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool none = t.page[i] < 0 || t.n[i] == 0;
                const T* at8 = base + (none ? 0 : (int64_t)t.page[i] * p.c.sp + (int64_t)t.row[i] * p.c.sl);
                const v4i rs = make_rsrc(at8, none ? 0u : (uint32_t)(t.n[i] - 1) * row_bytes + 2u * (uint32_t)p.c.D);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    dma16(rs, is_k ? ofs_k[2 * i + u] : ofs_v[u], 0u,
                          __builtin_amdgcn_readfirstlane(dst + 1024u * (uint32_t)(2 * i + u)));
            }
            if (is_k && lane == 0) nbuf[j % PT_KST][pr] = (t.page[0] < 0 ? 1 : 0) | (t.page[1] < 0 ? 2 : 0);
        };
        Src sv = lookup(0), s1 = lookup(1), s2 = lookup(2);
        request(sv, true, 0);
        request(s1, true, 1);
        request(s2, true, 2);
        request(sv, false, 0);
        Src sk = lookup(3);   // K of block j + 3 is next, V of block j + 1
        sv = s1;
        s1 = s2;

        uint32_t vb0[NDT];
        {
            const int jj = (lane & 15) >> 2, q = lane & 3, dh = (lane >> 4) & 1;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                vb0[dt] = lds_addr(&vbuf[0][0]) +
                          (uint32_t)((4 * h + jj) * RB + (((4 * dt + 2 * dh + (q >> 1)) ^ (4 * jj)) << 4) + ((q & 1) << 3));
        }
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
        for (int j = 0; j < nblk; ++j) {
            const int buf = j & 1;
            // K_{j+3} into K_j's stage, V_{j+1} into V_{j-1}'s, both read in iteration j - 1
            request(sk, true, j + 3);
            request(sv, false, j + 1);
            sv = s1;
            s1 = sk;
            sk = lookup(j + 4);
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
                uint32_t va[NDT];
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    va[dt] = vb0[dt] + (uint32_t)((j % PT_VST) * TILE);
                    asm("; lds address" : "+v"(va[dt]));
                }
                auto vread = [&](int f) __attribute__((always_inline)) -> v8 {   // f = NDT kk + dt
                    const int kk = 16 * (f / NDT), dt = f % NDT;
                    const pg_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va[dt] + (uint32_t)(kk * RB)));
                    const pg_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(va[dt] + (uint32_t)((kk + 8) * RB)));
                    return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                auto pread = [&](int kk, int qh) __attribute__((always_inline)) -> v8 {
                    return *(const lds_v8*)(uintptr_t)paddr(buf, kk >> 1, kk & 1, qh);
                };
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
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // K_{j+3}, V_{j+1} are here
            __syncthreads();
        }
        __syncthreads();   // the maxima are published
#pragma unroll
        for (int qh = 0; qh < QH; ++qh) {
            float a, c;
            pg_xor32_pair(l[qh], a, c);
            const float sum = a + c, inv = sum == 0.f ? 0.f : 1.f / sum;
            if (!live[qh]) continue;
            const int64_t out_row = (int64_t)row_t[qh] * p.Hq + row_h[qh];
            if (whole && b >= 0) {
                T* orow = (T*)p.O + (int64_t)row_t[qh] * p.ost + (int64_t)row_h[qh] * p.osh;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        const int d = 32 * dt + 8 * g4 + 4 * h;
                        const v4 v = {(T)(o[dt][qh][4 * g4] * inv), (T)(o[dt][qh][4 * g4 + 1] * inv), (T)(o[dt][qh][4 * g4 + 2] * inv),
                                      (T)(o[dt][qh][4 * g4 + 3] * inv)};
                        if (d < p.c.D) *reinterpret_cast<v4*>(orow + d) = v;
                    }
                if (p.lse && h == 0) p.lse[out_row] = sum == 0.f ? -INFINITY : (mbuf[pr][32 * qh + r32] + log2f(sum)) * PA_LN2;
            } else {
                const int64_t part = whole ? out_row : (int64_t)(2 * wg + (blk0 == 0 ? 1 : 0)) * BQ + pr * PQ + 32 * qh + r32;
                float* prow = (whole ? p.row_o : prefix ? p.pre_o : p.ws_o) + part * DE + 4 * h;
                if (sum != 0.f) {
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                        for (int g4 = 0; g4 < 4; ++g4) {
                            pa_put(prow + 32 * dt + 8 * g4, o[dt][qh][4 * g4], o[dt][qh][4 * g4 + 1]);
                            pa_put(prow + 32 * dt + 8 * g4 + 2, o[dt][qh][4 * g4 + 2], o[dt][qh][4 * g4 + 3]);
                        }
                }
                if (h == 0) pa_put((float*)((whole ? p.row_ml : prefix ? p.pre_ml : p.ws_ml) + part), mbuf[pr][32 * qh + r32], sum);
            }
        }
    }
    if (!whole && !prefix) {
        const uint32_t a = before + ((uint32_t)head * (uint32_t)sw.tiles + (uint32_t)tile) * (uint32_t)nb;   // the tile's first block
        pa_arrive<T, DE, 2 * PT_PAIRS>(p, a / per, (a + (uint32_t)nb - 1) / per, BQ, min(BQ, rows - tile * BQ), tile * BQ, seq.first,
                                       head, w, lane, &arrived);
    }
    at += (uint32_t)nseg;
    }
}

// ---- host -----------------------------------------------------------------------------

int paged_tile_launch(const PaParams& p, int qh, bool prefix, int dtype, hipStream_t s) {
    const bool plain = p.cap2 == 0.f && !p.slopes && p.mul > 0.f;
    const int64_t tiles = ((int64_t)p.b.T * p.G / (128 * qh) + p.b.B) * p.c.heads;   // no fewer than there are
    LAVA_REQUIRE(tiles <= 0x7fffffff, LAVA_HIP_ERR_UNSUPPORTED, "paged attention: problem too large");
    const unsigned grid = prefix ? PT_GRID : (unsigned)std::max<int64_t>(tiles, PT_GRID);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(128 * PT_PAIRS), 0, s, p, prefix ? 1 : 0); };
    auto by_d = [&](auto type, auto q, auto mode) {
        typedef decltype(type) T;
        constexpr int QH = decltype(q)::value, MODE = decltype(mode)::value;
        p.c.D <= 64 ? go(paged_tile_kernel<T, 64, QH, MODE>) : go(paged_tile_kernel<T, 128, QH, MODE>);
    };
    auto by_mode = [&](auto q) {
        if (dtype == LAVA_HIP_F16)
            plain && p.mul <= 1.f ? by_d(f16{}, q, pg_int<0>{}) : by_d(f16{}, q, pg_int<2>{});
        else
            plain ? by_d(bf16{}, q, pg_int<1>{}) : by_d(bf16{}, q, pg_int<2>{});
    };
    qh == 1 ? by_mode(pg_int<1>{}) : by_mode(pg_int<2>{});
    return check_launch(qh == 1 ? "paged_tile_kernel+paged_tile_kernel<32>" : "paged_tile_kernel");
}

}  // namespace lava
