// kv_append.hip -- new tokens' keys and values into the paged cache, rotated on the way.
//
// Per token at position pos and pair j: angle = pos * inv_freq[j]; (x, y) -> (x cos - y sin, y cos + x sin),
// the pair's elements (j, j + R/2) or (2j, 2j + 1).  Keys, and queries beside them, turn; values are copied.
//
// Bound by HBM for prompts and by its chain of lookups for a decode step.  A workgroup takes one token: each of its
// wavefronts finds the token's sequence and page by one ballot over q_start (not a chain of dependent loads), the
// token's cosines and sines are computed once into LDS for all heads, and every thread moves two 16-byte
// chunks, those of a pair where halves turn.  The angle in turns, pos * inv_freq / 2 pi, is reduced in 64 bits
// (at position 2^20 32 bits would be off by 0.06 of a radian); sine and cosine of the rest are in 32.
// Measured (32 + 2 x 8 heads, D = 128): 64 decoded tokens 4.6 us, of which the launch and its lookups are all but 0.3; 16 prompts
// of 333 to 4096 tokens 122 us, 5.5 TB/s of what is read and written.

#include "paged.hpp"

#include <algorithm>

namespace lava {

struct AppendParams {
    PagedCache c;
    PagedBatch b;
    const void* K;
    const void* V;
    const void* Q;
    void* Qo;
    int64_t ksh, kst, qsh, qst, osh, ost;   // head and token strides
    int Hq;                                  // 0: no queries
    const float* inv_freq;
    const int* positions;
    int offset, rot, interleaved;
};

constexpr int KA_THREADS = 256;
constexpr double KA_TURN = 0.15915494309189533577;   // 1 / 2 pi

__device__ __forceinline__ float2 ka_cos_sin(int pos, float inv_freq) {
    const double t = (double)pos * ((double)inv_freq * KA_TURN);
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    return make_float2(c, s);
}

// Where token t goes: its position (for the rotation), and the cache's element offset of its row in head 0
// (-1: no page).  Computed by a wavefront together.
struct KaToken {
    int live, pos;
    int64_t at;
};
__device__ __forceinline__ KaToken ka_token(const AppendParams& p, int t, int lane) {
    KaToken r = {0, 0, -1};
    if (t >= p.b.T) return r;
    const int b = paged_find(p.b, t, lane);
    if (b >= p.b.B) return r;
    const PagedSeq s = paged_seq(p.b, b);
    if (t < s.first || t >= s.first + s.n) return r;   // in front of the first sequence, or starts out of order
    r.live = 1;
    const int slot = s.kv - s.n + (t - s.first);        // negative: more new tokens than the cache is said to hold
    r.pos = p.positions ? p.positions[t] : p.offset + slot;
    if (slot >= 0) {
        const int page_no = (int)div_of((uint32_t)slot, p.c.by_page);
        const int page = p.b.table[(int64_t)b * p.b.max_pages + page_no];
        if (page >= 0 && page < p.c.pages)
            r.at = (int64_t)page * p.c.sp + (int64_t)(slot - page_no * p.c.page) * p.c.sl;
    }
    return r;
}

// Vectors of 8: D a multiple of 8, the rotation's halves whole vectors, 16-byte alignment everywhere.
// A token a workgroup.
template <typename T>
__global__ void __launch_bounds__(KA_THREADS) kv_append_kernel(AppendParams p) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    extern __shared__ float2 turn[];   // rot / 2
    const int tid = threadIdx.x, lane = tid & 63;
    const int t = (int)pg_block();
    const KaToken k = ka_token(p, t, lane);   // by every wavefront: the same
    if (!k.live) return;
    for (int j = tid; j < p.rot / 2; j += KA_THREADS) turn[j] = ka_cos_sin(k.pos, p.inv_freq[j]);
    __syncthreads();

    const int chunks = p.c.D / 8, items = (chunks + 1) / 2, half = p.interleaved ? 0 : p.rot / 16;
    const int heads = p.Hq + 2 * p.c.heads;
    for (int n = tid; n < heads * items; n += KA_THREADS) {
        const int h = n / items, m = n - h * items;
        const int c0 = m < half ? m : 2 * m, c1 = m < half ? m + half : 2 * m + 1;
        const bool two = c1 < chunks;
        const T* src;
        T* dst;
        bool turns = p.rot > 0;
        if (h < p.Hq) {
            src = (const T*)p.Q + (int64_t)t * p.qst + (int64_t)h * p.qsh;
            dst = (T*)p.Qo + (int64_t)t * p.ost + (int64_t)h * p.osh;
        } else {
            if (k.at < 0) continue;
            const bool is_v = h >= p.Hq + p.c.heads;
            const int hk = h - p.Hq - (is_v ? p.c.heads : 0);
            src = (const T*)(is_v ? p.V : p.K) + (int64_t)t * p.kst + (int64_t)hk * p.ksh;
            dst = (T*)(is_v ? p.c.v : p.c.k) + k.at + (int64_t)hk * p.c.sh;
            turns = turns && !is_v;
        }
        v8 x = *reinterpret_cast<const v8*>(src + 8 * c0), y{};
        if (two) y = *reinterpret_cast<const v8*>(src + 8 * c1);
        if (turns) {
            if (m < half) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 cs = turn[8 * m + e];
                    const float a = (float)x[e], b = (float)y[e];
                    x[e] = (T)(a * cs.x - b * cs.y);
                    y[e] = (T)(b * cs.x + a * cs.y);
                }
            } else if (p.interleaved) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    v8& z = u ? y : x;
                    const int c = u ? c1 : c0;
                    if (8 * c >= p.rot) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 cs = turn[4 * c + e];
                        const float a = (float)z[2 * e], b = (float)z[2 * e + 1];
                        z[2 * e] = (T)(a * cs.x - b * cs.y);
                        z[2 * e + 1] = (T)(b * cs.x + a * cs.y);
                    }
                }
            }
        }
        *reinterpret_cast<v8*>(dst + 8 * c0) = x;
        if (two) *reinterpret_cast<v8*>(dst + 8 * c1) = y;
    }
}

// Any head dimension, strides and alignment: one wavefront a token, a pair (or an element that does not turn) a lane.
template <typename T>
__global__ void __launch_bounds__(64) kv_append_any_kernel(AppendParams p) {
    const int t = (int)pg_block(), lane = threadIdx.x;
    const KaToken k = ka_token(p, t, lane);
    if (!k.live) return;
    const int half = p.rot / 2, D = p.c.D;
    for (int m = lane; m < D - half; m += 64) {   // pairs m < half, then the elements behind them
        const bool pair = m < half;
        const int e0 = pair ? (p.interleaved ? 2 * m : m) : m + half;
        const int e1 = pair ? (p.interleaved ? 2 * m + 1 : m + half) : e0;
        const float2 cs = pair ? ka_cos_sin(k.pos, p.inv_freq[m]) : make_float2(1.f, 0.f);
        for (int h = 0; h < p.Hq + 2 * p.c.heads; ++h) {
            const T* src;
            T* dst;
            bool turns = pair;
            if (h < p.Hq) {
                src = (const T*)p.Q + (int64_t)t * p.qst + (int64_t)h * p.qsh;
                dst = (T*)p.Qo + (int64_t)t * p.ost + (int64_t)h * p.osh;
            } else {
                if (k.at < 0) continue;
                const bool is_v = h >= p.Hq + p.c.heads;
                const int hk = h - p.Hq - (is_v ? p.c.heads : 0);
                src = (const T*)(is_v ? p.V : p.K) + (int64_t)t * p.kst + (int64_t)hk * p.ksh;
                dst = (T*)(is_v ? p.c.v : p.c.k) + k.at + (int64_t)hk * p.c.sh;
                turns = pair && !is_v;
            }
            const T x = src[e0], y = src[e1];
            const float a = (float)x, b = (float)y;
            dst[e0] = turns ? (T)(a * cs.x - b * cs.y) : x;
            if (pair) dst[e1] = turns ? (T)(b * cs.x + a * cs.y) : y;
        }
    }
}

}  // namespace lava

using namespace lava;

extern "C" int lava_hip_kv_append(const lava_hip_kv_cache* cache, const lava_hip_kv_batch* batch, const void* K,
                                  const void* V, const int64_t* kv_strides, const void* Q, void* Q_out, int64_t q_heads,
                                  const int64_t* q_strides, const int64_t* qo_strides, const lava_hip_rope* rope,
                                  void* stream) {
    AppendParams p = {};
    int rc = paged_check("kv_append", cache, batch, &p.c, &p.b);
    if (rc != LAVA_HIP_OK) return rc;
    const int D = p.c.D;
    if (rope) {
        LAVA_ARG(rope->rot_dim >= 0 && rope->rot_dim <= D && rope->rot_dim % 2 == 0,
                 "kv_append: rot_dim = %d is not an even number up to the head dimension %d", rope->rot_dim, D);
        LAVA_ARG(rope->rot_dim == 0 || rope->inv_freq, "kv_append: null inv_freq");
        LAVA_ARG(aligned(rope->inv_freq, 4) && aligned(rope->positions, 4), "kv_append: inv_freq or positions misaligned");
        LAVA_ARG(rope->offset >= 0 && rope->offset <= 0x40000000, "kv_append: offset = %d is outside [0, 2^30]", rope->offset);
        p.inv_freq = rope->inv_freq;
        p.rot = rope->rot_dim;
        p.interleaved = rope->interleaved != 0;
        p.positions = rope->positions;
        p.offset = rope->offset;
    }
    LAVA_ARG(q_heads >= 0 && q_heads <= 65535, "kv_append: q_heads = %lld is outside [0, 65535]", (long long)q_heads);
    if (p.b.T == 0 || p.b.B == 0) return LAVA_HIP_OK;
    LAVA_ARG(K && V && kv_strides, "kv_append: null pointer");
    LAVA_ARG((Q == nullptr) == (Q_out == nullptr), "kv_append: Q and Q_out go together");
    rc = paged_check_strides("kv_append", "kv_strides", kv_strides, D, p.c.heads, p.b.T);
    if (rc != LAVA_HIP_OK) return rc;
    p.K = K;
    p.V = V;
    p.ksh = kv_strides[1];
    p.kst = kv_strides[2];
    bool vec = D % 8 == 0 && p.c.sl % 8 == 0 && p.c.sh % 8 == 0 && p.c.sp % 8 == 0 && p.ksh % 8 == 0 && p.kst % 8 == 0 &&
               aligned(p.c.k, 16) && aligned(p.c.v, 16) && aligned(K, 16) && aligned(V, 16) &&
               p.rot % (p.interleaved ? 8 : 16) == 0;
    LAVA_ARG(aligned(K, 2) && aligned(V, 2) && aligned(Q, 2) && aligned(Q_out, 2), "kv_append: misaligned");
    if (Q && q_heads > 0) {
        LAVA_ARG(q_strides && qo_strides, "kv_append: null pointer");
        rc = paged_check_strides("kv_append", "q_strides", q_strides, D, q_heads, p.b.T);
        if (rc != LAVA_HIP_OK) return rc;
        rc = paged_check_strides("kv_append", "qo_strides", qo_strides, D, q_heads, p.b.T);
        if (rc != LAVA_HIP_OK) return rc;
        LAVA_ARG(Q != Q_out || (q_strides[1] == qo_strides[1] && q_strides[2] == qo_strides[2]),
                 "kv_append: Q in place needs the strides of Q_out");
        p.Q = Q;
        p.Qo = Q_out;
        p.Hq = (int)q_heads;
        p.qsh = q_strides[1];
        p.qst = q_strides[2];
        p.osh = qo_strides[1];
        p.ost = qo_strides[2];
        vec = vec && aligned(Q, 16) && aligned(Q_out, 16) && p.qsh % 8 == 0 && p.qst % 8 == 0 && p.osh % 8 == 0 && p.ost % 8 == 0;
    }
    rc = lava_hip_init();
    if (rc != LAVA_HIP_OK) return rc;
    rc = paged_check_device("kv_append", p.c.k, stream);
    if (rc != LAVA_HIP_OK) return rc;
    hipStream_t s = as_stream(stream);
    const bool f16s = cache->dtype == LAVA_HIP_F16;
    if (!vec) {
        if (f16s)
            hipLaunchKernelGGL((kv_append_any_kernel<f16>), pg_grid(p.b.T), dim3(64), 0, s, p);
        else
            hipLaunchKernelGGL((kv_append_any_kernel<bf16>), pg_grid(p.b.T), dim3(64), 0, s, p);
        LAVA_LAUNCH_CHECK("kv_append_any_kernel");
        return LAVA_HIP_OK;
    }
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, pg_grid(p.b.T), dim3(KA_THREADS), (size_t)(p.rot / 2) * sizeof(float2), s, p);
    };
    f16s ? go(kv_append_kernel<f16>) : go(kv_append_kernel<bf16>);
    LAVA_LAUNCH_CHECK("kv_append_kernel");
    return LAVA_HIP_OK;
}
