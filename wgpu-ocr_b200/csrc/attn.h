// Attention, what its kernels share: the score of a query and a key, which keys a query sees, warp
// matrix instructions, the join of partial results, and one query row by a warp straight from the
// definition.
#pragma once

#include <cooperative_groups.h>

#include "elem.h"
#include "ops.h"

namespace wocr {
namespace k {
namespace attn {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234e38f; }

// What the masks leave of a batch element: rows below nq are its queries, keys below nk its keys;
// query i stands at position off + i among the keys.
struct Span {
    int nq, nk, off, prefix;
};
__device__ __forceinline__ Span span_of(const AttnP &p, int b) {
    Span s;
    // lengths come from the caller's device memory: held to the tensors' sizes
    s.nk = p.kv_lens ? min(max(p.kv_lens[b], 0), p.kv_len) : p.kv_len;
    s.nq = p.q_lens ? min(max(p.q_lens[b], 0), p.q_len) : p.q_len;
    s.off = s.nk - s.nq;
    s.prefix = p.prefix ? p.prefix[b] : 0;
    return s;
}
// keys that query i may see: j < key_end(i) (documents apart)
__device__ __forceinline__ int key_end(const AttnP &p, const Span &s, int i) {
    return p.causal ? min(s.nk, max(s.prefix, s.off + i + 1)) : s.nk;
}

// cap tanh(y / cap) in units of log 2.  A score's error is a relative error of its weight: with
// 32-bit values tanhf (within 2 ulp), with 16-bit values 1 - 2 / (1 + e^2y) from two approximate
// instructions, within 2^-22 of the cap: up to a cap of 256 an eighth of a weight's rounding to fp16.
// Wider caps, whose scores may all be near zero, take tanhf.
static __device__ __noinline__ float capped32(float y, float cap) { return cap * tanhf(y / cap) * kLog2e; }
template <typename T>
__host__ __device__ __forceinline__ bool by_tanh(float cap) { return sizeof(T) == 4 || cap > 256.f || cap < 0x1p-100f; }
__device__ __forceinline__ float capped16(float y, float cap) {
    y *= 2.f * kLog2e / cap;
    if (y > 126.f) y = 126.f;  // (a NaN passes)
    return cap * kLog2e * (1.f - __fdividef(2.f, 1.f + ex2(y)));
}
template <typename T>
__device__ __forceinline__ float capped2(float y, float cap) {
    return by_tanh<T>(cap) ? capped32(y, cap) : capped16(y, cap);  // a call: inlined over a tile it fills the instruction caches
}
// Scores that are more than a product, or documents: kernels are built with and without them, since
// the code of all of them together, unrolled over a tile, does not fit in the instruction caches.
inline bool extra_scores(const AttnP &p) { return p.cap > 0.f || p.slopes || p.q_docs; }
// A score in units of log 2 from the dot product: cap tanh(scale dot / cap) (or scale dot) less
// slope |distance|.
template <typename T>
__device__ __forceinline__ float score2(const AttnP &p, float dot, float slope, int dist) {
    float s = p.cap > 0.f ? capped2<T>(dot * p.scale, p.cap) : dot * (p.scale * kLog2e);
    return s - slope * kLog2e * fabsf((float)dist);
}

// Row i of (b, h) by one warp from global memory, two passes over the keys: the maximum and the sum
// of the weights, then the weighted values.  Keys behind a mask are never read into a sum, so NaN
// and infinities there stay where they are.  Slow and right for every shape: the kernels hand it
// the rows whose sums came out non-finite.
template <typename T>
__device__ __noinline__ void row_by_warp(const AttnP &p, int b, int h, int i) {
    const int lane = threadIdx.x & 31;
    const Span sp = span_of(p, b);
    if (i >= sp.nq) return;
    const int hk = h / (p.heads / p.kv_heads);
    const T *q = (const T *)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)i * p.qs[2];
    const T *kb = (const T *)p.k + b * p.ks[0] + hk * p.ks[1];
    const T *vb = (const T *)p.v + b * p.vs[0] + hk * p.vs[1];
    T *o = (T *)p.o + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
    const int end = key_end(p, sp, i);
    const float slope = p.slopes ? p.slopes[h] : 0.f;
    const int doc = p.q_docs ? p.q_docs[b * p.qds + i] : 0;
    auto sees = [&](int j) -> bool { return j < end && !(p.q_docs && (doc < 0 || p.kv_docs[b * p.kds + j] != doc)); };
    auto score = [&](int j) -> float {
        if (!sees(j)) return -INFINITY;
        const T *kr = kb + (int64_t)j * p.ks[2];
        float dot = 0.f;
        for (int d = 0; d < p.dim; d++) dot = fmaf(to_f(q[d]), to_f(kr[d]), dot);
        return score2<T>(p, dot, slope, sp.off + i - j);
    };
    float m = -INFINITY, l = 0.f;
    bool any = false;
    for (int j0 = 0; j0 < end; j0 += 32) {
        any |= sees(j0 + lane);
        const float s = score(j0 + lane);
        const float mn = fmaxf(m, s);
        const float base = mn == -INFINITY ? 0.f : mn;
        l = l * ex2(m - base) + ex2(s - base);
        m = mn;
    }
    for (int k = 16; k; k >>= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m, k), lo = __shfl_xor_sync(0xffffffffu, l, k);
        const float mn = fmaxf(m, mo);
        const float base = mn == -INFINITY ? 0.f : mn;
        l = l * ex2(m - base) + lo * ex2(mo - base);
        m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
    // a row that sees nothing is zero; one whose every score is -inf has no weights, 0 / 0
    const float inv = l == 0.f ? 0.f : 1.f / l, start = __any_sync(0xffffffffu, any) && l == 0.f ? NAN : 0.f;
    float acc[8];  // dimensions lane, lane + 32, ... of at most 256
#pragma unroll
    for (int x = 0; x < 8; x++) acc[x] = start;
    for (int j0 = 0; j0 < end; j0 += 32) {
        const float s = score(j0 + lane);
        // NaN scores stay NaN.  Divided here, so that the sum stays below the largest value.
        float w = s == -INFINITY ? 0.f : ex2(s - base) * inv;
        // The exponential ends at 2^-126.  What is seen keeps a weight above zero, so that its infinities come
        // through as they do by the definition; the mark stands for zero with finite values.
        constexpr float mark = 0x1p-149f;
        if (w == 0.f && s > -INFINITY) w = mark;
        const uint32_t seen = __ballot_sync(0xffffffffu, sees(j0 + lane));
        for (int jj = 0; jj < 32; jj++) {
            const float wj = __shfl_sync(0xffffffffu, w, jj);
            if (!(seen >> jj & 1)) continue;  // unseen keys' values are not touched
            const T *vr = vb + (int64_t)(j0 + jj) * p.vs[2];
#pragma unroll
            for (int x = 0; x < 8; x++)
                if (lane + 32 * x < p.dim) {
                    const float u = to_f(vr[lane + 32 * x]);
                    acc[x] = fmaf(wj == mark && finite(u) ? 0.f : wj, u, acc[x]);
                }
        }
    }
#pragma unroll
    for (int x = 0; x < 8; x++)
        if (lane + 32 * x < p.dim) o[lane + 32 * x] = from_f<T>(acc[x]);
}

// Whether row i may see a key, as far as its lengths and its own document tell.
__device__ __forceinline__ bool may_see(const AttnP &p, const Span &s, int b, int i) {
    return i >= 0 && key_end(p, s, i) > 0 && (!p.q_docs || p.q_docs[b * p.qds + i] >= 0);
}
// A document that is not among the first `end` keys.
struct Absent {
    int doc = -1, end = 0;
};
// row_by_warp for a row whose sums are not finite, or whose weights are all zero although it may see keys: where a
// document has no keys (rows of padding, a run of one document) one look at the ids serves all of them, so the
// rows of a block come last to first.
template <typename T>
__device__ __noinline__ Absent row_again(const AttnP &p, int b, int h, int i, Absent none) {
    if (p.q_docs) {
        const int lane = threadIdx.x & 31, doc = p.q_docs[b * p.qds + i], end = key_end(p, span_of(p, b), i);
        const int *ids = p.kv_docs + b * p.kds;
        bool in = false;
        if (doc >= 0 && !(doc == none.doc && end <= none.end))
            for (int j0 = lane; j0 - lane < end && !in; j0 += 256) {
                int d[8];
#pragma unroll
                for (int x = 0; x < 8; x++) d[x] = j0 + x * 32 < end ? ids[j0 + x * 32] : -1;
#pragma unroll
                for (int x = 0; x < 8; x++) in |= d[x] == doc;
                in = __any_sync(0xffffffffu, in);
            }
        if (!in) {
            if (doc >= 0 && !(doc == none.doc && end <= none.end)) none = {doc, end};
            T *o = (T *)p.o + b * p.os[0] + h * p.os[1] + (int64_t)i * p.os[2];
            for (int d = lane; d < p.dim; d += 32) o[d] = from_f<T>(0.f);
            return none;
        }
    }
    row_by_warp<T>(p, b, h, i);
    return none;
}

// ---- warp matrix instructions (16 x 8 x 16, fp32 accumulators) -----------------------------
template <typename E>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<E, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
            "%2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
            "%2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p))
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p))
                 : "memory");
}
// two values rounded to E in one word, the first in the low half
template <typename E>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if constexpr (std::is_same<E, __half>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}

// 32-bit values on 16-bit matrix instructions: x = h0 + h1 + h2 with three bf16 parts hold its 24
// bits exactly, and the six products of order 2^-16 and more leave 2^-23 of |x y| out.
// Operand element and number of parts of a tensor type:
template <typename T>
struct Parts {
    using E = T;
    static constexpr int n = 1;
};
template <>
struct Parts<float> {
    using E = __nv_bfloat16;
    static constexpr int n = 3;
};
// parts[x] of two values, packed
template <typename T>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&parts)[Parts<T>::n]) {
    using E = typename Parts<T>::E;
    parts[0] = pack2<E>(x, y);
    if constexpr (Parts<T>::n == 3) {
#pragma unroll
        for (int i = 1; i < 3; i++) {
            x -= __uint_as_float(parts[i - 1] << 16);
            y -= __uint_as_float(parts[i - 1] & 0xffff0000u);
            parts[i] = pack2<E>(x, y);
        }
    }
}

// ---- partial results ------------------------------------------------------------------------
// Sums over some of the keys for 16 rows: maximum and sum of the weights, and the weighted values.
template <int DP>
struct PartSums {
    float o[16][DP];
    float m[16], l[16];
};
struct JoinSmem {
    float weight[512], l[512];  // per part and row of the cluster: maximum, then share; sum
    uint8_t odd[64];            // rows to work out again
};

// The parts of a cluster's blocks, joined and stored.  Four warps of a block wrote parts[warp]:
// with PER = 4 the same 16 rows each, with PER = 1 rows 16 warp ..; row r is query query(r) of head
// head(r), query < 0: none.  The blocks share the values out.
template <typename T, int DP, int PER, typename Head, typename Query>
__device__ __forceinline__ void join_parts(const AttnP &p, int b, PartSums<DP> *parts, JoinSmem &js, Head &&head, Query &&query) {
    constexpr int ROWS = PER == 4 ? 16 : 64;
    cg::cluster_group cl = cg::this_cluster();
    const int cs = cl.num_blocks(), rank = cl.block_rank();
    cl.sync();
    // the loads from other blocks go out together: one after another they take longer than the sums
    const int n = cs * PER;  // parts of a row
    for (int x = threadIdx.x; x < n * ROWS; x += 128) {
        const int r = x % ROWS, c = x / ROWS / PER, w = PER == 4 ? x / ROWS % 4 : r / 16;
        const PartSums<DP> &pt = cl.map_shared_rank(parts, c)[w];
        js.weight[x] = pt.m[r % 16];
        js.l[x] = pt.l[r % 16];
    }
    __syncthreads();
    if (threadIdx.x < ROWS) {
        const int r = threadIdx.x;
        float m = -INFINITY, l = 0.f;
        js.odd[r] = 0;
        for (int x = 0; x < n; x++) m = fmaxf(m, js.weight[x * ROWS + r]);
        const float z = m == -INFINITY ? 0.f : m;
        for (int x = 0; x < n; x++) {
            const float f = ex2(js.weight[x * ROWS + r] - z);
            l += f * js.l[x * ROWS + r];
            js.weight[x * ROWS + r] = f;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (l == 0.f && rank == 0) js.odd[r] = may_see(p, span_of(p, b), b, query(r));
        for (int x = 0; x < n; x++) js.weight[x * ROWS + r] *= inv;
    }
    __syncthreads();
    for (int u = rank * 128 + threadIdx.x; u < ROWS * DP; u += cs * 128) {
        const int r = u / DP, d = u % DP, i = query(r);
        if (i < 0 || d >= p.dim) continue;
        float of[8][PER], v = 0.f;
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int w = 0; w < PER; w++)
                of[c][w] = c < cs ? cl.map_shared_rank(parts, c)[PER == 4 ? w : r / 16].o[r % 16][d] : 0.f;
#pragma unroll
        for (int c = 0; c < 8; c++)
#pragma unroll
            for (int w = 0; w < PER; w++)
                if (c < cs) v += js.weight[(c * PER + w) * ROWS + r] * of[c][w];
        if (!finite(v)) js.odd[r] = 1;
        ((T *)p.o)[b * p.os[0] + head(r) * p.os[1] + (int64_t)i * p.os[2] + d] = from_f<T>(v);
    }
    cl.sync();  // the parts are read until here; non-finite rows are written after the others
    Absent none;
    for (int r = ROWS - 1 - (threadIdx.x >> 5); r >= 0; r -= 4)
        if (js.odd[r] && query(r) >= 0) none = row_again<T>(p, b, head(r), query(r), none);
}

// Blocks of `kernel` that an SM holds at a time, or four: more do not read faster.
template <typename K>
inline int resident(K *kernel, int threads, size_t smem) {
    int n = 0;
    if (smem > 48 * 1024) WOCR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    WOCR_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem));
    return n < 1 ? 1 : (n > 4 ? 4 : n);
}
// Blocks of a cluster that share the keys of one unit of work: the number whose rounds of blocks
// (`per_sm` at a time on an SM, `step` keys at a time) over its keys, and 512 keys' worth of beginning and joining, take
// least (8,192 keys, 32 x 8 key heads, four rows: of 128, 208 us with one block a unit against 236 with
// four; of 64, 123 us with four against 157 with eight).
inline int key_split(const Ctx *c, int64_t units, int per_sm, int kv_len, int step) {
    constexpr int start = 512;
    int best = 1;
    int64_t least = INT64_MAX;
    for (int cs = 1; cs <= 8 && (cs == 1 || kv_len >= cs * step); cs *= 2) {
        const int64_t at_once = (int64_t)per_sm * c->sm_count, rounds = (units * cs + at_once - 1) / at_once;
        const int64_t cost = rounds * ((kv_len + cs - 1) / cs + start);
        if (cost < least) least = cost, best = cs;
    }
    return best;
}
template <typename... A>
inline void launch_cluster(void (*kernel)(A...), dim3 grid, int threads, int cs, size_t smem, cudaStream_t s, A... args) {
    if (smem > 48 * 1024) WOCR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    WOCR_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace attn
}  // namespace k
}  // namespace wocr
