// Attention, what its kernels share: the score of a query and a key, which keys a query sees, and
// one query row by a warp straight from the definition.
#pragma once

#include "elem.h"
#include "ops.h"

namespace wocr {
namespace k {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// The score in units of log 2 from the dot product: cap tanh(scale dot / cap) (or scale dot),
// less slope |distance|.  tanhf is within 2 ulp; the 32-bit path needs that (a score error is a
// relative error of the weight).
__device__ __forceinline__ float score2(const AttnP &p, float dot, float slope, int dist) {
    float s = dot * p.scale;
    if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
    s -= slope * fabsf((float)dist);
    return s * kLog2e;
}

// Row i of (b, h) by one warp from global memory, two passes over the keys: the maximum and the sum
// of the weights, then the weighted values.  Keys behind a mask are never read into a sum, so NaN
// and infinities there stay where they are.  Slow and right for every shape: the other kernels hand
// it the rows whose sums came out non-finite.
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
    auto score = [&](int j) -> float {
        if (j >= end) return -INFINITY;
        if (p.q_docs && (doc < 0 || p.kv_docs[b * p.kds + j] != doc)) return -INFINITY;
        const T *kr = kb + (int64_t)j * p.ks[2];
        float dot = 0.f;
        for (int d = 0; d < p.dim; d++) dot = fmaf(to_f(q[d]), to_f(kr[d]), dot);
        return score2(p, dot, slope, sp.off + i - j);
    };
    float m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 < end; j0 += 32) {
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
    float acc[8];  // dimensions lane, lane + 32, ... of at most 256
#pragma unroll
    for (int x = 0; x < 8; x++) acc[x] = 0.f;
    for (int j0 = 0; j0 < end; j0 += 32) {
        const float s = score(j0 + lane);
        const float w = s == -INFINITY ? 0.f : ex2(s - base);  // NaN scores stay NaN
        for (int jj = 0; jj < 32; jj++) {
            const float wj = __shfl_sync(0xffffffffu, w, jj);
            if (wj == 0.f) continue;  // unseen keys' values are not touched
            const T *vr = vb + (int64_t)(j0 + jj) * p.vs[2];
#pragma unroll
            for (int x = 0; x < 8; x++)
                if (lane + 32 * x < p.dim) acc[x] = fmaf(wj, to_f(vr[lane + 32 * x]), acc[x]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is zero
#pragma unroll
    for (int x = 0; x < 8; x++)
        if (lane + 32 * x < p.dim) o[lane + 32 * x] = from_f<T>(acc[x] * inv);
}

}  // namespace attn
}  // namespace k
}  // namespace wocr
