// The best of many, in order: keys kept one per lane, sorted and merged by a warp.
#pragma once

#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

namespace wocr {
namespace k {
namespace topk {

// A candidate: its value, and its place, which is unique and breaks ties (the lower goes first).
struct Cand {
    double v;
    uint32_t i;
};
__device__ __forceinline__ Cand worst(Cand *) { return {-INFINITY, 0xffffffffu}; }
__device__ __forceinline__ bool better(const Cand &a, const Cand &b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ Cand shfl_xor(const Cand &a, int m) {
    return {__shfl_xor_sync(0xffffffffu, a.v, m), __shfl_xor_sync(0xffffffffu, a.i, m)};
}
__device__ __forceinline__ Cand shfl(const Cand &a, int l) {
    return {__shfl_sync(0xffffffffu, a.v, l), __shfl_sync(0xffffffffu, a.i, l)};
}

// The same for 32-bit values: the value's bits made monotone above the complement of the place.
using Key = unsigned long long;
__device__ __forceinline__ Key worst(Key *) { return 0; }
__device__ __forceinline__ bool better(Key a, Key b) { return a > b; }
__device__ __forceinline__ Key shfl_xor(Key a, int m) { return __shfl_xor_sync(0xffffffffu, a, m); }
__device__ __forceinline__ Key shfl(Key a, int l) { return __shfl_sync(0xffffffffu, a, l); }
__device__ __forceinline__ Key make_key(float v, uint32_t place) {
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 as 0: the two are the same value
    return (Key)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (0xffffffffu - place);
}
__device__ __forceinline__ float key_value(Key k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint32_t key_place(Key k) { return 0xffffffffu - (uint32_t)k; }

// A warp's 32 keys in descending order by lane (Batcher's bitonic network).
template <typename K>
__device__ __forceinline__ K sort32(K a) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int d = size / 2; d; d /= 2) {
            const K o = shfl_xor(a, d);
            const bool first = ((lane & d) == 0) == ((lane & size) == 0 || size == 32);
            if (better(o, a) == first) a = o;
        }
    return a;
}
// The best 32 of two descending lists, descending.
template <typename K>
__device__ __forceinline__ K merge32(K a, K b) {
    const int lane = threadIdx.x & 31;
    b = shfl(b, 31 - lane);
    if (better(b, a)) a = b;
#pragma unroll
    for (int d = 16; d; d /= 2) {
        const K o = shfl_xor(a, d);
        if (better(o, a) == ((lane & d) == 0)) a = o;
    }
    return a;
}
// The best 32 of a block's keys (one per thread, WARPS warps), descending in lanes of warp 0;
// lists: WARPS * 32 keys of shared memory, free again after the block's next barrier.
template <int WARPS, typename K>
__device__ __forceinline__ K block_best32(K a, K *lists) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    a = sort32(a);
#pragma unroll
    for (int n = WARPS / 2; n; n /= 2) {
        if (warp >= n && warp < 2 * n) lists[warp * 32 + lane] = a;
        __syncthreads();
        if (warp < n) a = merge32(a, lists[(warp + n) * 32 + lane]);
    }
    return a;
}

// Logits and scores that are no number never win; an infinite one counts as the largest number.
__device__ __forceinline__ float clean(float x) { return x <= FLT_MAX ? x : (x > FLT_MAX ? FLT_MAX : -INFINITY); }

}  // namespace topk
}  // namespace k
}  // namespace wocr
