// The best of many, in order: keys that compare as (value, place), and a bound of the k best.
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

// The best key of each of 32 groups of N threads (N / 32 lanes each), into slots[32] of shared memory:
// the k-th best of them (kth_slot, after a barrier) has k - 1 keys of other groups before it, so it
// bounds the k best keys of all N threads' values from below, and few others pass it.
template <int N, typename K>
__device__ __forceinline__ void best_slots(K a, int tid, K *slots) {
#pragma unroll
    for (int d = 1; d < N / 32; d *= 2) {
        const K o = shfl_xor(a, d);
        if (better(o, a)) a = o;
    }
    if (tid % (N / 32) == 0) slots[tid / (N / 32)] = a;
}
template <typename K>
__device__ __forceinline__ K kth_slot(const K *slots, int k) {  // by a whole warp
    const K mine = slots[threadIdx.x & 31];
    int before = 0;
#pragma unroll 8
    for (int o = 0; o < 32; o++) before += better(slots[o], mine);
    const uint32_t at = __ballot_sync(0xffffffffu, before == k - 1);
    return at ? shfl(mine, __ffs(at) - 1) : worst((K *)nullptr);  // fewer than k groups have a key
}

// Logits and scores that are no number never win; an infinite one counts as the largest number.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }  // (of a NaN and a number, the number)

}  // namespace topk
}  // namespace k
}  // namespace wocr
