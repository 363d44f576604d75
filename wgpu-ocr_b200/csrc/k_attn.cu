// Softmax attention with capped scores, a bias by distance and causal, prefix and document masks.
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(s_ij - max_j s_ij) over the keys that i sees
// One pass over the keys: the running maximum and sum of a row rescale what it has summed.
#include <algorithm>
#include <type_traits>

#include "attn.h"
#include "attn_tc.h"

namespace wocr {
namespace k {

namespace {
using namespace attn;

// Keys of a tile.  32-bit heads above 128 take half tiles: three parts of queries, keys and values
// have to fit in shared memory.
template <typename T, int DP>
constexpr int tile_keys() { return Parts<T>::n * DP > 384 ? 32 : 64; }

template <typename T, int DP>
struct TileSmem {
    static constexpr int P = Parts<T>::n, BK = tile_keys<T, DP>();
    static constexpr int LD = DP + 8;  // elements per row: eight rows start in eight different 16-byte banks
    static constexpr bool q_in_regs = P * DP <= 128;
    static constexpr int q_rows = q_in_regs ? 0 : 64;
    static constexpr int stages = P == 1 ? 2 : 1;  // 16-bit tiles arrive behind the one in work
    static constexpr size_t q = (size_t)P * q_rows * LD * 2, kv = (size_t)P * BK * LD * 2;
    static constexpr size_t tiles = q + 2 * stages * kv, parts = 4 * sizeof(PartSums<DP>);
    static constexpr size_t bytes = tiles > parts ? tiles : parts;
};

// ROWS rows of a [.., dim] tensor from row r0 on for shared memory, 8 elements a unit: fetched into a
// thread's registers, all loads under way together, and put as parts.  Rows from `end` on and
// dimensions from dim on become zero.
template <typename T, int DP, int ROWS>
struct Units {
    static constexpr int n = ROWS * DP / 8 / 128;
    T v[n][8];
    __device__ __forceinline__ void fetch(const T *src, int64_t stride, int r0, int end, int dim, bool vec) {
#pragma unroll
        for (int y = 0; y < n; y++) {
            const int u = y * 128 + threadIdx.x, r = u / (DP / 8), d0 = u % (DP / 8) * 8;
            const bool in = r0 + r < end;
            const T *s = src + (int64_t)(r0 + r) * stride + d0;
            if (in && vec && d0 + 8 <= dim) {
#pragma unroll
                for (int x = 0; x < (int)sizeof(T) / 2; x++) reinterpret_cast<uint4 *>(v[y])[x] = reinterpret_cast<const uint4 *>(s)[x];
            } else {
#pragma unroll
                for (int x = 0; x < 8; x++) v[y][x] = in && d0 + x < dim ? s[x] : from_f<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ void put(uint16_t *dst) const {
        constexpr int P = Parts<T>::n, LD = DP + 8;
#pragma unroll
        for (int y = 0; y < n; y++) {
            const int u = y * 128 + threadIdx.x, r = u / (DP / 8), d0 = u % (DP / 8) * 8;
            if constexpr (P == 1) {
                *reinterpret_cast<uint4 *>(dst + r * LD + d0) = *reinterpret_cast<const uint4 *>(v[y]);
            } else {
                uint32_t w[4][P];
#pragma unroll
                for (int x = 0; x < 4; x++) split2<T>(v[y][2 * x], v[y][2 * x + 1], w[x]);
#pragma unroll
                for (int z = 0; z < P; z++)
                    *reinterpret_cast<uint4 *>(dst + (z * ROWS + r) * LD + d0) = make_uint4(w[0][z], w[1][z], w[2][z], w[3][z]);
            }
        }
    }
};
// The same of 16-bit rows with 16-byte loads, straight to shared memory behind the thread's back.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void copy_rows(uint16_t *dst, const T *src, int64_t stride, int r0, int end, int dim) {
#pragma unroll
    for (int u = threadIdx.x; u < ROWS * DP / 8; u += 128) {
        const int r = u / (DP / 8), d0 = u % (DP / 8) * 8;
        const int bytes = r0 + r < end ? min(max(dim - d0, 0), 8) * 2 : 0;  // the rest is filled with zeros
        const T *s = bytes ? src + (int64_t)(r0 + r) * stride + d0 : src;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(dst + r * (DP + 8) + d0)),
                     "l"(s), "r"(bytes)
                     : "memory");
    }
}

// Products of parts (x, y) with x + y < the number of parts, the pair of leading parts into c and the
// others into low: the matrix instruction cuts its sums off instead of rounding them, so the small
// products do not go through the large sums (32-bit results over 400 keys were 1e-6 off with one sum).
template <typename T, int N>
__device__ __forceinline__ void mma_parts(float (&c)[4], float (&low)[4], const uint32_t (&a)[N][4], const uint32_t (&b0)[N],
                                          const uint32_t (&b1)[N]) {
#pragma unroll
    for (int y = N - 1; y >= 0; y--)
#pragma unroll
        for (int x = N - 1 - y; x >= 0; x--) mma16816<typename Parts<T>::E>(x + y ? low : c, a[x], b0[y], b1[y]);
}

// Four warps.  FEW: all have the same 16 rows of the queries of all heads that share a key head (row
// r: head r / q_len, query r % q_len), and each a quarter of a tile's keys; otherwise 64 queries of
// one head, 16 to a warp.  A cluster's blocks share the keys out tile by tile; partial
// results are joined in shared memory.  Bound: matrix instructions (32 bits: six a product) and the
// softmax's arithmetic (400 x 400, 512 heads of 15: 148 us in 32 bits, 72 us in 16).
// TANH: capped scores by tanhf (32 bits, wide caps); chosen score by score, 16-bit tiles took 14 % longer (16 x 8
// heads of 15, 400 x 400: 47.5 us against 41.5).
template <typename T, int DP, bool FEW, bool EXTRA, bool TANH>
__global__ void __launch_bounds__(128) k_attn_tiles(const __grid_constant__ AttnP p, int vec) {
    using S = TileSmem<T, DP>;
    using E = typename Parts<T>::E;
    constexpr int P = S::P, BK = S::BK, LD = S::LD, KS = DP / 16;
    constexpr int WK = FEW ? BK / 4 : BK;  // keys of a warp in a tile
    constexpr int NT = WK / 8;
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ JoinSmem js;
    __shared__ int ends[64], seen;
    uint16_t *sq = (uint16_t *)dyn, *tiles = (uint16_t *)(dyn + S::q);
    cg::cluster_group cl = cg::this_cluster();
    const int cs = cl.num_blocks(), rank = cl.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = p.heads / p.kv_heads;
    const int hx = FEW ? p.kv_heads : p.heads;
    const int tile = blockIdx.y;
    const int b = blockIdx.x / cs / hx, hq = blockIdx.x / cs % hx;
    const int hk = FEW ? hq : hq / group;
    const Span sp = span_of(p, b);
    const int nrows = group * p.q_len;
    // head and query of a row of the block; -1 for rows past the last
    auto row_head = [&](int r) { return FEW ? hk * group + min(tile * 16 + r, nrows - 1) / p.q_len : hq; };
    auto row_query = [&](int r) {
        const int i = FEW ? (tile * 16 + r) % p.q_len : tile * 64 + r;
        return (!FEW || tile * 16 + r < nrows) && i < sp.nq ? i : -1;
    };
    if (threadIdx.x == 0) seen = 0;
    if (threadIdx.x < 64) js.odd[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x < (FEW ? 16 : 64)) {
        const int i = row_query(threadIdx.x);
        const int e = i >= 0 ? key_end(p, sp, i) : 0;
        ends[threadIdx.x] = e;
        atomicMax(&seen, e);
    }
    const T *kb = (const T *)p.k + b * p.ks[0] + hk * p.ks[1];
    const T *vb = (const T *)p.v + b * p.vs[0] + hk * p.vs[1];
    const int wr = FEW ? 0 : warp * 16;  // the warp's first row
    // this thread's two rows
    const int r0 = wr + (lane >> 2), r1 = r0 + 8;
    const int i0 = row_query(r0), i1 = row_query(r1);
    uint32_t qf[S::q_in_regs ? KS : 1][P][4];
    const T *q0 = (const T *)p.q + b * p.qs[0] + row_head(r0) * p.qs[1] + (int64_t)i0 * p.qs[2];
    const T *q1 = (const T *)p.q + b * p.qs[0] + row_head(r1) * p.qs[1] + (int64_t)i1 * p.qs[2];
    if constexpr (S::q_in_regs) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int d = ks * 16 + (x >> 1) * 8 + (lane & 3) * 2;
                const T *q = x & 1 ? q1 : q0;
                const bool in = (x & 1 ? i1 : i0) >= 0;
                uint32_t w[P];
                split2<T>(in && d < p.dim ? to_f(q[d]) : 0.f, in && d + 1 < p.dim ? to_f(q[d + 1]) : 0.f, w);
#pragma unroll
                for (int y = 0; y < P; y++) qf[ks][y][x] = w[y];
            }
    } else if constexpr (FEW) {
        for (int u = threadIdx.x; u < 16 * DP / 2; u += 128) {
            const int r = u / (DP / 2), d = u % (DP / 2) * 2, i = row_query(r);
            const T *q = (const T *)p.q + b * p.qs[0] + row_head(r) * p.qs[1] + (int64_t)i * p.qs[2];
            uint32_t w[P];
            split2<T>(i >= 0 && d < p.dim ? to_f(q[d]) : 0.f, i >= 0 && d + 1 < p.dim ? to_f(q[d + 1]) : 0.f, w);
#pragma unroll
            for (int y = 0; y < P; y++) *reinterpret_cast<uint32_t *>(sq + (y * 64 + r) * LD + d) = w[y];
        }
    } else {
        Units<T, DP, 64> u;
        u.fetch((const T *)p.q + b * p.qs[0] + hq * p.qs[1], p.qs[2], tile * 64, sp.nq, p.dim, vec);
        u.put(sq);
    }
    __syncthreads();
    const int last = seen;  // keys that any row sees
    const int e0 = ends[r0], e1 = ends[r1];
    int all;                // keys below it are seen by both rows of every thread of the warp
    {
        int e = min(i0 >= 0 ? e0 : 0x7fffffff, i1 >= 0 ? e1 : 0x7fffffff);
        all = __reduce_min_sync(0xffffffffu, e);
    }
    const float sl0 = EXTRA && p.slopes ? p.slopes[row_head(r0)] * kLog2e : 0.f;
    const float sl1 = EXTRA && p.slopes ? p.slopes[row_head(r1)] * kLog2e : 0.f;
    const int d0 = EXTRA && p.q_docs && i0 >= 0 ? p.q_docs[b * p.qds + i0] : 0, d1 = EXTRA && p.q_docs && i1 >= 0 ? p.q_docs[b * p.qds + i1] : 0;
    const int *kd = EXTRA && p.kv_docs ? p.kv_docs + b * p.kds : nullptr;
    const int pos0 = sp.off + i0, pos1 = sp.off + i1;
    const float scale2 = p.scale * kLog2e;
    float acc[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll
        for (int x = 0; x < 4; x++) acc[n][x] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const bool async = P == 1 && vec;
    // 32-bit tiles of up to 64 dimensions wait in registers while the tile before is in work
    constexpr bool AHEAD = P == 3 && DP <= 64;
    Units<T, DP, BK> nk, nv;
    auto copy = [&](int j, int stage) {
        if constexpr (P == 1) {
            copy_rows<T, DP, BK>(tiles + stage * S::kv, kb, p.ks[2], j, sp.nk, p.dim);  // (kv bytes: two stages' elements)
            copy_rows<T, DP, BK>(tiles + stage * S::kv + S::kv / 2, vb, p.vs[2], j, sp.nk, p.dim);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int stage = 0;
    if (async && rank * BK < last) copy(rank * BK, 0);
    else if (AHEAD && rank * BK < last) {
        nk.fetch(kb, p.ks[2], rank * BK, sp.nk, p.dim, vec);
        nv.fetch(vb, p.vs[2], rank * BK, sp.nk, p.dim, vec);
    }
    for (int j0 = rank * BK; j0 < last; j0 += cs * BK, stage ^= async) {
        uint16_t *sk = tiles + stage * S::kv, *sv = sk + S::kv / 2;
        if (async) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();  // this tile is there, and the one before has been read
            if (j0 + cs * BK < last) copy(j0 + cs * BK, stage ^ 1);
        } else {
            __syncthreads();  // the tile before has been read
            if (!AHEAD) nk.fetch(kb, p.ks[2], j0, sp.nk, p.dim, vec);
            nk.put(sk);
            if (!AHEAD) nv.fetch(vb, p.vs[2], j0, sp.nk, p.dim, vec);
            nv.put(sv);
            __syncthreads();
            if (AHEAD && j0 + cs * BK < last) {
                nk.fetch(kb, p.ks[2], j0 + cs * BK, sp.nk, p.dim, vec);
                nv.fetch(vb, p.vs[2], j0 + cs * BK, sp.nk, p.dim, vec);
            }
        }
        const int jw = j0 + (FEW ? warp * WK : 0), kw = FEW ? warp * WK : 0;
        float s[NT][4], low[P > 1 ? NT : 1][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < 4; x++) s[n][x] = low[P > 1 ? n : 0][x] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t a[P][4];
#pragma unroll
            for (int y = 0; y < P; y++) {
                if constexpr (S::q_in_regs) {
#pragma unroll
                    for (int x = 0; x < 4; x++) a[y][x] = qf[ks][y][x];
                } else {
                    ldsm4(a[y], sq + (y * 64 + wr + (lane & 15)) * LD + ks * 16 + (lane >> 4) * 8);
                }
            }
            // two n-tiles of 8 keys per load: keys (lane & 7) + 8 (lane >> 4), dims 8 ((lane >> 3) & 1)
            if constexpr (NT >= 2) {
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t bb[P][4], b0[P], b1[P];
#pragma unroll
                    for (int y = 0; y < P; y++)
                        ldsm4(bb[y], sk + (y * BK + kw + n * 8 + (lane & 7) + (lane >> 4) * 8) * LD + ks * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll
                    for (int y = 0; y < P; y++) b0[y] = bb[y][0], b1[y] = bb[y][1];
                    mma_parts<T, P>(s[n], low[P > 1 ? n : 0], a, b0, b1);
#pragma unroll
                    for (int y = 0; y < P; y++) b0[y] = bb[y][2], b1[y] = bb[y][3];
                    mma_parts<T, P>(s[n + 1], low[P > 1 ? n + 1 : 0], a, b0, b1);
                }
            } else {
                uint32_t b0[P], b1[P];
#pragma unroll
                for (int y = 0; y < P; y++) {
                    const uint16_t *at = sk + (y * BK + kw + (lane >> 2)) * LD + ks * 16 + (lane & 3) * 2;
                    b0[y] = *reinterpret_cast<const uint32_t *>(at);
                    b1[y] = *reinterpret_cast<const uint32_t *>(at + 8);
                }
                mma_parts<T, P>(s[0], low[0], a, b0, b1);
            }
        }
        // scores in units of log 2, masked
        const bool whole = jw + WK <= all && !kd;
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int j = jw + n * 8 + (lane & 3) * 2 + x;
                float u = s[n][x], w = s[n][2 + x];
                if constexpr (P > 1) {
                    u += low[n][x];
                    w += low[n][2 + x];
                }
                if (EXTRA && p.cap > 0.f) {
                    u = TANH ? capped32(u * p.scale, p.cap) : capped16(u * p.scale, p.cap);
                    w = TANH ? capped32(w * p.scale, p.cap) : capped16(w * p.scale, p.cap);
                } else {
                    u *= scale2;
                    w *= scale2;
                }
                if (EXTRA && p.slopes) {
                    u -= sl0 * fabsf((float)(pos0 - j));
                    w -= sl1 * fabsf((float)(pos1 - j));
                }
                if (!whole) {
                    bool in0 = j < e0, in1 = j < e1;
                    if (kd) {
                        const int doc = j < sp.nk ? kd[j] : -1;
                        in0 = in0 && doc == d0 && doc >= 0;
                        in1 = in1 && doc == d1 && doc >= 0;
                    }
                    if (!in0) u = -INFINITY;
                    if (!in1) w = -INFINITY;
                }
                s[n][x] = u;
                s[n][2 + x] = w;
                t0 = fmaxf(t0, u);
                t1 = fmaxf(t1, w);
            }
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        const float c0 = ex2(m0 - z0), c1 = ex2(m1 - z1);
        m0 = n0;
        m1 = n1;
        l0 *= c0;
        l1 *= c1;
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                s[n][x] = ex2(s[n][x] - z0);
                s[n][2 + x] = ex2(s[n][2 + x] - z1);
                l0 += s[n][x];
                l1 += s[n][2 + x];
            }
        }
        // the weights as the left operand, 16 keys at a time, rounded to the parts (16-bit types: once,
        // to the values' type, as the matrix instruction asks)
        constexpr int KN = (NT + 1) / 2;
        uint32_t a[KN][P][4];
#pragma unroll
        for (int n = 0; n < KN; n++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int nt = 2 * n + (x >> 1);
                uint32_t w[P];
                if (nt < NT) split2<T>(s[nt < NT ? nt : 0][(x & 1) * 2], s[nt < NT ? nt : 0][(x & 1) * 2 + 1], w);
#pragma unroll
                for (int y = 0; y < P; y++) a[n][y][x] = nt < NT ? w[y] : 0u;
            }
#pragma unroll
        for (int dn = 0; dn < DP / 16; dn++) {
            // 32 bits: a tile's sums on their own, added to the row's in ordinary (rounded) arithmetic
            float t[2][4], tl[2][4];
#pragma unroll
            for (int z = 0; z < 2; z++) {
                float (&o)[4] = acc[2 * dn + z];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    t[z][x] = P > 1 ? 0.f : o[x] * (x < 2 ? c0 : c1);
                    tl[z][x] = 0.f;
                }
            }
#pragma unroll
            for (int n = 0; n < KN; n++) {
                uint32_t bb[P][4], b0[P], b1[P];
                // keys (lane & 15), dims 8 (lane >> 4); with 8 keys only, the upper half repeats the lower
                const int key = kw + n * 16 + (NT == 1 ? lane & 7 : lane & 15);
#pragma unroll
                for (int y = 0; y < P; y++) ldsm4t(bb[y], sv + (y * BK + key) * LD + dn * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int y = 0; y < P; y++) b0[y] = bb[y][0], b1[y] = bb[y][1];
                mma_parts<T, P>(t[0], tl[0], a[n], b0, b1);
#pragma unroll
                for (int y = 0; y < P; y++) b0[y] = bb[y][2], b1[y] = bb[y][3];
                mma_parts<T, P>(t[1], tl[1], a[n], b0, b1);
            }
#pragma unroll
            for (int z = 0; z < 2; z++) {
                float (&o)[4] = acc[2 * dn + z];
#pragma unroll
                for (int x = 0; x < 4; x++) o[x] = P > 1 ? fmaf(o[x], x < 2 ? c0 : c1, t[z][x] + tl[z][x]) : t[z][x];
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (async) asm volatile("cp.async.wait_group 0;" ::: "memory");
    T *ob = (T *)p.o + b * p.os[0];
    if (!FEW && cs == 1) {
        const float v0 = l0 == 0.f ? 0.f : 1.f / l0, v1 = l1 == 0.f ? 0.f : 1.f / l1;
        bool bad0 = l0 == 0.f && may_see(p, sp, b, i0), bad1 = l1 == 0.f && may_see(p, sp, b, i1);
#pragma unroll
        for (int n = 0; n < DP / 8; n++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int d = n * 8 + (lane & 3) * 2 + x;
                const float u = acc[n][x] * v0, w = acc[n][2 + x] * v1;
                bad0 |= !finite(u);
                bad1 |= !finite(w);
                if (d < p.dim) {
                    if (i0 >= 0) ob[hq * p.os[1] + (int64_t)i0 * p.os[2] + d] = from_f<T>(u);
                    if (i1 >= 0) ob[hq * p.os[1] + (int64_t)i1 * p.os[2] + d] = from_f<T>(w);
                }
            }
        if (bad0) js.odd[r0] = 1;
        if (bad1) js.odd[r1] = 1;
        __syncwarp();
        Absent none;
        for (int r = wr + 15; r >= wr; r--)
            if (js.odd[r] && row_query(r) >= 0) none = row_again<T>(p, b, hq, row_query(r), none);
        return;
    }
    __syncthreads();  // the tiles have been read: their place holds the parts now
    PartSums<DP> *parts = (PartSums<DP> *)dyn;
    {
        PartSums<DP> &pt = parts[warp];
        const int a = lane >> 2;
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
            const int d = n * 8 + (lane & 3) * 2;
            *reinterpret_cast<float2 *>(&pt.o[a][d]) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(&pt.o[a + 8][d]) = make_float2(acc[n][2], acc[n][3]);
        }
        if ((lane & 3) == 0) {
            pt.m[a] = m0;
            pt.m[a + 8] = m1;
            pt.l[a] = l0;
            pt.l[a + 8] = l1;
        }
    }
    join_parts<T, DP, FEW ? 4 : 1>(p, b, parts, js, row_head, row_query);
}

// A few queries over 16-bit keys and values, straight from global memory into the matrix
// instructions' operands: a dot product may take the dimensions, and a weighted sum the keys, in any
// order that both sides share.  A thread's 16-byte load of key (lane / 4) holds its words of two
// left-hand steps (dimensions 8 (lane % 4) .. of a 32), and its loads of values at its own four
// weights' keys hold dimensions DP / 8 (lane / 4) .., paired by byte permutes.  No shared memory or
// barrier until the parts are joined; keys of the next 16 are loaded while the softmax of these runs.
// Bound: the keys' and values' bytes.  16 rows of the queries of all heads that share a key head.
template <typename T, int DP, bool EXTRA>
__global__ void __launch_bounds__(128) k_attn_token(const __grid_constant__ AttnP p) {
    constexpr int C = DP / 32, VW = DP / 64;  // 32-dimension chunks; 16-byte words of a value row per thread
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ JoinSmem js;
    PartSums<DP> *parts = (PartSums<DP> *)dyn;
    cg::cluster_group cl = cg::this_cluster();
    const int cs = cl.num_blocks(), rank = cl.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q4 = lane & 3;
    const int group = p.heads / p.kv_heads, nrows = group * p.q_len, tile = blockIdx.y;
    const int b = blockIdx.x / cs / p.kv_heads, hk = blockIdx.x / cs % p.kv_heads;
    const Span sp = span_of(p, b);
    auto row_head = [&](int r) { return hk * group + min(tile * 16 + r, nrows - 1) / p.q_len; };
    auto row_query = [&](int r) {
        const int i = (tile * 16 + r) % p.q_len;
        return tile * 16 + r < nrows && i < sp.nq ? i : -1;
    };
    const int i0 = row_query(g), i1 = row_query(g + 8);
    const int e0 = i0 >= 0 ? key_end(p, sp, i0) : 0, e1 = i1 >= 0 ? key_end(p, sp, i1) : 0;
    const int last = __reduce_max_sync(0xffffffffu, max(e0, e1));
    const int all = __reduce_min_sync(0xffffffffu, min(i0 >= 0 ? e0 : 0x7fffffff, i1 >= 0 ? e1 : 0x7fffffff));
    const uint4 none = make_uint4(0, 0, 0, 0);
    uint4 q0[C], q1[C];
    const T *qb = (const T *)p.q + b * p.qs[0];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = c * 32 + q4 * 8;
        q0[c] = i0 >= 0 && d < p.dim ? *(const uint4 *)(qb + row_head(g) * p.qs[1] + (int64_t)i0 * p.qs[2] + d) : none;
        q1[c] = i1 >= 0 && d < p.dim ? *(const uint4 *)(qb + row_head(g + 8) * p.qs[1] + (int64_t)i1 * p.qs[2] + d) : none;
    }
    const float sl0 = EXTRA && p.slopes ? p.slopes[row_head(g)] * kLog2e : 0.f, sl1 = EXTRA && p.slopes ? p.slopes[row_head(g + 8)] * kLog2e : 0.f;
    const int d0 = EXTRA && p.q_docs && i0 >= 0 ? p.q_docs[b * p.qds + i0] : 0, d1 = EXTRA && p.q_docs && i1 >= 0 ? p.q_docs[b * p.qds + i1] : 0;
    const int *kd = EXTRA && p.kv_docs ? p.kv_docs + b * p.kds : nullptr;
    const int pos0 = sp.off + i0, pos1 = sp.off + i1;
    const float scale2 = p.scale * kLog2e;
    const T *kb = (const T *)p.k + b * p.ks[0] + hk * p.ks[1] + q4 * 8;
    const T *vb = (const T *)p.v + b * p.vs[0] + hk * p.vs[1] + g * (DP / 8);
    uint4 kw[2][C], vw[4][VW];
    auto load_k = [&](int j0) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int j = j0 + t * 8 + g;
            const T *at = kb + (int64_t)j * p.ks[2];
#pragma unroll
            for (int c = 0; c < C; c++) kw[t][c] = j < last && c * 32 + q4 * 8 < p.dim ? __ldg((const uint4 *)(at + c * 32)) : none;
        }
    };
    auto load_v = [&](int j0) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int j = j0 + (t >> 1) * 8 + q4 * 2 + (t & 1);
            const T *at = vb + (int64_t)j * p.vs[2];
#pragma unroll
            for (int c = 0; c < VW; c++) vw[t][c] = j < last && g * (DP / 8) + c * 8 < p.dim ? __ldg((const uint4 *)(at + c * 8)) : none;
        }
    };
    float acc[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; n++)
#pragma unroll
        for (int x = 0; x < 4; x++) acc[n][x] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const int step = cs * 64;
    int j0 = (rank * 4 + warp) * 16;
    load_k(j0);
    load_v(j0);
    for (; j0 < last; j0 += step) {
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int x = 0; x < 4; x++) s[t][x] = 0.f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const uint32_t a0[4] = {q0[c].x, q1[c].x, q0[c].y, q1[c].y}, a1[4] = {q0[c].z, q1[c].z, q0[c].w, q1[c].w};
                mma16816<T>(s[t], a0, kw[t][c].x, kw[t][c].y);
                mma16816<T>(s[t], a1, kw[t][c].z, kw[t][c].w);
            }
        }
        load_k(j0 + step);
        const bool whole = j0 + 16 <= all && !kd;
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int j = j0 + t * 8 + q4 * 2 + x;
                float u = s[t][x], w = s[t][2 + x];
                if (EXTRA && p.cap > 0.f) {
                    u = capped2<T>(u * p.scale, p.cap);
                    w = capped2<T>(w * p.scale, p.cap);
                } else {
                    u *= scale2;
                    w *= scale2;
                }
                if (EXTRA && p.slopes) {
                    u -= sl0 * fabsf((float)(pos0 - j));
                    w -= sl1 * fabsf((float)(pos1 - j));
                }
                if (!whole) {
                    bool in0 = j < e0, in1 = j < e1;
                    if (kd) {
                        const int doc = j < sp.nk ? kd[j] : -1;
                        in0 = in0 && doc == d0 && doc >= 0;
                        in1 = in1 && doc == d1 && doc >= 0;
                    }
                    if (!in0) u = -INFINITY;
                    if (!in1) w = -INFINITY;
                }
                s[t][x] = u;
                s[t][2 + x] = w;
                t0 = fmaxf(t0, u);
                t1 = fmaxf(t1, w);
            }
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
        }
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        const float c0 = ex2(m0 - z0), c1 = ex2(m1 - z1);
        const bool grown = __any_sync(0xffffffffu, n0 > m0 || n1 > m1);
        m0 = n0;
        m1 = n1;
        l0 *= c0;
        l1 *= c1;
        uint32_t a[4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const float x0 = ex2(s[t][0] - z0), x1 = ex2(s[t][1] - z0), y0 = ex2(s[t][2] - z1), y1 = ex2(s[t][3] - z1);
            l0 += x0 + x1;
            l1 += y0 + y1;
            a[2 * t] = pack2<T>(x0, x1);  // rounded once, to the values' type
            a[2 * t + 1] = pack2<T>(y0, y1);
        }
        if (grown) {
#pragma unroll
            for (int n = 0; n < DP / 8; n++) {
                acc[n][0] *= c0;
                acc[n][1] *= c0;
                acc[n][2] *= c1;
                acc[n][3] *= c1;
            }
        }
#pragma unroll
        for (int n = 0; n < DP / 8; n += 2) {
            uint32_t w[4];  // dimensions n, n + 1 of the thread's four keys
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const uint4 &v = vw[t][n / 8];
                w[t] = (n & 7) == 0 ? v.x : (n & 7) == 2 ? v.y : (n & 7) == 4 ? v.z : v.w;
            }
            mma16816<T>(acc[n], a, __byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
            mma16816<T>(acc[n + 1], a, __byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
        }
        load_v(j0 + step);
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    PartSums<DP> &pt = parts[warp];
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int n = 0; n < DP / 8; n += 2) {
            const int d = (2 * q4 + x) * (DP / 8) + n;
            *reinterpret_cast<float2 *>(&pt.o[g][d]) = make_float2(acc[n][x], acc[n + 1][x]);
            *reinterpret_cast<float2 *>(&pt.o[g + 8][d]) = make_float2(acc[n][2 + x], acc[n + 1][2 + x]);
        }
    if (q4 == 0) {
        pt.m[g] = m0;
        pt.m[g + 8] = m1;
        pt.l[g] = l0;
        pt.l[g + 8] = l1;
    }
    join_parts<T, DP, 4>(p, b, parts, js, row_head, row_query);
}

// One query (32 bits: up to four), in 32-bit multiply-adds: eight lanes have a key, 16-byte words of it in turn, so
// a key's row is read in 128-byte pieces and its score takes three exchanges; a warp's four groups of
// lanes go over keys of their own, two at a time, with running maxima and sums of their own, joined at
// the end.  Bound: the keys' and values' bytes (32 x 8,192 keys, 8 key heads of 128, four rows: 6.0 TB/s
// in 32 bits).  R rows of the queries of all heads that share a key head.
template <typename T>
__device__ __forceinline__ void widen(const uint4 &w, float (&f)[16 / sizeof(T)]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(x[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        } else {
            f[2 * i] = __uint_as_float(x[i] << 16);
            f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
        }
    }
}
template <typename T, int DP, int R, bool EXTRA>
__global__ void __launch_bounds__(128) k_attn_row(const __grid_constant__ AttnP p) {
    constexpr int E = 16 / sizeof(T), W = DP / (8 * E), U = 2;  // elements of a word; words of a key per lane; keys under way
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ JoinSmem js;
    PartSums<DP> *parts = (PartSums<DP> *)dyn;
    cg::cluster_group cl = cg::this_cluster();
    const int cs = cl.num_blocks(), rank = cl.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 3, e = lane & 7;
    const int group = p.heads / p.kv_heads, nrows = group * p.q_len, tile = blockIdx.y;
    const int b = blockIdx.x / cs / p.kv_heads, hk = blockIdx.x / cs % p.kv_heads;
    const Span sp = span_of(p, b);
    auto row_head = [&](int r) { return hk * group + min(tile * R + r, nrows - 1) / p.q_len; };
    auto row_query = [&](int r) {
        const int i = (tile * R + r) % p.q_len;
        return r < R && tile * R + r < nrows && i < sp.nq ? i : -1;
    };
    const uint4 none = make_uint4(0, 0, 0, 0);
    float q[R][W][E], o[R][W][E], m[R], l[R], slope[R];
    int end[R], pos[R], doc[R], last = 0;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = row_query(r), h = row_head(r);
        const T *qr = (const T *)p.q + b * p.qs[0] + h * p.qs[1] + (int64_t)i * p.qs[2];
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int d = (w * 8 + e) * E;
            widen<T>(i >= 0 && d < p.dim ? *(const uint4 *)(qr + d) : none, q[r][w]);
#pragma unroll
            for (int x = 0; x < E; x++) o[r][w][x] = 0.f;
        }
        m[r] = -INFINITY;
        l[r] = 0.f;
        end[r] = i >= 0 ? key_end(p, sp, i) : 0;
        pos[r] = sp.off + i;
        last = max(last, end[r]);
        slope[r] = EXTRA && p.slopes ? p.slopes[h] : 0.f;
        doc[r] = EXTRA && p.q_docs && i >= 0 ? p.q_docs[b * p.qds + i] : 0;
    }
    const T *kb = (const T *)p.k + b * p.ks[0] + hk * p.ks[1] + e * E;
    const T *vb = (const T *)p.v + b * p.vs[0] + hk * p.vs[1] + e * E;
    const int *kd = EXTRA && p.kv_docs ? p.kv_docs + b * p.kds : nullptr;
    const float scale2 = p.scale * kLog2e;
    uint4 kw[U][W], vw[U][W];
    auto load = [&](uint4(&x)[U][W], const T *base, int64_t stride, int j0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = j0 + u * 4;
#pragma unroll
            for (int w = 0; w < W; w++)
                x[u][w] = j < last && (w * 8 + e) * E < p.dim ? __ldg((const uint4 *)(base + j * stride + w * 8 * E)) : none;
        }
    };
    const int step = cs * 16 * U;
    int j0 = (rank * 4 + warp) * 4 * U + g;
    load(kw, kb, p.ks[2], j0);
    load(vw, vb, p.vs[2], j0);
    for (int base = (rank * 4 + warp) * 4 * U; base < last; base += step, j0 += step) {
        float s[U][R];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int r = 0; r < R; r++) s[u][r] = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                float f[E];
                widen<T>(kw[u][w], f);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int x = 0; x < E; x++) s[u][r] = fmaf(q[r][w][x], f[x], s[u][r]);
            }
        }
        load(kw, kb, p.ks[2], j0 + step);
#pragma unroll
        for (int d = 1; d < 8; d *= 2)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < R; r++) s[u][r] += __shfl_xor_sync(0xffffffffu, s[u][r], d);
        float c[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int j = j0 + u * 4;
                const float x = EXTRA ? score2<T>(p, s[u][r], slope[r], pos[r] - j) : s[u][r] * scale2;
                bool in = j < end[r];
                if (kd) {
                    const int d = j < sp.nk ? kd[j] : -1;
                    in = in && d == doc[r] && d >= 0;
                }
                s[u][r] = in ? x : -INFINITY;
                top = fmaxf(top, s[u][r]);
            }
            const float z = top == -INFINITY ? 0.f : top;
            c[r] = ex2(m[r] - z);
            m[r] = top;
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                s[u][r] = ex2(s[u][r] - z);
                sum += s[u][r];
            }
            l[r] = fmaf(l[r], c[r], sum);
        }
#pragma unroll
        for (int w = 0; w < W; w++) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int x = 0; x < E; x++) o[r][w][x] *= c[r];
#pragma unroll
            for (int u = 0; u < U; u++) {
                float f[E];
                widen<T>(vw[u][w], f);
#pragma unroll
                for (int r = 0; r < R; r++)
#pragma unroll
                    for (int x = 0; x < E; x++) o[r][w][x] = fmaf(s[u][r], f[x], o[r][w][x]);
            }
        }
        load(vw, vb, p.vs[2], j0 + step);
    }
    PartSums<DP> &pt = parts[warp];
#pragma unroll
    for (int r = 0; r < R; r++) {
        float top = m[r];
#pragma unroll
        for (int d = 8; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float z = top == -INFINITY ? 0.f : top, f = ex2(m[r] - z);
        float sum = l[r] * f;
#pragma unroll
        for (int d = 8; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int x = 0; x < E; x++) {
                float a = o[r][w][x] * f;
#pragma unroll
                for (int d = 8; d < 32; d *= 2) a += __shfl_xor_sync(0xffffffffu, a, d);
                if (g == 0) pt.o[r][(w * 8 + e) * E + x] = a;
            }
        if (lane == 0) {
            pt.m[r] = top;
            pt.l[r] = sum;
        }
    }
    join_parts<T, DP, 4>(p, b, parts, js, row_head, row_query);
}

dim3 grid_of(int64_t units, int cs, int64_t tiles) {
    if (units * cs > 0x7fffffff || tiles > 65535) fail(WOCR_ERR_UNSUPPORTED, "attention: too many heads or queries");
    return dim3((unsigned)(units * cs), (unsigned)tiles);
}

template <typename T, int DP, bool FEW>
void launch_tiles(Ctx *c, const AttnP &p, int vec, cudaStream_t s) {
    using S = TileSmem<T, DP>;
    const int64_t units = (int64_t)p.batch * (FEW ? p.kv_heads : p.heads);
    const int tiles = FEW ? (p.heads / p.kv_heads * p.q_len + 15) / 16 : (p.q_len + 63) / 64;
    constexpr bool is32 = Parts<T>::n == 3;
    auto kernel = extra_scores(p) ? (by_tanh<T>(p.cap) && p.cap > 0.f ? k_attn_tiles<T, DP, FEW, true, true> : k_attn_tiles<T, DP, FEW, true, is32>)
                                  : k_attn_tiles<T, DP, FEW, false, is32>;
    static const int per_sm = resident(k_attn_tiles<T, DP, FEW, false, is32>, 128, S::bytes);
    const int cs = key_split(c, units * tiles, per_sm, p.kv_len, S::BK);
    launch_cluster<AttnP, int>(kernel, grid_of(units, cs, tiles), 128, cs, S::bytes, s, p, vec);
    WOCR_LAUNCHED(c);
}

template <typename T, int DP>
void launch_token(Ctx *c, const AttnP &p, cudaStream_t s) {
    const int64_t units = (int64_t)p.batch * p.kv_heads;
    const int tiles = (p.heads / p.kv_heads * p.q_len + 15) / 16;
    static const int per_sm = resident(k_attn_token<T, DP, false>, 128, 4 * sizeof(PartSums<DP>));
    const int cs = key_split(c, units * tiles, per_sm, p.kv_len, 64);
    auto kernel = extra_scores(p) ? k_attn_token<T, DP, true> : k_attn_token<T, DP, false>;
    launch_cluster<AttnP>(kernel, grid_of(units, cs, tiles), 128, cs, 4 * sizeof(PartSums<DP>), s, p);
    WOCR_LAUNCHED(c);
}

template <typename T, int DP, int R>
void launch_row(Ctx *c, const AttnP &p, cudaStream_t s) {
    const int64_t units = (int64_t)p.batch * p.kv_heads;
    const int tiles = (p.heads / p.kv_heads * p.q_len + R - 1) / R;
    static const int per_sm = resident(k_attn_row<T, DP, R, false>, 128, 4 * sizeof(PartSums<DP>));
    const int cs = key_split(c, units * tiles, per_sm, p.kv_len, 32);
    auto kernel = extra_scores(p) ? k_attn_row<T, DP, R, true> : k_attn_row<T, DP, R, false>;
    launch_cluster<AttnP>(kernel, grid_of(units, cs, tiles), 128, cs, 4 * sizeof(PartSums<DP>), s, p);
    WOCR_LAUNCHED(c);
}
// 32-bit rows four at a time, although the cache is then read once for each four: 16 rows over 8 caches of 8,192
// keys of 128, 39 us against 65 in tiles that share it; 64 rows, 125 against 128.
template <typename T, int DP>
void launch_row(Ctx *c, const AttnP &p, cudaStream_t s) {
    const int rows = p.heads / p.kv_heads * p.q_len;
    if constexpr (Parts<T>::n == 3) {
        if (rows == 2) return launch_row<T, DP, 2>(c, p, s);
        if (rows > 2) return launch_row<T, DP, 4>(c, p, s);
    }
    launch_row<T, DP, 1>(c, p, s);
}

// The queries of the heads that share a key head are taken together: a few tokens of a decoder.  (8 caches of
// 8,192 keys of 128, 64 heads over one key head: 37 us in 16 bits and 125 us in 32, against 661 and 3,362 us head by
// head.  Beyond the limit it is head by head still: 128 heads 1,197 and 6,654 us, where together they would
// take 58 and 240 us.)
bool few_rows(const AttnP &p) { return p.q_len <= 16 && (int64_t)p.heads / p.kv_heads * p.q_len <= 64; }

template <typename T, int DP>
void launch_dim(Ctx *c, const AttnP &p, int vec, cudaStream_t s) {
    if (few_rows(p)) launch_tiles<T, DP, true>(c, p, vec, s);
    else launch_tiles<T, DP, false>(c, p, vec, s);
}

template <typename T>
void launch_type(Ctx *c, const AttnP &p, cudaStream_t s) {
    // 16-byte loads where every row of queries, keys and values allows them
    const int n = 16 / sizeof(T);
    bool vec = ((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0;
    for (int i = 0; i < 3; i++) vec = vec && p.qs[i] % n == 0 && p.ks[i] % n == 0 && p.vs[i] % n == 0;
    if constexpr (Parts<T>::n == 1)
        // (16 x 4,096 keys, 8 key heads of 128: two rows 62 us in this one, 77 in the row's; 32 x 8,192: one row
        // 208 us in this one, 164 in the row's)
        if (few_rows(p) && p.heads / p.kv_heads * p.q_len > 1 && vec && p.dim % 8 == 0 && p.dim <= 128)
            return p.dim <= 64 ? launch_token<T, 64>(c, p, s) : launch_token<T, 128>(c, p, s);
    if (few_rows(p) && vec && p.dim % n == 0 && p.dim <= 128) {
        if constexpr (Parts<T>::n == 3)
            if (p.dim <= 32) return launch_row<T, 32>(c, p, s);
        return p.dim <= 64 ? launch_row<T, 64>(c, p, s) : launch_row<T, 128>(c, p, s);
    }
    if (p.dim <= 16) launch_dim<T, 16>(c, p, vec, s);
    else if (p.dim <= 32) launch_dim<T, 32>(c, p, vec, s);
    else if (p.dim <= 64) launch_dim<T, 64>(c, p, vec, s);
    else if (p.dim <= 128) launch_dim<T, 128>(c, p, vec, s);
    else launch_dim<T, 256>(c, p, vec, s);
}
}  // namespace

void attention(Ctx *c, const AttnP &p, cudaStream_t s) {
    const double rows = (double)p.batch * p.heads * p.q_len;
    OpProf pf(c, s, "attention", 4.0 * rows * p.kv_len * p.dim,
              elem_size(p.type) * (double)p.dim * (2.0 * rows + 2.0 * p.batch * p.kv_heads * p.kv_len));
    // Tiles of 128 queries on tcgen05 once they are half full, or the keys are many: 64 queries over 64
    // keys, 128 x 8 heads of 64: 25 us against 33, 40 over 40: 37 both; 20 over 4,096, 16 x 16 heads of
    // 128: 113 us against 617.
    if (p.q_len > 16 && (p.q_len >= 64 || p.kv_len >= 512) && attention_tc_ok(p)) return attention_tc(c, p, s);
    if (p.type == WOCR_F32) launch_type<float>(c, p, s);
    else if (p.type == WOCR_F16) launch_type<__half>(c, p, s);
    else launch_type<__nv_bfloat16>(c, p, s);
}

}  // namespace k
}  // namespace wocr
