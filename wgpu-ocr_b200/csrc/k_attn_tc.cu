// Attention of many queries over 16-bit keys and values on the tensor cores: tcgen05 with scores,
// weights and sums in tensor memory, tiles fed by TMA.
//
// A block takes NT tiles of 128 queries of one head (one tensor-memory lane each) and walks the keys in
// tiles of 128: two tiles, or, for short sequences of heads of up to 64 dimensions, one, with two
// blocks on an SM, which hide each other's start and end as well.  Roles (of two tiles):
//   warps 0-3, 4-7  softmax of query tile 0 and 1, a thread per row: scores from tensor memory, mask,
//                   running maximum and sum, weights back into tensor memory as the left operand of
//                   the second product, in the columns of the scores they came from
//   warp 8          (one thread) issues S = Q K^T and O += P V.  While one tile's softmax runs, the
//                   other tile's products do, so the matrix pipe and the exponentials overlap
//   warp 9          (one thread) TMA loads of queries, keys and values, two stages each
//   warps 10, 11    help to look at documents before the loop
// Where there are fewer blocks than SMs, a cluster's blocks share a query tile's keys out, tile by
// tile, and join their sums through distributed shared memory.
// A row's sums are rescaled only when its maximum has grown by more than 2^8 since it was last used
// (the weights stay below 2^8, the quotient is the same), so the accumulator is seldom touched
// between products.
// Measured: 32 heads of 128, 8,192 queries and keys, causal, bf16: 445 us on the same tensors call after
// call (1.24 PFLOP/s), 518 us on others each time (1.06 PFLOP/s, 64 % of the measured matrix peak; the power
// cap); not causal, 16 heads of 4,096: 122 to 140 us, 1.0 to 1.1 PFLOP/s; of 64: 123 us.
// Bound: 4 D flops and one exponential a pair.  An SM's matrix pipe takes 128 x 128 x 128 in 512
// cycles and its 16 exponentials a cycle take as long for two such products (D = 128).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "attn.h"
#include "attn_tc.h"
#include "tc.h"

namespace wocr {
namespace k {

namespace {
using namespace attn;
using namespace tc;

// registers: softmax warps hold a row's 128 scores; 256 x 192 + 128 x 120 = 384 x 168, what the block has
// (224 and 56 left the issuing warp 15 % of the kernel's time in spills)
constexpr int kSoftmaxRegs = 192, kIssueRegs = 120;
constexpr int kMaxTiles = 8192;              // key tiles of a call (2^20 keys): their bits fit in shared memory
constexpr int kWords = kMaxTiles / 32;
constexpr float kSlack = 8.f;                // growth of a maximum (log 2) that leaves the sums alone

template <int DP, int NT>
struct Smem {
    static constexpr int tile = 128 * DP * 2;
    // values first: a stage ends inside the block's shared memory whatever follows it
    static constexpr int v = 0, k = v + 2 * tile, q = k + 2 * tile, bits = q + NT * tile, docs = bits + 2 * NT * kWords * 4,
                         bars = docs + 4 * NT * 128 * 4, bytes = bars + 256 + 1024;  // 1,024: alignment of the start
};

struct TcArgs {
    AttnP a;
    int *status;
    long long budget;
    int tiles, vec_out;  // blocks of a head; rows of out take 16-byte stores
};

// kind::f16, D fp32, M = 128; B is K-major (scores) or N-major (values: dimensions contiguous)
__host__ __device__ constexpr uint32_t idesc(bool bf16, int n, bool b_n_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_n_major ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// N-major operand in the 128-byte swizzle: rows (keys) of 64 dimensions, eight rows an atom of
// 1,024 bytes (the stride between groups of eight keys); the next 64 dimensions a panel further.
__device__ __forceinline__ uint64_t desc_n_major(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, float *f) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
#pragma unroll
    for (int i = 0; i < 32; i++) f[i] = __uint_as_float(r[i]);
}
// waits for the thread's tensor-memory loads; the values pass through, so that no use moves ahead
__device__ __forceinline__ void tmem_wait32(float *f) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]),
                   "+f"(f[8]), "+f"(f[9]), "+f"(f[10]), "+f"(f[11]), "+f"(f[12]), "+f"(f[13]), "+f"(f[14]), "+f"(f[15]),
                   "+f"(f[16]), "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]), "+f"(f[23]),
                   "+f"(f[24]), "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29]), "+f"(f[30]), "+f"(f[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const float *f) {
    uint32_t r[16];
#pragma unroll
    for (int y = 0; y < 2; y++) {
#pragma unroll
        for (int x = 0; x < 16; x++) r[x] = __float_as_uint(f[y * 16 + x]);
        tmem_st16(at + y * 16, r);
    }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// the greatest of 32 values and t, in four chains
__device__ __forceinline__ float max32(const float *f, float t) {
    float a[4] = {t, f[0], f[1], f[2]};
#pragma unroll
    for (int x = 3; x + 1 < 32; x += 2) a[(x >> 1) & 3] = max3(a[(x >> 1) & 3], f[x], f[x + 1]);
    return fmaxf(max3(a[0], a[1], a[2]), fmaxf(a[3], f[31]));
}
__device__ constexpr float kTanh[6] = {1.f, -0.333332121f, 0.133305937f, -0.0536993034f, 0.0205612238f, -0.00565812876f};
// cap tanh(scale f / cap) in units of log 2.  |y| < 0.6, the rule for capped scores, takes y times a
// polynomial in y^2 (least squares in Chebyshev points, within 2^-24 of tanh); a warp with a larger
// one takes the exponential and the quotient.
template <typename T>
__device__ __forceinline__ void cap32(float *f, float scale, float cap) {
    const float to_y = scale / cap, to_s = scale * kLog2e;
    float a = 0.f;
#pragma unroll
    for (int x = 0; x < 32; x += 2) a = max3(a, fabsf(f[x]), fabsf(f[x + 1]));
    if (__any_sync(0xffffffffu, !(a * fabsf(to_y) < 0.6f))) {
#pragma unroll
        for (int x = 0; x < 32; x++) f[x] = capped2<T>(f[x] * scale, cap);
        return;
    }
    const float2 yy = make_float2(to_y, to_y), ss = make_float2(to_s, to_s);
#pragma unroll
    for (int x = 0; x < 32; x += 2) {
        const float2 v = make_float2(f[x], f[x + 1]), y = __fmul2_rn(v, yy), t = __fmul2_rn(y, y);
        float2 r = make_float2(kTanh[5], kTanh[5]);
#pragma unroll
        for (int k = 4; k >= 0; k--) r = __ffma2_rn(r, t, make_float2(kTanh[k], kTanh[k]));
        r = __fmul2_rn(r, __fmul2_rn(v, ss));
        f[x] = r.x;
        f[x + 1] = r.y;
    }
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// the value of lane 0, known to be the same in every lane
__device__ __forceinline__ int same(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ uint32_t same(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool elect() {  // one lane of the warp, always the same
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// EXTRA: scores that are more than a plain product (capped, biased by distance, a scale that is not
// positive), or documents.  Apart, since their code, unrolled over a row, cost plain tiles 15 % in
// the instruction caches.  SPLIT: a cluster shares the keys out (its code costs the others 7 %).
constexpr int threads_of(int nt) { return nt == 2 ? 384 : 192; }

template <typename T, int DP, int NT, bool EXTRA, bool SPLIT>
__global__ void __launch_bounds__(threads_of(NT), 3 - NT)
    k_attn_tc(const __grid_constant__ TcArgs ta, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
              const __grid_constant__ CUtensorMap mv) {
    using L = Smem<DP, NT>;
    constexpr int kThreads = threads_of(NT), kMmaWarp = 4 * NT, kTmaWarp = kMmaWarp + 1;  // (NT 2: two more fill the warpgroup)
    constexpr uint32_t kColS = 0, kColO = NT * 128, kCols = NT * 256;  // tensor-memory columns: scores, sums
    constexpr int kPanels = DP / 64, kPanel = 128 * 128;  // 64 dimensions of 128 rows
    extern __shared__ uint8_t raw[];
    uint8_t *sm = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const AttnP &p = ta.a;
    uint32_t *act = (uint32_t *)(sm + L::bits), *full = act + NT * kWords;  // per query tile: key tiles to visit, without masks
    int *docs = (int *)(sm + L::docs);
    uint64_t *bars = (uint64_t *)(sm + L::bars);
    uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7,
             *s_full = bars + 9, *o_full = bars + 11, *tail = bars + 13, *p_half = bars + 14, *p_full = bars + 16;
    uint32_t *slot = (uint32_t *)(bars + 18);
    volatile int *stop = (volatile int *)(slot + 1);
    int *lim = (int *)(slot + 2);  // [4] least and greatest document of the two query tiles
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // long rows first: with a causal mask the last queries see the most keys
    const int heads = p.heads * p.batch;
    cg::cluster_group cl = cg::this_cluster();
    const int cs = SPLIT ? cl.num_blocks() : 1, rank = SPLIT ? cl.block_rank() : 0, unit = blockIdx.x / cs;
    const int tile = ta.tiles - 1 - unit / heads, bh = unit % heads;
    const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kv_heads);
    const Span sp = span_of(p, b);
    const int i_first = tile * 128 * NT;
    if (i_first >= sp.nq) return;
    // keys that the first and the last row of each query tile may see
    int emin[2] = {0, 0}, emax[2] = {0, 0};
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int a = i_first + t * 128, z = min(a + 127, sp.nq - 1);
        emin[t] = a < sp.nq ? max(key_end(p, sp, a), 0) : 0;
        emax[t] = a < sp.nq ? max(key_end(p, sp, z), 0) : 0;
    }
    const int ntiles = (max(emax[0], emax[1]) + 127) / 128;
    if (tid == 0) {
        for (int i = 0; i < 18; i++) mbar_init(bars + i, i < 14 ? 1 : 4);  // weights: four warps
        *stop = 0;
        for (int i = 0; i < 4; i++) lim[i] = i & 1 ? -1 : 0x7fffffff;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    const int my = warp >> 2;  // softmax: the thread's query tile and row
    const int i = i_first + my * 128 + (tid & 127);
    const bool row = warp < kMmaWarp && i < sp.nq;
    int doc = -1;
    const bool by_doc = EXTRA && p.q_docs != nullptr;
    if (by_doc) {
        for (int w = tid; w < 2 * NT * kWords; w += kThreads) act[w] = 0;
        __syncthreads();
        if (row) doc = p.q_docs[b * p.qds + i];
        if (warp < kMmaWarp) {
            // -1: a row that sees nothing, no tile goes without its mask
            const int lo = __reduce_min_sync(0xffffffffu, row ? max(doc, -1) : 0x7fffffff), hi = __reduce_max_sync(0xffffffffu, doc);
            if (lane == 0) {
                atomicMin(&lim[2 * my], lo);
                atomicMax(&lim[2 * my + 1], hi);
            }
        }
        __syncthreads();
        // a key tile's documents against the query tiles': none shared, all the same, or some; four key
        // tiles of a warp at a time, their loads under way together
        const int *ids = p.kv_docs + b * p.kds;
        for (int j0 = warp * 4; j0 < ntiles; j0 += kThreads / 32 * 4) {
            int d[4][4];
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int key = (j0 + y) * 128 + x * 32 + lane;
                    d[y][x] = key < sp.nk ? ids[key] : -1;
                }
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int j = j0 + y;
                int lo = 0x7fffffff, hi = -1;
                bool odd = false;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    odd |= d[y][x] < 0;
                    if (d[y][x] >= 0) lo = min(lo, d[y][x]);
                    hi = max(hi, d[y][x]);
                }
                lo = __reduce_min_sync(0xffffffffu, lo);
                hi = __reduce_max_sync(0xffffffffu, hi);
                odd = __any_sync(0xffffffffu, odd);
                if (lane < NT && j < ntiles) {
                    const int t = lane, ql = max(lim[2 * t], 0), qh = lim[2 * t + 1];
                    if (j * 128 < (t ? emax[1] : emax[0]) && lo <= qh && hi >= ql) atomicOr(&act[t * kWords + j / 32], 1u << (j & 31));
                    if (!odd && lo == hi && lim[2 * t] == lo && qh == lo && (j + 1) * 128 <= (t ? emin[1] : emin[0]))
                        atomicOr(&full[t * kWords + j / 32], 1u << (j & 31));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const int whole = my == 0 ? emin[0] : emin[1], reach = my == 0 ? emax[0] : emax[1];  // of the thread's query tile
    auto visits = [&](int t, int e, int j) -> bool { return by_doc ? (act[t * kWords + j / 32] >> (j & 31)) & 1 : j * 128 < e; };

    // the next key tile from j on that is this block's and is visited by the query tiles of `tiles` (bits), which reach to key e
    auto next = [&](int tiles, int e, int j) -> int {
        if constexpr (EXTRA)
            if (by_doc) {
                for (; j < ntiles; j = (j | 31) + 1) {
                    const uint32_t mine = cs == 8 ? 0x01010101u : cs == 4 ? 0x11111111u : cs == 2 ? 0x55555555u : ~0u;
                    const uint32_t w = (((tiles & 1 ? act[j / 32] : 0) | (NT == 2 && tiles & 2 ? act[kWords + j / 32] : 0)) & mine << rank) >> (j & 31);
                    if (w) return j + __ffs(w) - 1;
                }
                return ntiles;
            }
        if (SPLIT) j += (rank - j) & (cs - 1);
        return j * 128 < e ? j : ntiles;
    };
    const int ends = max(emax[0], emax[1]);
    float row_m = -INFINITY, row_l = 0.f;  // a softmax thread's row
    bool got = false;

    if (warp >= kMmaWarp) {
        // (a warpgroup changes its registers as one)
        if constexpr (NT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == kTmaWarp) {
            const uint32_t qbytes = 128 * DP * 2;
            bool any = false;
            int it = 0;
            bool ok = true;
            for (int j = next(3, ends, 0); j < ntiles && ok; j = next(3, ends, j + 1)) {
                const int s = it & 1;
                const uint32_t par = (it >> 1) & 1;
                uint8_t *sk = sm + L::k + s * L::tile, *sv = sm + L::v + s * L::tile;
                // values behind the last key must be finite: they are multiplied by weights of zero
                const bool edge = sp.nk < (j + 1) * 128 && sp.nk < p.kv_len;
                if (lane == 0) {
                    if (!any) {
                        mbar_expect_tx(q_full, NT * qbytes);
                        for (int t = 0; t < NT; t++)
                            for (int x = 0; x < kPanels; x++)
                                tma_load_4d(sm + L::q + t * L::tile + x * kPanel, &mq, q_full, x * 64, i_first + t * 128, h, b);
                        any = true;
                    }
                    ok = mbar_wait_spin(&k_empty[s], par ^ 1, ta.status, stop, 41, ta.budget);
                    if (ok) {
                        mbar_expect_tx(&k_full[s], qbytes);
                        for (int x = 0; x < kPanels; x++) tma_load_4d(sk + x * kPanel, &mk, &k_full[s], x * 64, j * 128, hk, b);
                        ok = mbar_wait_spin(&v_empty[s], par ^ 1, ta.status, stop, 42, ta.budget);
                    }
                    if (ok) {
                        uint64_t *bar = edge ? tail : &v_full[s];
                        mbar_expect_tx(bar, qbytes);
                        for (int x = 0; x < kPanels; x++) tma_load_4d(sv + x * kPanel, &mv, bar, x * 64, j * 128, hk, b);
                        if (edge) ok = mbar_wait_spin(tail, 0, ta.status, stop, 43, ta.budget);  // the last tile: once
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                __syncwarp();
                if (edge && ok) {
                    const int from = sp.nk - j * 128;  // a row is 128 bytes of each panel, wherever the swizzle puts its pieces
                    for (int u = lane; u < (128 - from) * 8 * kPanels; u += 32) {
                        const int x = u / ((128 - from) * 8), v = u % ((128 - from) * 8);
                        *(uint4 *)(sv + x * kPanel + (from + v / 8) * 128 + (v % 8) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[s]);
                }
                it++;
            }
            if (lane == 0) {
                // copies land before the block may exit, however it ends (bounded)
                const long long t0 = clock64();
                if (it > 0)
                    while (!mbar_try(q_full, 0) && clock64() - t0 < ta.budget) {
                    }
                for (int j = it > 2 ? it - 2 : 0; j < it; j++)
                    for (uint64_t *bar : {&k_full[j & 1], &v_full[j & 1]})
                        while (!mbar_try(bar, (j >> 1) & 1) && clock64() - t0 < ta.budget && !*stop) {
                        }
                if (*stop) {  // given up: some loads may never have been asked for, others are on their way
                    const long long t1 = clock64();
                    while (clock64() - t1 < 2000000) {
                    }
                }
            }
            __syncwarp();
        } else if (warp == kMmaWarp) {
            // The whole warp walks the loop, on values that are the same in every lane, and one lane
            // issues: an instruction's descriptors are uniform registers, and from one lane's own ones
            // they took 75 to 100 cycles an instruction to move there.
            constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
            const int ksteps = (p.dim + 15) / 16;
            const uint32_t id_s = idesc(bf, 128, false), id_o = idesc(bf, ksteps * 16, true), tm = same(tmem);
            const uint64_t dq = smem_desc(same(smem_u32(sm + L::q))), dk = smem_desc(same(smem_u32(sm + L::k))),
                           dv = desc_n_major(same(smem_u32(sm + L::v)), kPanel);
            const int e0 = same(emax[0]), e1 = same(emax[1]), eb = max(e0, e1), nt = (eb + 127) / 128;
            constexpr int kUnits = L::tile / 16;  // descriptors count 16 bytes
            bool ok = true;
            int pend[2] = {-1, -1};  // number of the key tile whose values a tile's weights wait for
            int np[2] = {0, 0};      // weights consumed
            int it = 0;
            auto wait = [&](uint64_t *bar, int parity, int code) -> bool {
                return __all_sync(0xffffffffu, mbar_wait_spin(bar, parity & 1, ta.status, stop, code, ta.budget));
            };
            auto product = [&](int t) {  // O_t += P_t V
                if (pend[t] < 0) return;
                const int s = pend[t] & 1;
                const uint64_t v = dv + s * kUnits;
                const uint32_t weights = tm + kColS + t * 128, sums = tm + kColO + t * 128, more = np[t] > 0;
                ok = ok && wait(&v_full[s], pend[t] >> 1, 45) && wait(&p_half[t], np[t], 44);
                if (!ok) return;
                tc_fence_after();
                if (elect()) {
                    umma_ts(sums, weights, v, id_o, more);
#pragma unroll
                    for (int x = 1; x < 4; x++) umma_ts(sums, weights + x * 8, v + x * (2048 / 16), id_o, 1);
                }
                __syncwarp();
                ok = wait(&p_full[t], np[t], 44);
                if (!ok) return;
                tc_fence_after();
                if (elect()) {
#pragma unroll
                    for (int x = 4; x < 8; x++) umma_ts(sums, weights + x * 8, v + x * (2048 / 16), id_o, 1);
                }
                __syncwarp();
                pend[t] = -1;
                np[t]++;
            };
            for (int j = same(next(3, eb, 0)); j < nt && ok; j = same(next(3, eb, j + 1)), it++) {
                const bool v0 = same((int)visits(0, e0, j)), v1 = same((int)visits(1, e1, j));
                const int s = it & 1;
                if (it == 0) ok = wait(q_full, 0, 46);
                ok = ok && wait(&k_full[s], it >> 1, 47);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    product(t);
                    if (!ok) break;
                    if (!(t ? v1 : v0)) continue;
                    const uint64_t q = dq + t * kUnits, k = dk + s * kUnits;
                    const uint32_t scores = tm + kColS + t * 128;
                    if (elect()) {
                        umma(scores, q, k, id_s, 0);
#pragma unroll
                        for (int x = 1; x < DP / 16; x++) {
                            const int off = ((x >> 2) * kPanel + (x & 3) * 32) / 16;
                            if (x < ksteps) umma(scores, q + off, k + off, id_s, 1);
                        }
                        umma_commit(&s_full[t]);
                    }
                    __syncwarp();
                    pend[t] = it;
                }
                if (!ok) break;
                if (elect()) {
                    umma_commit(&k_empty[s]);
                    if (it > 0) umma_commit(&v_empty[s ^ 1]);
                }
                __syncwarp();
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                product(t);
                if (elect()) umma_commit(&o_full[t]);
                __syncwarp();
            }
            const long long t0 = clock64();
            for (int t = 0; t < NT; t++)
                while (!mbar_try(&o_full[t], 0) && clock64() - t0 < ta.budget) {
                }
            __syncwarp();
        }
    } else {
        if constexpr (NT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 tensor-memory lanes
        const uint32_t ts = tmem + lanes + kColS + my * 128, to = tmem + lanes + kColO + my * 128;
        const bool live = row && (!by_doc || doc >= 0);
        const int end = live ? key_end(p, sp, i) : 0, pos = sp.off + i;
        if (doc < 0) doc = INT_MIN;  // sees nothing: the ids staged below are -1 or more
        const float slope = p.slopes ? p.slopes[h] * kLog2e : 0.f, scale2 = p.scale * kLog2e;
        const bool capped = p.cap > 0.f, special = capped || p.slopes || !(scale2 > 0.f);
        int *dk = docs + warp * 128;
        float m = -INFINITY, l = 0.f;
        int n = 0;
        bool ok = true;
        for (int j = next(1 << my, reach, 0); j < ntiles && ok; j = next(1 << my, reach, j + 1)) {
            const int j0 = j * 128;
            const bool plain = by_doc ? (full[my * kWords + j / 32] >> (j & 31)) & 1 : j0 + 128 <= whole;
            if (by_doc && !plain) {
                __syncwarp();  // the ids of the tile before have been read
#pragma unroll
                for (int x = lane; x < 128; x += 32) dk[x] = j0 + x < sp.nk ? max(p.kv_docs[b * p.kds + j0 + x], -1) : -1;
                __syncwarp();
            }
            // one outcome for the warp, whose lanes then load tensor memory together
            ok = __all_sync(0xffffffffu, mbar_wait_spin(&s_full[my], n & 1, ta.status, stop, 48, ta.budget));
            if (!ok) break;
            tc_fence_after();
            float f[128], top = -INFINITY, mul = scale2;
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(ts + c * 32, f + c * 32);
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_wait32(f + c * 32);
            if (EXTRA && special) {
                mul = 1.f;
                if (capped) {
#pragma unroll
                    for (int c = 0; c < 4; c++) cap32<T>(f + c * 32, p.scale, p.cap);
                } else {
#pragma unroll
                    for (int x = 0; x < 128; x++) f[x] *= scale2;
                }
                if (p.slopes) {
                    const float far = (float)(pos - j0);
#pragma unroll
                    for (int x = 0; x < 128; x++) f[x] = fmaf(-slope, fabsf(far - (float)x), f[x]);
                }
            }
            if (!plain) {
                const int left = end - j0;
                if (!by_doc || p.causal) {  // (documents' ids end with the keys)
#pragma unroll
                    for (int x = 0; x < 128; x++)
                        if (x >= left) f[x] = -INFINITY;
                }
                if (EXTRA && by_doc) {
#pragma unroll
                    for (int x = 0; x < 128; x += 4) {
                        const int4 d = *(const int4 *)(dk + x);
                        if (d.x != doc) f[x] = -INFINITY;
                        if (d.y != doc) f[x + 1] = -INFINITY;
                        if (d.z != doc) f[x + 2] = -INFINITY;
                        if (d.w != doc) f[x + 3] = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; c++) top = max32(f + c * 32, top);
            top *= mul;
            top = fmaxf(m, top);
            if (m == -INFINITY) m = top;  // nothing seen so far: nothing to rescale
            const bool grown = m > -INFINITY && top - m > kSlack;
            if (__any_sync(0xffffffffu, grown) && n > 0) {
                // the second product of the tile before is complete: s_full follows it
                const float c = grown ? ex2(m - top) : 1.f;
                if (grown) m = top;
                l *= c;
#pragma unroll 1
                for (int c0 = 0; c0 < p.dim; c0 += 32) {
                    float o[32];
                    tmem_ld32(to + c0, o);
                    tmem_wait32(o);
#pragma unroll
                    for (int x = 0; x < 32; x++) o[x] *= c;
                    tmem_st32(to + c0, o);
                }
            }
            // Weights, their sum, and the weights as 16-bit operands where the scores were.
            const float base = m == -INFINITY ? 0.f : m;
            const float2 mul2 = make_float2(mul, mul), off2 = make_float2(-base, -base);
            float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[16];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    float2 e = __ffma2_rn(make_float2(f[c * 32 + 2 * x], f[c * 32 + 2 * x + 1]), mul2, off2);
                    e.x = ex2(e.x);
                    e.y = ex2(e.y);
                    if (x & 1) sum1 = __fadd2_rn(sum1, e);
                    else sum0 = __fadd2_rn(sum0, e);
                    w[x] = pack2<T>(e.x, e.y);  // the one rounding of a weight: the matrix instruction takes 16 bits
                }
                tmem_st16(ts + c * 16, w);
                if (c == 1) {  // the product of the first 64 keys may begin
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_half[my]);
                }
            }
            sum0 = __fadd2_rn(sum0, sum1);
            l += sum0.x + sum0.y;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[my]);
            n++;
        }
        if (ok) ok = warp_wait(&o_full[my], 0, ta.status, stop, 49, ta.budget);
        if (ok) {
            tc_fence_after();
            if (!SPLIT) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                bool bad = !finite(l) || (l == 0.f && end > 0);
                // rows through shared memory (the queries' tile is done with), 16-byte pieces XORed with the
                // row against bank conflicts, so that a warp's stores cover whole rows
                T *o = (T *)p.o + b * p.os[0] + h * p.os[1] + (int64_t)(i - lane) * p.os[2];
                uint8_t *stage = sm + L::q + my * L::tile + (warp & 3) * (L::tile / 4);
                constexpr int kPieces = DP / 8;
#pragma unroll 1
                for (int c0 = 0; c0 < p.dim; c0 += 32) {
                    float f[32];
                    if (n > 0) {
                        tmem_ld32(to + c0, f);
                        tmem_wait32(f);
                    } else {
#pragma unroll
                        for (int x = 0; x < 32; x++) f[x] = 0.f;
                    }
#pragma unroll
                    for (int x = 0; x < 32; x++) {
                        bad |= c0 + x < p.dim && !finite(f[x]);
                        f[x] *= inv;
                    }
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        *(uint4 *)(stage + lane * DP * 2 + ((c0 / 8 + x) ^ (lane & 7)) * 16) =
                            make_uint4(pack2<T>(f[8 * x], f[8 * x + 1]), pack2<T>(f[8 * x + 2], f[8 * x + 3]),
                                       pack2<T>(f[8 * x + 4], f[8 * x + 5]), pack2<T>(f[8 * x + 6], f[8 * x + 7]));
                }
                __syncwarp();
                const int pieces = p.dim / 8, rows_left = sp.nq - (i - lane);
#pragma unroll 4
                for (int u = lane; u < 32 * kPieces; u += 32) {
                    const int r = u / kPieces, c = u % kPieces;
                    if (r >= rows_left || c >= pieces) continue;
                    const uint4 v = *(const uint4 *)(stage + r * DP * 2 + (c ^ (r & 7)) * 16);
                    T *at = o + r * p.os[2] + c * 8;
                    if (ta.vec_out) {
                        *(uint4 *)at = v;
                    } else {
                        const T *e = (const T *)&v;
#pragma unroll
                        for (int x = 0; x < 8; x++) at[x] = e[x];
                    }
                }
                __syncwarp();
                uint32_t rows = __ballot_sync(0xffffffffu, bad && row);
                Absent none;
                while (rows) {
                    const int r = 31 - __clz(rows);
                    rows ^= 1u << r;
                    __syncwarp();
                    none = row_again<T>(p, b, h, i - lane + r, none);
                }
            }
        }
        got = ok && n > 0;
        row_m = m;
        row_l = l;
        tc_fence_before();
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT) {
        // every product and load of the block is done: values and keys make room for the sums, rows of
        // 32-bit pieces of 16 bytes XORed with the row
        tc_fence_after();
        float *sums = (float *)sm, *ml = (float *)(sm + L::docs);
        if (warp < kMmaWarp) {
            const int r = my * 128 + (tid & 127);
            const uint32_t to = tmem + ((uint32_t)(warp & 3) << 21) + kColO + my * 128;
#pragma unroll 1
            for (int c0 = 0; c0 < p.dim; c0 += 32) {
                float f[32];
                if (got) {
                    tmem_ld32(to + c0, f);
                    tmem_wait32(f);
                } else {
#pragma unroll
                    for (int x = 0; x < 32; x++) f[x] = 0.f;
                }
#pragma unroll
                for (int x = 0; x < 8; x++)
                    *(float4 *)(sums + r * DP + ((c0 / 4 + x) ^ (r & 7)) * 4) = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
            }
            ml[2 * r] = row_m;
            ml[2 * r + 1] = row_l;
        }
        tc_fence_before();
        cl.sync();
        // a warp per row, the rows shared out
        Absent none;
        for (int r = 128 * NT - 1 - rank * (kThreads / 32) - warp; r >= 0; r -= cs * (kThreads / 32)) {
            const int at = i_first + r;
            if (at >= sp.nq) continue;
            float top = -INFINITY, total = 0.f, share[8];
            for (int c = 0; c < cs; c++) top = fmaxf(top, cl.map_shared_rank(ml, c)[2 * r]);
            const float z = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int c = 0; c < 8; c++) {
                share[c] = 0.f;
                if (c >= cs) continue;
                const float *of = cl.map_shared_rank(ml, c) + 2 * r;
                share[c] = ex2(of[0] - z);
                total = fmaf(share[c], of[1], total);
            }
            const float inv = total == 0.f ? 0.f : 1.f / total;
            bool bad = !finite(total) || (total == 0.f && may_see(p, sp, b, at));
            T *o = (T *)p.o + b * p.os[0] + h * p.os[1] + (int64_t)at * p.os[2];
            if (lane * 4 < p.dim) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    if (c >= cs) continue;
                    const float4 x = *(const float4 *)(cl.map_shared_rank(sums, c) + r * DP + (lane ^ (r & 7)) * 4);
                    const float f = share[c] * inv;
                    v = make_float4(fmaf(f, x.x, v.x), fmaf(f, x.y, v.y), fmaf(f, x.z, v.z), fmaf(f, x.w, v.w));
                }
                bad |= !finite(v.x) || !finite(v.y) || !finite(v.z) || !finite(v.w);
                const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int x = 0; x < 4; x++) o[lane * 4 + x] = from_f<T>(e[x]);
            }
            __syncwarp();
            if (__any_sync(0xffffffffu, bad)) none = row_again<T>(p, b, h, at, none);
        }
        cl.sync();  // the sums are read until here
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
    }
}

// [batch][heads][tokens][dim] with element strides, boxes of 128 tokens x 64 dimensions; what lies
// outside reads as zero
void make_map(CUtensorMap &m, bool bf16, const void *p, const int64_t *st, int batch, int heads, int tokens, int dim) {
    auto fn = encode_fn();
    if (!fn) fail(WOCR_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
    // the stride of a dimension of one is not used, but has to be valid
    auto stride = [&](int64_t s, int n) { return (cuuint64_t)((n > 1 ? s : dim) * 2); };
    const cuuint64_t strides[3] = {stride(st[2], tokens), stride(st[1], heads), stride(st[0], batch)};
    const cuuint32_t box[4] = {64, 128, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = fn(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(p),
                          dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(WOCR_ERR_CUDA, "cuTensorMapEncodeTiled (attention) failed: " + std::to_string((int)r));
}

template <typename T, int DP, int NT, bool EXTRA>
void launch(Ctx *c, TcArgs ta, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t s) {
    const int bytes = Smem<DP, NT>::bytes;
    ta.tiles = (ta.a.q_len + 128 * NT - 1) / (128 * NT);
    const int64_t units = (int64_t)ta.tiles * ta.a.batch * ta.a.heads;
    // while there is room on the GPU and a block keeps three key tiles (8 heads of 128, 20 queries over
    // 4,096 keys: 55 us in one block a head)
    int cs = 1;
    while (cs < 8 && units * cs * 2 <= c->sm_count * (3 - NT) && ta.a.kv_len >= 2 * cs * 384) cs *= 2;
    if (cs > 1) {
        auto kernel = k_attn_tc<T, DP, NT, EXTRA, true>;
        launch_cluster<TcArgs, CUtensorMap, CUtensorMap, CUtensorMap>(kernel, dim3((unsigned)(units * cs)), threads_of(NT), cs, bytes, s, ta, mq, mk, mv);
    } else {
        auto kernel = k_attn_tc<T, DP, NT, EXTRA, false>;
        WOCR_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        kernel<<<(unsigned)units, threads_of(NT), bytes, s>>>(ta, mq, mk, mv);
    }
    WOCR_LAUNCHED(c);
}
template <typename T>
void launch_dim(Ctx *c, const TcArgs &ta, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t s) {
    const AttnP &p = ta.a;
    const bool extra = extra_scores(p) || !(p.scale > 0.f);
    if (p.dim <= 64) {
        // one tile a block up to 1,024 queries: 128 sequences of 128 queries, 8 heads of 64: 26 us
        // against 48; 16 of 1,024: 70 us both; 8 of 2,048: 121 us against 118
        if (p.q_len <= 1024) {
            if (extra) launch<T, 64, 1, true>(c, ta, mq, mk, mv, s);
            else launch<T, 64, 1, false>(c, ta, mq, mk, mv, s);
        } else {
            if (extra) launch<T, 64, 2, true>(c, ta, mq, mk, mv, s);
            else launch<T, 64, 2, false>(c, ta, mq, mk, mv, s);
        }
    } else {
        if (extra) launch<T, 128, 2, true>(c, ta, mq, mk, mv, s);
        else launch<T, 128, 2, false>(c, ta, mq, mk, mv, s);
    }
}
}  // namespace

bool attention_tc_ok(const AttnP &p) {
    if (p.type == WOCR_F32 || p.dim % 8 || p.dim > 128 || p.kv_len < 1) return false;
    if (p.kv_len > kMaxTiles * 128 || (int64_t)p.batch * p.heads * ((p.q_len + 127) / 128) > 0x7fffffff) return false;
    // TMA: 16-byte rows, at most 2^40 bytes apart, and no broadcast dimension
    auto fits = [](const void *x, const int64_t *st, int batch, int heads, int tokens) {
        const int n[3] = {batch, heads, tokens};
        if ((uintptr_t)x % 16) return false;
        for (int d = 0; d < 3; d++)
            if (n[d] > 1 && (st[d] % 8 || st[d] <= 0 || st[d] >= 1ll << 38)) return false;
        return true;
    };
    return fits(p.q, p.qs, p.batch, p.heads, p.q_len) && fits(p.k, p.ks, p.batch, p.kv_heads, p.kv_len) &&
           fits(p.v, p.vs, p.batch, p.kv_heads, p.kv_len);
}

void attention_tc(Ctx *c, const AttnP &p, cudaStream_t s) {
    const bool bf = p.type == WOCR_BF16;
    TcArgs ta;
    ta.a = p;
    ta.status = c->status;
    ta.budget = kWaitBudget;
    ta.vec_out = (uintptr_t)p.o % 16 == 0 && p.os[0] % 8 == 0 && p.os[1] % 8 == 0 && p.os[2] % 8 == 0;
    CUtensorMap mq, mk, mv;
    make_map(mq, bf, p.q, p.qs, p.batch, p.heads, p.q_len, p.dim);
    make_map(mk, bf, p.k, p.ks, p.batch, p.kv_heads, p.kv_len, p.dim);
    make_map(mv, bf, p.v, p.vs, p.batch, p.kv_heads, p.kv_len, p.dim);
    if (bf) launch_dim<__nv_bfloat16>(c, ta, mq, mk, mv, s);
    else launch_dim<__half>(c, ta, mq, mk, mv, s);
}

}  // namespace k
}  // namespace wocr
