// Beam search's selection over beams and vocabulary, and the reordering of the beams' states.
//   candidate (j, v) of a batch element: score_j + x_jv - log sum_u exp x_ju;  the best kout of all
//   kin x vocab, ties to the lower place j vocab + v
#include <cooperative_groups.h>

#include <algorithm>

#include "elem.h"
#include "ops.h"
#include "topk.h"

namespace cg = cooperative_groups;

namespace wocr {
namespace k {

namespace {
using namespace topk;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGather = 2048;  // candidates a block gathers before it falls back to rounds
constexpr size_t kSmemMax = 227 * 1024;

struct SelectSmem {
    Cand lists[32];
    Cand got[kGather];
    Cand top[kMaxBeams];                                     // the block's best, read by its cluster
    double base[kMaxBeams];                                  // score - log-sum-exp
    double ws[kMaxBeams][kWarps], bs[kMaxBeams];             // sums of exponentials: per warp; per block, read by its cluster
    float wm[kMaxBeams][kWarps], bm[kMaxBeams];              // maxima, the same
    uint8_t fin[kMaxBeams];
    Cand cut;
    int count;
};

// One cluster per batch element; a block holds `slice` tokens of every beam's row, in shared memory
// when `cached`, so that the logits are read from HBM once: maximum, then exponentials, then (with
// the cluster's log-sum-exps) the best candidate of each thread.  The kout-th best of those is a
// lower bound of the answer's last candidate, and few pass it: they are gathered and ranked.
// Bound: the four passes over a block's logits, an element a load, and the barriers between them, not the
// bytes (256 rows of 18,709 in 16 bits, 9.6 MB, whose floor is 1.5 us: 34.5 us call after call, 40 us cold; 512
// threads a block took 10 % longer, eight beams' loads under way together 20 %; sums in 64 bits cost 3 %).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_beam_select(const BeamP p, int slice, int cached) {
    extern __shared__ __align__(16) uint8_t dyn[];
    SelectSmem &sm = *reinterpret_cast<SelectSmem *>(dyn);
    T *store = reinterpret_cast<T *>(dyn + sizeof(SelectSmem));
    cg::cluster_group cl = cg::this_cluster();
    const int cs = cl.num_blocks(), rank = cl.block_rank();
    const int b = blockIdx.x / cs;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int v0 = rank * slice, n = max(0, min(slice, p.vocab - v0));
    const T *rows = (const T *)p.logits + b * p.lb + v0;
    if (tid < p.kin) sm.fin[tid] = p.finished ? p.finished[(int64_t)b * p.kin + tid] != 0 : 0;
    if (tid == 0) sm.count = 0;
    __syncthreads();
    for (int j = 0; j < p.kin; j++) {
        if (sm.fin[j]) continue;
        const T *row = rows + j * p.lk;
        float m = -INFINITY;
#pragma unroll 8
        for (int e = tid; e < n; e += kThreads) {
            const T x = row[e];
            if (cached) store[(int64_t)j * slice + e] = x;
            m = fmaxf(m, clean(to_f(x)));
        }
        for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (lane == 0) sm.wm[j][warp] = m;
    }
    __syncthreads();
    // a thread reads the tokens that it stored itself from here on
    auto at = [&](int j, int e) -> float {
        if (sm.fin[j]) return v0 + e == p.end ? 0.f : -INFINITY;  // an ended beam: `end` at its own score
        return clean(to_f(cached ? store[(int64_t)j * slice + e] : rows[j * p.lk + e]));
    };
    for (int j = 0; j < p.kin; j++) {
        if (sm.fin[j]) continue;
        float m = sm.wm[j][0];
        for (int w = 1; w < kWarps; w++) m = fmaxf(m, sm.wm[j][w]);
        double s = 0;  // (beside a certain token, what the others add decides between beams)
        if (m > -INFINITY)
#pragma unroll 8
            for (int e = tid; e < n; e += kThreads) s += exp2f((at(j, e) - m) * 1.4426950408889634f);
        for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) sm.ws[j][warp] = s;
        if (tid == 0) sm.bm[j] = m;
    }
    __syncthreads();
    if (tid < p.kin) {
        double s = 0;
        for (int w = 0; w < kWarps; w++) s += sm.ws[tid][w];
        sm.bs[tid] = s;
    }
    cl.sync();
    if (tid < p.kin) {
        // the log-sum-exp of a beam decides between beams: joined in 64 bits
        const float sc = clean(p.scores[(int64_t)b * p.kin + tid]);
        double base = sc;
        if (!sm.fin[tid]) {
            float m = -INFINITY;
            for (int r = 0; r < cs; r++) m = fmaxf(m, cl.map_shared_rank(sm.bm, r)[tid]);
            double s = 0;
            for (int r = 0; r < cs; r++) {
                const float mr = cl.map_shared_rank(sm.bm, r)[tid];
                if (mr > -INFINITY) s += cl.map_shared_rank(sm.bs, r)[tid] * exp((double)mr - m);
            }
            base = m > -INFINITY ? base - (m + log(s)) : -INFINITY;
        }
        sm.base[tid] = base;
    }
    __syncthreads();
    Cand best = worst((Cand *)nullptr);
    for (int j = 0; j < p.kin; j++) {
        const double base = sm.base[j];
        float xm = -INFINITY;
        int xe = tid;
        if (base > -INFINITY)
#pragma unroll 8
            for (int e = tid; e < n; e += kThreads) {
                const float x = at(j, e);
                if (x > xm) xm = x, xe = e;
            }
        if (tid < n) {
            const Cand c = {base + xm, (uint32_t)j * p.vocab + v0 + xe};
            if (better(c, best)) best = c;
        }
    }
    best_slots<kThreads>(best, tid, sm.lists);
    __syncthreads();
    if (warp == 0) {
        const Cand cut = kth_slot(sm.lists, p.kout);
        if (lane == 0) sm.cut = cut;
    }
    __syncthreads();
    const Cand cut = sm.cut;
    for (int j = 0; j < p.kin; j++) {
        // Where base + x rounds to cut or more, it is at least cut less half a step of 64 bits, below 2^-52 |cut|.
        // The difference is rounded down: |base| may be so large that many x give the same sum.
        const double base = sm.base[j];
        float least = -INFINITY;
        if (cut.v > -INFINITY)
            least = base > -INFINITY ? __double2float_rd(__dsub_rd(__dsub_rd(cut.v, base), fabs(cut.v) * 0x1p-52)) : INFINITY;
#pragma unroll 4
        for (int e = tid; e < n; e += kThreads) {
            const float x = at(j, e);
            if (x >= least) {
                const Cand c = {base + x, (uint32_t)j * p.vocab + v0 + e};
                if (!better(cut, c)) {
                    const int g = atomicAdd(&sm.count, 1);
                    if (g < kGather) sm.got[g] = c;
                }
            }
        }
    }
    __syncthreads();
    const int got = sm.count;
    if (tid < kMaxBeams) sm.top[tid] = worst((Cand *)nullptr);
    __syncthreads();
    if (got <= kGather) {
        for (int g = tid; g < got; g += kThreads) {
            const Cand c = sm.got[g];
            int r = 0;
            for (int o = 0; o < got; o++) r += better(sm.got[o], c);
            if (r < p.kout) sm.top[r] = c;
        }
    } else {
        // many candidates on one side of the bound (sorted rows): the best, then the next, in rounds
        Cand last = {INFINITY, 0};
        for (int r = 0; r < p.kout; r++) {
            Cand next = worst((Cand *)nullptr);
            for (int j = 0; j < p.kin; j++)
                for (int e = tid; e < n; e += kThreads) {
                    const Cand c = {sm.base[j] + at(j, e), (uint32_t)j * p.vocab + v0 + e};
                    if (better(last, c) && better(c, next)) next = c;
                }
            for (int d = 16; d; d /= 2) {
                const Cand o = shfl_xor(next, d);
                if (better(o, next)) next = o;
            }
            if (lane == 0) sm.lists[warp] = next;
            __syncthreads();
            for (int w = 0; w < kWarps; w++)
                if (better(sm.lists[w], next)) next = sm.lists[w];
            if (tid == 0) sm.top[r] = next;
            last = next;
            __syncthreads();
        }
    }
    cl.sync();
    if (rank == 0) {
        const int all = cs * p.kout;  // at most 8 x 32
        if (tid < all) sm.got[tid] = cl.map_shared_rank(sm.top, tid / p.kout)[tid % p.kout];
        __syncthreads();
        if (tid < all) {
            const Cand c = sm.got[tid];
            int r = 0;
            for (int o = 0; o < all; o++) r += better(sm.got[o], c);
            if (r < p.kout && c.i != 0xffffffffu) {
                const int64_t w = (int64_t)b * p.kout + r;
                const int j = c.i / p.vocab, tok = c.i % p.vocab;
                p.out_scores[w] = (float)c.v;
                p.out_parents[w] = j;
                p.out_tokens[w] = tok;
                if (p.out_finished) p.out_finished[w] = sm.fin[j] || tok == p.end;
            }
        }
    }
    cl.sync();  // the blocks' shared memory is read until here
}

struct ReorderArgs {
    ReorderState st[kMaxStates];
    const int *parents;
    int kin, kout;
};

// A block copies 8 x 256 words of V of one row of one state.  Bound: the bytes, once in and once out
// (629 MB of caches in 70 us cold, 8.9 TB/s with what the L2 cache holds).
template <typename V>
__global__ void __launch_bounds__(256) k_beam_reorder(const __grid_constant__ ReorderArgs a) {
    const ReorderState &st = a.st[blockIdx.z];
    const int row = blockIdx.y;
    const int parent = a.parents[row];
    if (parent < 0 || parent >= a.kin) return;  // no such beam: the row stays as it was
    const uint32_t per = (uint32_t)(st.bytes / sizeof(V)), total = (uint32_t)st.pieces * per;  // below 2^31
    const uint8_t *src = (const uint8_t *)st.src + ((int64_t)(row / a.kout) * a.kin + parent) * st.row;
    uint8_t *dst = (uint8_t *)st.dst + row * st.row;
    V v[8];
    int64_t off[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
        const uint32_t w = blockIdx.x * 2048u + u * 256 + threadIdx.x;
        off[u] = w < total ? (int64_t)(w / per) * st.step + (int64_t)(w % per) * sizeof(V) : -1;
        if (off[u] >= 0) v[u] = *(const V *)(src + off[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
        if (off[u] >= 0) *(V *)(dst + off[u]) = v[u];
}

template <typename T>
void select_t(Ctx *c, const BeamP &p, cudaStream_t s) {
    // blocks per batch element: more while a block still has 4,096 logits or more and the GPU room
    int cs = 1;
    auto bytes = [&](int n) { return (size_t)p.kin * ((p.vocab + n - 1) / n) * sizeof(T); };
    while (cs < 8 && (int64_t)p.kin * p.vocab / cs > 4096 &&
           (p.batch * cs < 2 * c->sm_count || sizeof(SelectSmem) + bytes(cs) > kSmemMax))
        cs *= 2;
    const int slice = (p.vocab + cs - 1) / cs;
    const int cached = sizeof(SelectSmem) + bytes(cs) <= kSmemMax;
    const size_t smem = sizeof(SelectSmem) + (cached ? bytes(cs) : 0);
    WOCR_CUDA(cudaFuncSetAttribute(k_beam_select<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.batch * cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    WOCR_CUDA(cudaLaunchKernelEx(&cfg, k_beam_select<T>, p, slice, cached));
    WOCR_LAUNCHED(c);
}
}  // namespace

void beam_select(Ctx *c, const BeamP &p, cudaStream_t s) {
    if (p.batch == 0) return;
    OpProf pf(c, s, "beam_select", 0, (double)p.batch * p.kin * p.vocab * elem_size(p.type));
    if (p.type == WOCR_F32) select_t<float>(c, p, s);
    else if (p.type == WOCR_F16) select_t<__half>(c, p, s);
    else select_t<__nv_bfloat16>(c, p, s);
}

void beam_reorder(Ctx *c, const int *parents, int batch, int kin, int kout, const ReorderState *st, int n,
                  cudaStream_t s) {
    if (batch == 0) return;
    const int rows = batch * kout;
    double bytes = 0;
    for (int i = 0; i < n; i++) bytes += 2.0 * rows * st[i].pieces * st[i].bytes;
    OpProf pf(c, s, "beam_reorder", 0, bytes);
    for (int i = 0; i < n;) {
        ReorderArgs a;
        a.parents = parents;
        a.kin = kin;
        a.kout = kout;
        // states that allow the same word go in one launch
        auto word = [](const ReorderState &t) {
            const uint64_t all = (uint64_t)t.src | (uint64_t)t.dst | t.bytes | t.step | t.row;
            return all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
        };
        const int w = word(st[i]);
        int m = 0;
        int64_t most = 0;
        for (; i < n && m < kMaxStates && word(st[i]) == w; i++) {
            if (st[i].pieces * st[i].bytes == 0) continue;
            if (st[i].pieces * st[i].bytes / w > 0x7fff0000ll)
                fail(WOCR_ERR_UNSUPPORTED, "a state's row has more than 2^31 words to copy");
            a.st[m++] = st[i];
            most = std::max(most, st[i].pieces * st[i].bytes / w);
        }
        if (!m) continue;
        // a grid's second dimension ends at 65,535: whole batch elements per launch
        for (int r0 = 0, step; r0 < rows; r0 += step) {
            step = std::min(rows - r0, 65535 / kout * kout);
            ReorderArgs part = a;
            part.parents += r0;
            for (int q = 0; q < m; q++) {
                part.st[q].src = (const uint8_t *)part.st[q].src + (int64_t)(r0 / kout) * kin * part.st[q].row;
                part.st[q].dst = (uint8_t *)part.st[q].dst + (int64_t)r0 * part.st[q].row;
            }
            const dim3 grid((unsigned)((most + 2047) / 2048), step, m);
            if (w == 16) k_beam_reorder<uint4><<<grid, 256, 0, s>>>(part);
            else if (w == 4) k_beam_reorder<uint32_t><<<grid, 256, 0, s>>>(part);
            else k_beam_reorder<uint8_t><<<grid, 256, 0, s>>>(part);
            WOCR_LAUNCHED(c);
        }
    }
}

}  // namespace k
}  // namespace wocr
