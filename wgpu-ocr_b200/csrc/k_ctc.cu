// CTC prefix beam search on the device.
//   A beam is a text with the log masses of its alignments that end in a blank (pb) and in its last
//   class (pn).  A step with logits x keeps a text, pb' = log(e^pb + e^pn) + x_blank and
//   pn' = pn + x_last, or appends a class c, pn' = log(e^pb + e^pn) + x_c (pb + x_c when c is its
//   last class again); a text reached both ways adds the masses up.  The best `width` go on.
// What a step adds to all classes alike shifts every beam alike: x is taken from the step's largest logit, so that
// masses stay near zero and 64 bits hold their differences, and the log-sum-exp above it enters the scores only.
#include <algorithm>
#include <climits>

#include "elem.h"
#include "ops.h"
#include "topk.h"

namespace wocr {
namespace k {

namespace {
using namespace topk;

// Masses are compared in multiples of 2^-30, ties to the lower place, so that no order hangs on
// the last bits of exp and log; logits are held to the same multiples (32-bit values of 2^-6 and
// more are multiples already).
constexpr float kStep = 1073741824.f;
__device__ __forceinline__ float on_step(float x) {
    x = clean(x);
    return fabsf(x) < 0.015625f ? rintf(x * kStep) * (1.f / kStep) : x;
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a step's logits leave for the search: its best classes apart from the blank (value, class;
// class -1 behind the last), the blank's logit, the largest logit (0 where all are -inf) and the
// log-sum-exp above it.
struct Step {
    float *val;
    int *cls;
    float *blank, *max;
    double *lse;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGather = 2048;
constexpr size_t kSmemMax = 227 * 1024;

struct RowSmem {
    Key lists[32];
    Key got[kGather];
    Key top[32];
    float wm[kWarps];
    double ws[kWarps];
    int count;
};

// A block per row: maximum and best class of each thread, exponentials, then (as in beam selection)
// the classes that pass the K-th best of the threads' best.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_ctc_rows(const CtcP p, const Step out, int K, int cached) {
    extern __shared__ __align__(16) uint8_t dyn[];
    RowSmem &sm = *reinterpret_cast<RowSmem *>(dyn);
    T *store = reinterpret_cast<T *>(dyn + sizeof(RowSmem));
    const int64_t r = blockIdx.x;
    const int line = (int)(r / p.steps), t = (int)(r % p.steps);
    if (p.lens && t >= p.lens[line]) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.classes;
    const T *row = (const T *)p.logits + line * p.ln + t * p.lt;
    if (tid == 0) sm.count = 0;
    Key best = 0;
    float m = -INFINITY;
#pragma unroll 8
    for (int e = tid; e < n; e += kThreads) {
        const T raw = row[e];
        if (cached) store[e] = raw;
        const float x = on_step(to_f(raw));
        m = fmaxf(m, x);
        const Key key = make_key(x, e);
        if (e != p.blank && key > best) best = key;
        if (e == p.blank) out.blank[r] = x;
    }
    for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) sm.wm[warp] = m;
    best_slots<kThreads>(best, tid, sm.lists);
    if (tid < 32) sm.top[tid] = 0;
    __syncthreads();
    const Key cut = kth_slot(sm.lists, K);
    m = sm.wm[0];
    for (int w = 1; w < kWarps; w++) m = fmaxf(m, sm.wm[w]);
    float s = 0.f;
#pragma unroll 8
    for (int e = tid; e < n; e += kThreads) {
        const float x = on_step(to_f(cached ? store[e] : row[e]));
        if (m > -INFINITY) s += exp2_of((x - m) * kLog2e);
        const Key key = make_key(x, e);
        if (key >= cut && e != p.blank) {
            const int g = atomicAdd(&sm.count, 1);
            if (g < kGather) sm.got[g] = key;
        }
    }
    for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) sm.ws[warp] = s;
    __syncthreads();
    const int got = sm.count;
    if (got <= kGather) {
        for (int g = tid; g < got; g += kThreads) {
            const Key c = sm.got[g];
            int place = 0;
            for (int o = 0; o < got; o++) place += sm.got[o] > c;
            if (place < K) sm.top[place] = c;
        }
    } else {
        Key last = ~0ull;
        for (int q = 0; q < K; q++) {  // many classes on one side of the bound: the best, then the next
            Key next = 0;
            for (int e = tid; e < n; e += kThreads) {
                const Key c = make_key(on_step(to_f(cached ? store[e] : row[e])), e);
                if (e != p.blank && c < last && c > next) next = c;
            }
            for (int d = 16; d; d /= 2) next = max(next, shfl_xor(next, d));
            if (lane == 0) sm.lists[warp] = next;
            __syncthreads();
            for (int w = 0; w < kWarps; w++) next = max(next, sm.lists[w]);
            if (tid == 0) sm.top[q] = next;
            last = next;
            __syncthreads();
        }
    }
    __syncthreads();
    if (tid < K) {
        const Key c = sm.top[tid];
        out.val[r * K + tid] = c ? key_value(c) : -INFINITY;
        out.cls[r * K + tid] = c ? (int)key_place(c) : -1;
    }
    if (tid == 0) {
        double sum = 0;
        for (int w = 0; w < kWarps; w++) sum += sm.ws[w];
        out.max[r] = m > -INFINITY ? m : 0.f;
        out.lse[r] = m > -INFINITY ? log(sum) : -INFINITY;
    }
}

// log(1 + e^-d) for d >= 0, on 608 intervals of 1/16 up to 38 (beyond, it is below 2^-54): the Taylor
// polynomial of degree 7 about an interval's middle leaves (1/32)^8 / 8! max |f^(8)| < 2^-55.  With
// s = 1 / (1 + e^d) and u = s (1 - s): f' = -s, f'' = u and f^(n+1) = -u df^(n)/ds.
constexpr int kLogs = 608;
struct LogTable {
    double c[kLogs][8];
    __device__ void fill(int tid, int n) {
        for (int i = tid; i < kLogs; i += n) {
            const double d = (i + 0.5) / 16, e = exp(-d), s = e / (1 + e), u = s * (1 - s), w = 1 - 2 * s;
            c[i][0] = log1p(e);
            c[i][1] = -s;
            c[i][2] = u / 2;
            c[i][3] = -u * w / 6;
            c[i][4] = u * (1 - 6 * u) / 24;
            c[i][5] = -u * w * (1 - 12 * u) / 120;
            c[i][6] = u * (1 - 30 * u + 120 * u * u) / 720;
            c[i][7] = -u * w * (1 - 60 * u + 360 * u * u) / 5040;
        }
    }
    __device__ __forceinline__ double add(double a, double b) const {
        const double hi = fmax(a, b), d = hi - fmin(a, b);
        if (!(d < 38.0)) return hi;  // -inf and both -inf among them
        const int i = (int)(d * 16);
        const double x = d - (i + 0.5) / 16;
        const double2 *q = reinterpret_cast<const double2 *>(c[i]);
        const double2 q0 = q[0], q1 = q[1], q2 = q[2], q3 = q[3];
        // by halves: a shorter chain than Horner's
        const double x2 = x * x, x4 = x2 * x2;
        const double lo = fma(fma(q1.y, x, q1.x), x2, fma(q0.y, x, q0.x)), up = fma(fma(q3.y, x, q3.x), x2, fma(q2.y, x, q2.x));
        return hi + fma(up, x4, lo);
    }
};

// A text's identity: 64 bits mixed class by class (the multiply-xorshift finaliser of splitmix64,
// Steele, Lea and Flood, 2014).
__device__ __forceinline__ uint64_t grow(uint64_t h, int c) {
    h = (h ^ (uint64_t)(uint32_t)(c + 1)) + 0x9e3779b97f4a7c15ull;
    h = (h ^ (h >> 30)) * 0xbf58476d1ce4e5b9ull;
    h = (h ^ (h >> 27)) * 0x94d049bb133111ebull;
    return h ^ (h >> 31);
}

// Pairs of a beam i (from 0, in descending order) and a class k (from 0, best first) with
// k (i + 1) <= width.
constexpr int pairs(int width) {
    int n = 0;
    for (int i = 1; i <= width; i++) n += width / i + 1;
    return n;
}
constexpr int candidates(int width) { return 2 * width + pairs(width); }
constexpr int kMaxCand = candidates(kMaxWidth);
constexpr int kMaxSearch = (4 * kMaxCand + 31) / 32 * 32;
constexpr int kTrace = 64;                       // steps traced back per load

struct Beams {
    double pb[32], pn[32], tot[32];
    uint64_t hash[32], before[32];               // of the text, and of the text without its last class
    int last[32], len[32];
    double xl[32];                               // the step's logit of the last class, from its largest
    int live;
};
constexpr int64_t kNever = INT64_MIN;            // the key of what is no candidate

struct SearchSmem {
    LogTable log;
    Beams beams[2];
    int64_t key[kMaxCand];                       // log masses in steps, their bits made monotone
    uint32_t place[kMaxCand];
    double cn[kMaxCand], cb[32], ct[32];
    int floor;                                   // high word that a candidate's key needs
    uint8_t pi[kMaxCand], pk[kMaxCand];
    uint32_t kids[2][32];                        // beams that are a beam's text and a class more
    int parent[32];                              // and the beam that a text is one class more than, or -1
    double val[2][32];                           // logits of a step, from its largest
    int cls[2][32];
    double next[2][32];                          // the next step's logits of the beams' last classes, of the best classes
    double blank[2], norm;
    uint32_t back[kTrace * 32];
};

// A block per line, step after step.  Of beam i only the classes k with k (i + 1) <= width can be
// among the best: each pair before (i, k) in both orders is as good, but for one class that a beam
// repeats, and where a pair grows into a held text, that text's own candidate is as good.  Candidates
// in the order of their places: texts kept, then (beam, class); each one's rank is the number of
// better ones, counted by four threads.  With all beams alive the least of the kept texts bounds the
// candidates that are worth a count.
// Bound: latency, 1.4 us a step with 4 texts, 1.9 us with 16, of which a mass addition takes 0.17 us.
// What a step reads is loaded a step ahead: its best classes, and its logits of every
// class that a beam may then end in (the beams' last classes and the best classes of the step before),
// which a prefetch into L2 has asked for a step earlier still.
template <typename T>
__global__ void __launch_bounds__(kMaxSearch) k_ctc_search(const CtcP p, const Step st, uint32_t *back) {
    extern __shared__ __align__(16) uint8_t dyn[];
    SearchSmem &sm = *reinterpret_cast<SearchSmem *>(dyn);
    const int line = blockIdx.x, tid = threadIdx.x, N = blockDim.x, lane = tid & 31, warp = tid >> 5, W = p.width, K = W + 1;
    const int len = p.lens ? min(max(p.lens[line], 0), p.steps) : p.steps;
    const int cand = candidates(W), loader = N / 32 - 2;
    const T *x0 = (const T *)p.logits + line * p.ln;
    const int64_t r0 = (int64_t)line * p.steps;
    uint32_t *bk = back + r0 * W;
    sm.log.fill(tid, N);
    if (tid < 64) sm.kids[tid >> 5][lane] = 0;
    if (tid == 0) {
        int n = 2 * W;
        for (int i = 0; i < W; i++) {
            sm.pi[i] = sm.pi[W + i] = i;
            for (int k = 0; k * (i + 1) <= W; k++) {
                sm.pi[n] = i;
                sm.pk[n++] = k;
            }
        }
        Beams &b = sm.beams[0];
        b.live = 1;
        b.pb[0] = b.tot[0] = 0.0;
        b.pn[0] = -INFINITY;
        b.hash[0] = 0;
        b.before[0] = ~0ull;
        b.last[0] = -1;
        b.len[0] = 0;
        b.xl[0] = -INFINITY;
        if (len > 0) sm.blank[0] = (double)st.blank[r0] - st.max[r0];
    }
    if (tid < K && len > 0) {
        sm.val[0][tid] = (double)st.val[r0 * K + tid] - st.max[r0];
        sm.cls[0][tid] = st.cls[r0 * K + tid];
    }
    __syncthreads();
    int cur = 0;
    for (int t = 0; t < len; t++, cur ^= 1) {
        const int64_t r = r0 + t;
        Beams &now = sm.beams[cur], &then = sm.beams[cur ^ 1];
        const int n = now.live;
        // loads for the next step, stored at the end of this one's first half
        T nx = from_f<T>(0.f);
        float nv = 0.f, nb = 0.f, nm = 0.f;
        int nc = -1;
        const bool more = t + 1 < len;
        if (more && warp >= loader) {
            const int c = warp == loader ? (lane < n ? now.last[lane] : -1) : (lane < K ? sm.cls[cur][lane] : -1);
            const T *row = x0 + (t + 1) * p.lt;
            if (c >= 0) nx = row[c];
            nm = st.max[r + 1];
            if (warp > loader && lane < K) {
                nv = st.val[(r + 1) * K + lane];
                nc = st.cls[(r + 1) * K + lane];
            }
            if (warp > loader) nb = st.blank[r + 1];
            if (t + 2 < len && c >= 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + p.lt + c));
        }
        // which beams are one class more than another: a warp per longer text, lanes are the shorter
        {
            const uint64_t h = lane < n ? now.hash[lane] : 0;
            const int size = lane < n ? now.len[lane] + 1 : -1;
            for (int j = warp; j < n; j += N / 32) {
                const uint32_t m = __ballot_sync(0xffffffffu, h == now.before[j] && size == now.len[j]);
                if (lane == 0) {
                    sm.parent[j] = m ? __ffs(m) - 1 : -1;
                    if (m) atomicOr(&sm.kids[cur][__ffs(m) - 1], 1u << j);
                }
            }
        }
        if (tid == N - 1) then.live = 0;
        __syncthreads();
        auto monotone = [](double mass) -> int64_t {
            const int64_t bits = __double_as_longlong(rint(mass * (double)kStep) + 0.0);  // -0 as 0
            return mass > -INFINITY ? bits ^ ((bits >> 63) & INT64_MAX) : kNever;
        };
        if (warp == 0) {  // texts kept
            int64_t key = kNever;
            if (lane < n) {
                const int o = sm.parent[lane];
                const double b = now.tot[lane] + sm.blank[cur];
                double q = now.pn[lane] + now.xl[lane];
                if (o >= 0) q = sm.log.add(q, (now.last[o] == now.last[lane] ? now.pb[o] : now.tot[o]) + now.xl[lane]);
                const double total = sm.log.add(b, q);
                sm.cb[lane] = b;
                sm.cn[lane] = q;
                sm.ct[lane] = total;
                key = monotone(total);
            }
            if (lane < W) {
                sm.key[lane] = key;
                sm.place[lane] = lane;
            }
            const int least = __reduce_min_sync(0xffffffffu, lane < W ? (int)(key >> 32) : INT_MAX);
            if (lane == 0) sm.floor = least;
        } else if (W + tid - 32 < cand) {  // texts grown
            const int u = W + tid - 32, i = sm.pi[u];
            double q = -INFINITY;
            if (i < n) {
                const bool again = u < 2 * W;
                const int k = sm.pk[u], c = again ? now.last[i] : sm.cls[cur][k];
                if (c >= 0 && (again || c != now.last[i])) {
                    bool held = false;
                    for (uint32_t kids = sm.kids[cur][i]; kids; kids &= kids - 1) held |= now.last[__ffs(kids) - 1] == c;
                    if (!held) q = again ? now.pb[i] + now.xl[i] : now.tot[i] + sm.val[cur][k];
                    sm.place[u] = W + (uint32_t)i * p.classes + c;
                }
            }
            sm.cn[u] = q;
            sm.key[u] = monotone(q);
        }
        if (warp >= loader) {
            sm.kids[cur ^ 1][lane] = 0;
            if (more) {
                sm.next[warp - loader][lane] = (double)on_step(to_f(nx)) - nm;
                if (warp > loader) {
                    if (lane < K) {
                        sm.val[cur ^ 1][lane] = (double)nv - nm;
                        sm.cls[cur ^ 1][lane] = nc;
                    }
                    if (lane == 0) sm.blank[cur ^ 1] = (double)nb - nm;
                }
            }
        }
        __syncthreads();
        {
            const int u = tid >> 2;
            const int64_t key = u < cand ? sm.key[u] : kNever;
            const bool near = key != kNever && (int)(key >> 32) >= sm.floor;
            int rank = 0, same = 0;
            if (near) {
#pragma unroll 4
                for (int o = tid & 3; o < cand; o += 4) {
                    const int64_t other = sm.key[o];
                    rank += other > key;
                    same += other == key;
                }
            }
            same += __shfl_xor_sync(0xffffffffu, same, 1);
            same += __shfl_xor_sync(0xffffffffu, same, 2);
            if (same > 1)
                for (int o = tid & 3; o < cand; o += 4) rank += sm.key[o] == key && sm.place[o] < sm.place[u];
            rank += __shfl_xor_sync(0xffffffffu, rank, 1);
            rank += __shfl_xor_sync(0xffffffffu, rank, 2);
            if (near && rank < W && (tid & 3) == 0) {
                const bool kept = u < W, again = u < 2 * W;
                const int i = sm.pi[u], k = sm.pk[u];
                const int c = again ? now.last[i] : sm.cls[cur][k];
                const double q = sm.cn[u];
                then.pb[rank] = kept ? sm.cb[u] : -INFINITY;
                then.pn[rank] = q;
                then.tot[rank] = kept ? sm.ct[u] : q;
                then.hash[rank] = kept ? now.hash[i] : grow(now.hash[i], c);
                then.before[rank] = kept ? now.before[i] : now.hash[i];
                then.last[rank] = c;
                then.len[rank] = now.len[i] + !kept;
                then.xl[rank] = c >= 0 ? sm.next[again ? 0 : 1][again ? i : k] : -INFINITY;
                bk[(int64_t)t * W + rank] = (uint32_t)i << 27 | (uint32_t)(kept ? 0 : c + 1);
                atomicMax(&then.live, rank + 1);
            }
        }
        __syncthreads();
    }
    Beams &end = sm.beams[cur];
    const int n = end.live;
    if (warp == 0) {  // the steps' log-sum-exps above their largest logits
        double norm = 0;
        for (int t = lane; t < len; t += 32) norm += st.lse[r0 + t];
        for (int d = 16; d; d /= 2) norm += __shfl_xor_sync(0xffffffffu, norm, d);
        if (lane == 0) sm.norm = norm;
    }
    const int64_t o0 = (int64_t)line * p.paths;
    for (int64_t u = tid; u < (int64_t)p.paths * p.steps; u += N) {
        const int j = (int)(u / p.steps);
        if ((int)(u % p.steps) >= (j < n ? end.len[j] : 0)) p.tokens[(o0 + j) * p.steps + u % p.steps] = -1;
    }
    if (tid < p.paths) p.lengths[o0 + tid] = tid < n ? end.len[tid] : 0;
    __syncthreads();
    if (tid < p.paths) p.scores[o0 + tid] = tid < n ? (float)(end.tot[tid] - sm.norm) : -INFINITY;
    // each path traced back through the steps' origins, kTrace steps in shared memory at a time
    int j = tid, pos = tid < n ? end.len[tid] : 0;
    for (int t1 = len; t1 > 0; t1 -= kTrace) {
        const int t0 = max(0, t1 - kTrace);
        __syncthreads();
        for (int u = tid; u < (t1 - t0) * W; u += N) sm.back[u] = bk[(int64_t)t0 * W + u];
        __syncthreads();
        if (tid < p.paths && tid < n)
            for (int t = t1 - 1; t >= t0; t--) {
                const uint32_t e = sm.back[(t - t0) * W + j];
                if (e & 0x7ffffffu) p.tokens[(o0 + tid) * p.steps + --pos] = (int)(e & 0x7ffffffu) - 1;
                j = e >> 27;
            }
    }
}

// The same with a row's logits in the registers of N threads, E each: rows of up to N E classes.
// With N = 32 a block's eight warps have a row each.  Bound: issue slots, 60 % of them taken by 30
// instructions a logit (4,800 rows of 18,709 classes of 32 bits: 130 us, 2.7 TB/s; rounding only what is
// taken out saved a third of the instructions and took 15 % longer).
template <typename T, int N, int E>
__global__ void __launch_bounds__(N == 32 ? 256 : N, N == 512 ? 2 : 1) k_ctc_rows_reg(const CtcP p, const Step out, int K, int64_t rows) {
    constexpr int WARPS = N / 32, PER = N == 32 ? 8 : 1, GOT = 512;
    __shared__ struct {
        Key lists[32];
        Key got[GOT];
        Key top[32];
        Key cut;
        float wm[WARPS], ws[WARPS];
        int count;
    } smem[PER];
    const int part = N == 32 ? threadIdx.x >> 5 : 0, tid = N == 32 ? threadIdx.x & 31 : threadIdx.x;
    auto &sm = smem[part];
    auto sync = [] {
        if (N == 32) __syncwarp();
        else __syncthreads();
    };
    const int64_t r = (int64_t)blockIdx.x * PER + part;
    if (r >= rows) return;
    const int line = (int)(r / p.steps), t = (int)(r % p.steps);
    if (p.lens && t >= p.lens[line]) return;
    const int lane = tid & 31, warp = tid >> 5, n = p.classes;
    const T *row = (const T *)p.logits + line * p.ln + t * p.lt;
    // the blank is no candidate: it stays out of the row, but for the sum
    const float xb = tid == 0 ? on_step(to_f(row[p.blank])) : -INFINITY;
    float x[E];
#pragma unroll
    for (int k = 0; k < E; k++) {
        const int e = k * N + tid;
        x[k] = e < n && e != p.blank ? to_f(row[e]) : -INFINITY;
    }
    if (tid == 0) {
        sm.count = 0;
        out.blank[r] = xb;
    }
    float m = xb;
#pragma unroll
    for (int k = 0; k < E; k++) {
        x[k] = on_step(x[k]);
        m = fmaxf(m, x[k]);
    }
    float bv = x[0];
    int bk = 0;
#pragma unroll
    for (int k = 1; k < E; k++)
        if (x[k] > bv) bv = x[k], bk = k;
    const Key best = bv > -INFINITY ? make_key(bv, bk * N + tid) : 0;
    for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (lane == 0) sm.wm[warp] = m;
    best_slots<N>(best, tid, sm.lists);
    sync();
    if (warp == 0) {  // one warp only: the count is as long as a pass over a thread's logits
        const Key cut = kth_slot(sm.lists, K);
        if (lane == 0) sm.cut = cut;
        sm.top[lane] = 0;
    }
    sync();
    const Key cut = sm.cut;
    const float least = cut ? key_value(cut) : -INFINITY;
    m = sm.wm[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) m = fmaxf(m, sm.wm[w]);
    const float base = m > -INFINITY ? m : 0.f;
    float s = exp2_of((xb - base) * kLog2e);
#pragma unroll
    for (int k = 0; k < E; k++) {
        s += exp2_of((x[k] - base) * kLog2e);
        if (x[k] >= least && x[k] > -INFINITY) {
            const Key c = make_key(x[k], k * N + tid);
            if (c >= cut) {
                const int g = atomicAdd(&sm.count, 1);
                if (g < GOT) sm.got[g] = c;
            }
        }
    }
    for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) sm.ws[warp] = s;
    sync();
    const int got = sm.count;
    if (got <= GOT) {
        for (int g = tid; g < got; g += N) {
            const Key c = sm.got[g];
            int at = 0;
            for (int o = 0; o < got; o++) at += sm.got[o] > c;
            if (at < K) sm.top[at] = c;
        }
    } else {
        Key last = ~0ull;
        for (int q = 0; q < K; q++) {
            Key next = 0;
            for (int e = tid; e < n; e += N) {  // from memory again: seldom, and the registers are full
                const float v = on_step(to_f(row[e]));
                const Key c = v > -INFINITY && e != p.blank ? make_key(v, e) : 0;
                if (c < last && c > next) next = c;
            }
            for (int d = 16; d; d /= 2) next = max(next, shfl_xor(next, d));
            if (lane == 0) sm.lists[warp] = next;
            sync();
            for (int w = 0; w < WARPS; w++) next = max(next, sm.lists[w]);
            if (tid == 0) sm.top[q] = next;
            last = next;
            sync();
        }
    }
    sync();
    if (tid < K) {
        const Key c = sm.top[tid];
        out.val[r * K + tid] = c ? key_value(c) : -INFINITY;
        out.cls[r * K + tid] = c ? (int)key_place(c) : -1;
    }
    if (tid == 0) {
        double sum = 0;
        for (int w = 0; w < WARPS; w++) sum += sm.ws[w];
        out.max[r] = m > -INFINITY ? m : 0.f;
        out.lse[r] = m > -INFINITY ? log(sum) : -INFINITY;
    }
}

template <typename T, int N, int E>
void rows_reg(const CtcP &p, const Step &st, int K, int64_t rows, cudaStream_t s) {
    const int per = N == 32 ? 8 : 1;
    k_ctc_rows_reg<T, N, E><<<(unsigned)((rows + per - 1) / per), N == 32 ? 256 : N, 0, s>>>(p, st, K, rows);
}

template <typename T>
void run(Ctx *c, const CtcP &p, const Step &st, uint32_t *back, cudaStream_t s) {
    const int K = p.width + 1;
    const int64_t rows = (int64_t)p.lines * p.steps;
    if (rows > 0) {
        if (p.classes <= 32 * 4) {
            rows_reg<T, 32, 4>(p, st, K, rows, s);
        } else if (p.classes <= 32 * 16) {
            rows_reg<T, 32, 16>(p, st, K, rows, s);
        } else if (p.classes <= 128 * 16) {
            rows_reg<T, 128, 16>(p, st, K, rows, s);
        } else if (p.classes <= 256 * 24) {
            rows_reg<T, 256, 24>(p, st, K, rows, s);
        } else if (p.classes <= 512 * 40) {
            rows_reg<T, 512, 40>(p, st, K, rows, s);
        } else {
            const size_t row = (size_t)p.classes * sizeof(T);
            const int cached = sizeof(RowSmem) + row <= kSmemMax;
            WOCR_CUDA(cudaFuncSetAttribute(k_ctc_rows<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
            k_ctc_rows<T><<<(unsigned)rows, kThreads, sizeof(RowSmem) + (cached ? row : 0), s>>>(p, st, K, cached);
        }
        WOCR_LAUNCHED(c);
    }
    const int threads = std::max(96, (4 * candidates(p.width) + 31) / 32 * 32);  // a warp keeps, two load ahead
    WOCR_CUDA(cudaFuncSetAttribute(k_ctc_search<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SearchSmem)));
    k_ctc_search<T><<<p.lines, threads, sizeof(SearchSmem), s>>>(p, st, back);
    WOCR_LAUNCHED(c);
}
}  // namespace

void ctc_beam(Ctx *c, const CtcP &p, cudaStream_t s) {
    if (p.lines == 0) return;
    OpProf pf(c, s, "ctc_beam", 0, (double)p.lines * p.steps * p.classes * elem_size(p.type));
    // workspace of this call alone, ordered on the call's stream (a graph that captures the call
    // gets its own)
    const size_t rows = std::max<size_t>((size_t)p.lines * p.steps, 1), K = p.width + 1;
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t a = up(rows * 8), b = up(rows * K * 4), d = up(rows * 4);
    uint8_t *w = nullptr;
    WOCR_CUDA(cudaMallocFromPoolAsync((void **)&w, a + 2 * b + 2 * d + up(rows * p.width * 4), c->pool, s));
    Step st;
    st.lse = (double *)w;
    st.val = (float *)(w + a);
    st.cls = (int *)(w + a + b);
    st.blank = (float *)(w + a + 2 * b);
    st.max = (float *)(w + a + 2 * b + d);
    uint32_t *back = (uint32_t *)(w + a + 2 * b + 2 * d);
    try {
        if (p.type == WOCR_F32) run<float>(c, p, st, back, s);
        else if (p.type == WOCR_F16) run<__half>(c, p, st, back, s);
        else run<__nv_bfloat16>(c, p, st, back, s);
    } catch (...) {
        cudaFreeAsync(w, s);
        throw;
    }
    WOCR_CUDA(cudaFreeAsync(w, s));
}

}  // namespace k
}  // namespace wocr
