// CTC prefix beam search on the device.
//   A beam is a text with the log masses of its alignments that end in a blank (pb) and in its last
//   class (pn).  A step with logits x keeps a text, pb' = log(e^pb + e^pn) + x_blank and
//   pn' = pn + x_last, or appends a class c, pn' = log(e^pb + e^pn) + x_c (pb + x_c when c is its
//   last class again); a text reached both ways adds the masses up.  The best `width` go on.
// The steps' log-sum-exps shift every beam alike: they enter the scores only.
#include <algorithm>

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

// What a step's logits leave for the search: its best classes apart from the blank (value, class;
// class -1 behind the last), the blank's logit and the log-sum-exp.
struct Step {
    float *val;
    int *cls;
    float *blank;
    double *lse;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGather = 2048;
constexpr size_t kSmemMax = 227 * 1024;

struct RowSmem {
    Key lists[kWarps * 32];
    Key got[kGather];
    Key top[32];
    Key cut;
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
    const Key sorted = block_best32<kWarps>(best, sm.lists);
    if (tid < 32) sm.top[tid] = 0;
    if (tid == 0) sm.cut = 0;
    __syncthreads();
    if (warp == 0) {
        const Key cut = shfl(sorted, K - 1);
        if (lane == 0) sm.cut = cut;
    }
    __syncthreads();
    const Key cut = sm.cut;
    m = sm.wm[0];
    for (int w = 1; w < kWarps; w++) m = fmaxf(m, sm.wm[w]);
    float s = 0.f;
#pragma unroll 8
    for (int e = tid; e < n; e += kThreads) {
        const float x = on_step(to_f(cached ? store[e] : row[e]));
        if (m > -INFINITY) s += exp2f((x - m) * 1.4426950408889634f);
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
        out.lse[r] = m > -INFINITY ? m + log(sum) : -INFINITY;
    }
}

__device__ __forceinline__ double log_add(double a, double b) {
    const double hi = fmax(a, b), lo = fmin(a, b);
    return lo == -INFINITY ? hi : hi + log1p(exp(lo - hi));
}

// A text's identity: 64 bits mixed class by class (the multiply-xorshift finaliser of splitmix64,
// Steele, Lea and Flood, 2014).
__device__ __forceinline__ uint64_t grow(uint64_t h, int c) {
    h = (h ^ (uint64_t)(uint32_t)(c + 1)) + 0x9e3779b97f4a7c15ull;
    h = (h ^ (h >> 30)) * 0xbf58476d1ce4e5b9ull;
    h = (h ^ (h >> 27)) * 0x94d049bb133111ebull;
    return h ^ (h >> 31);
}

constexpr int kSearch = 128;                     // threads of a search block
constexpr int kMaxPairs = 160;                   // sum of floor(W / i) + 1 over i <= 31: 142
constexpr int kMaxCand = 2 * 32 + kMaxPairs;
constexpr int kTrace = 64;                       // steps traced back per load

struct SearchSmem {
    double pb[2][32], pn[2][32], tot[2][32];
    uint64_t hash[2][32];
    int last[2][32], len[2][32];
    double key[kMaxCand], cb[kMaxCand], cn[kMaxCand];
    uint32_t place[kMaxCand];
    uint8_t pi[kMaxPairs], pk[kMaxPairs];
    float xl[32];                                // the logit of each beam's last class
    float val[32];
    int cls[32];
    uint32_t back[kTrace * 32];
    int live[2];
    int pairs;
};

// A block per line, step after step.  Beams lie in descending order, so of beam i (from 0) only the
// classes k with k (i + 1) <= width can be among the best: each pair before (i, k) in both orders is
// as good, but for one class a beam repeats, and a pair that grows into a held text leaves that
// text's own candidate as good.  Candidates in the order of their places: texts kept, then (beam,
// class); each one's rank is the number of better ones.
template <typename T>
__global__ void __launch_bounds__(kSearch) k_ctc_search(const CtcP p, const Step st, uint32_t *back) {
    __shared__ SearchSmem sm;
    const int line = blockIdx.x, tid = threadIdx.x, W = p.width, K = W + 1;
    const int len = p.lens ? min(max(p.lens[line], 0), p.steps) : p.steps;
    const T *x0 = (const T *)p.logits + line * p.ln;
    uint32_t *bk = back + (int64_t)line * p.steps * W;
    if (tid == 0) {
        int n = 0;
        for (int i = 0; i < W; i++)
            for (int k = 0; k * (i + 1) <= W && k < K; k++) {
                sm.pi[n] = i;
                sm.pk[n++] = k;
            }
        sm.pairs = n;
        sm.live[0] = 1;
        sm.pb[0][0] = 0.0;
        sm.pn[0][0] = -INFINITY;
        sm.tot[0][0] = 0.0;
        sm.hash[0][0] = 0;
        sm.last[0][0] = -1;
        sm.len[0][0] = 0;
    }
    __syncthreads();
    const int cand = 2 * W + sm.pairs;
    double norm = 0;
    int cur = 0;
    for (int t = 0; t < len; t++, cur ^= 1) {
        const int64_t r = (int64_t)line * p.steps + t;
        const int n = sm.live[cur];
        if (tid < K) {
            sm.val[tid] = st.val[r * K + tid];
            sm.cls[tid] = st.cls[r * K + tid];
        }
        if (tid < n) {
            const int c = sm.last[cur][tid];
            sm.xl[tid] = c >= 0 ? on_step(to_f(x0[t * p.lt + c])) : -INFINITY;
        }
        if (tid == 0) {
            norm += st.lse[r];
            sm.live[cur ^ 1] = 0;
        }
        const double xb = st.blank[r];
        __syncthreads();
        for (int u = tid; u < cand; u += kSearch) {
            double b = -INFINITY, q = -INFINITY;
            uint32_t place = 0xffffffffu;
            if (u < W) {
                const int i = u;
                if (i < n) {
                    b = sm.tot[cur][i] + xb;
                    q = sm.pn[cur][i] + sm.xl[i];
                    if (sm.len[cur][i] > 0) {
                        const int c = sm.last[cur][i];
                        for (int o = 0; o < n; o++)
                            if (sm.len[cur][o] + 1 == sm.len[cur][i] && grow(sm.hash[cur][o], c) == sm.hash[cur][i])
                                q = log_add(q, (sm.last[cur][o] == c ? sm.pb[cur][o] : sm.tot[cur][o]) + sm.xl[i]);
                    }
                    place = i;
                }
            } else {
                const bool again = u < 2 * W;
                const int i = again ? u - W : sm.pi[u - 2 * W];
                if (i < n) {
                    const int c = again ? sm.last[cur][i] : sm.cls[sm.pk[u - 2 * W]];
                    if (c >= 0 && (again || c != sm.last[cur][i])) {
                        const uint64_t h = grow(sm.hash[cur][i], c);
                        bool held = false;
                        for (int o = 0; o < n; o++) held |= sm.hash[cur][o] == h && sm.len[cur][o] == sm.len[cur][i] + 1;
                        if (!held) {
                            q = again ? sm.pb[cur][i] + sm.xl[i] : sm.tot[cur][i] + sm.val[sm.pk[u - 2 * W]];
                            place = W + (uint32_t)i * p.classes + c;
                        }
                    }
                }
            }
            sm.cb[u] = b;
            sm.cn[u] = q;
            sm.key[u] = rint(log_add(b, q) * (double)kStep);
            sm.place[u] = place;
        }
        __syncthreads();
        for (int u = tid; u < cand; u += kSearch) {
            const double key = sm.key[u];
            if (!(key > -INFINITY)) continue;
            const uint32_t place = sm.place[u];
            int rank = 0;
            for (int o = 0; o < cand; o++) {
                const double ko = sm.key[o];
                rank += ko > key;
                if (ko == key) rank += sm.place[o] < place;
            }
            if (rank >= W) continue;
            const int nx = cur ^ 1;
            const bool kept = u < W;
            const int i = kept ? u : (u < 2 * W ? u - W : sm.pi[u - 2 * W]);
            const int c = kept ? -1 : (u < 2 * W ? sm.last[cur][i] : sm.cls[sm.pk[u - 2 * W]]);
            sm.pb[nx][rank] = sm.cb[u];
            sm.pn[nx][rank] = sm.cn[u];
            sm.tot[nx][rank] = log_add(sm.cb[u], sm.cn[u]);
            sm.hash[nx][rank] = kept ? sm.hash[cur][i] : grow(sm.hash[cur][i], c);
            sm.last[nx][rank] = kept ? sm.last[cur][i] : c;
            sm.len[nx][rank] = sm.len[cur][i] + !kept;
            bk[(int64_t)t * W + rank] = (uint32_t)i << 27 | (uint32_t)(c + 1);
            atomicMax(&sm.live[nx], rank + 1);
        }
        __syncthreads();
    }
    const int n = sm.live[cur];
    const int64_t o0 = (int64_t)line * p.paths;
    for (int64_t u = tid; u < (int64_t)p.paths * p.steps; u += kSearch) {
        const int j = (int)(u / p.steps);
        if ((int)(u % p.steps) >= (j < n ? sm.len[cur][j] : 0)) p.tokens[(o0 + j) * p.steps + u % p.steps] = -1;
    }
    if (tid < p.paths) {
        p.lengths[o0 + tid] = tid < n ? sm.len[cur][tid] : 0;
        if (tid == 0) sm.pb[cur ^ 1][0] = norm;
    }
    __syncthreads();
    if (tid < p.paths) p.scores[o0 + tid] = tid < n ? (float)(sm.tot[cur][tid] - sm.pb[cur ^ 1][0]) : -INFINITY;
    // each path traced back through the steps' origins, kTrace steps in shared memory at a time
    int j = tid, pos = tid < n ? sm.len[cur][tid] : 0;
    for (int t1 = len; t1 > 0; t1 -= kTrace) {
        const int t0 = max(0, t1 - kTrace);
        __syncthreads();
        for (int u = tid; u < (t1 - t0) * W; u += kSearch) sm.back[u] = bk[(int64_t)t0 * W + u];
        __syncthreads();
        if (tid < p.paths && tid < n)
            for (int t = t1 - 1; t >= t0; t--) {
                const uint32_t e = sm.back[(t - t0) * W + j];
                if (e & 0x7ffffffu) p.tokens[(o0 + tid) * p.steps + --pos] = (int)(e & 0x7ffffffu) - 1;
                j = e >> 27;
            }
    }
}

template <typename T>
void run(Ctx *c, const CtcP &p, const Step &st, uint32_t *back, cudaStream_t s) {
    const int K = p.width + 1;
    const int64_t rows = (int64_t)p.lines * p.steps;
    if (rows > 0) {
        const size_t row = (size_t)p.classes * sizeof(T);
        const int cached = sizeof(RowSmem) + row <= kSmemMax;
        WOCR_CUDA(cudaFuncSetAttribute(k_ctc_rows<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
        k_ctc_rows<T><<<(unsigned)rows, kThreads, sizeof(RowSmem) + (cached ? row : 0), s>>>(p, st, K, cached);
        WOCR_LAUNCHED(c);
    }
    k_ctc_search<T><<<p.lines, kSearch, 0, s>>>(p, st, back);
    WOCR_LAUNCHED(c);
}
}  // namespace

void ctc_beam(Ctx *c, const CtcP &p, cudaStream_t s) {
    if (p.lines == 0) return;
    // workspace of this call alone, ordered on the call's stream (a graph that captures the call
    // gets its own)
    const size_t rows = std::max<size_t>((size_t)p.lines * p.steps, 1), K = p.width + 1;
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t a = up(rows * 8), b = up(rows * K * 4), d = up(rows * 4);
    uint8_t *w = nullptr;
    WOCR_CUDA(cudaMallocFromPoolAsync((void **)&w, a + 2 * b + d + up(rows * p.width * 4), c->pool, s));
    Step st;
    st.lse = (double *)w;
    st.val = (float *)(w + a);
    st.cls = (int *)(w + a + b);
    st.blank = (float *)(w + a + 2 * b);
    uint32_t *back = (uint32_t *)(w + a + 2 * b + d);
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
