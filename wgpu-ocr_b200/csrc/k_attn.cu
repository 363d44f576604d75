// Softmax attention with capped scores, a bias by distance and causal, prefix and document masks.
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(s_ij - max_j s_ij) over the keys that i sees
#include <algorithm>

#include "attn.h"

namespace wocr {
namespace k {

namespace {
using namespace attn;

template <typename T>
__global__ void __launch_bounds__(128) k_attn_rows(const AttnP p) {
    const int64_t rows = (int64_t)p.batch * p.heads * p.q_len;
    for (int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 5); r < rows; r += gridDim.x * 4ll) {
        const int i = (int)(r % p.q_len);
        const int h = (int)(r / p.q_len % p.heads);
        row_by_warp<T>(p, (int)(r / p.q_len / p.heads), h, i);
    }
}
}  // namespace

void attention(Ctx *c, const AttnP &p, cudaStream_t s) {
    if (p.batch == 0 || p.q_len == 0) return;
    const int64_t rows = (int64_t)p.batch * p.heads * p.q_len;
    const int grid = (int)std::min<int64_t>((rows + 3) / 4, c->sm_count * 64);
    if (p.type == WOCR_F32) k_attn_rows<float><<<grid, 128, 0, s>>>(p);
    else if (p.type == WOCR_F16) k_attn_rows<__half><<<grid, 128, 0, s>>>(p);
    else k_attn_rows<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
    WOCR_LAUNCHED(c);
}

}  // namespace k
}  // namespace wocr
