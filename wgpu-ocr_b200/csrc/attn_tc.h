// The tensor-core attention kernel (k_attn_tc.cu): which calls it takes, and its launch.
#pragma once

#include "ops.h"

namespace wocr {
namespace k {

bool attention_tc_ok(const AttnP &p);
void attention_tc(Ctx *c, const AttnP &p, cudaStream_t s);

}  // namespace k
}  // namespace wocr
