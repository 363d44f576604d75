// Operators on the caller's device tensors: attention, beam search's selection and reordering of
// states, CTC prefix beam search.  Launchers take the stream they run on; the entry points
// (ops.cpp) have checked every argument.
#pragma once

#include <optional>

#include "common.h"

namespace wocr {
namespace k {

// Brackets an operator with events when the context profiles, on the context's own stream only (a
// caller's stream may be capturing, and is not waited for by the profile's report).
struct OpProf {
    std::optional<Prof> prof;
    OpProf(Ctx *c, cudaStream_t s, const char *name, double flops, double bytes) {
        if (c->prof && s == c->stream) prof.emplace(c, name, flops, bytes);
    }
};

// Softmax attention (wocr_attention in wocr.h): sizes, element strides (batch, head, token; the
// dimension within a head is contiguous) and masks.
struct AttnP {
    const void *q, *k, *v;
    void *o;
    int64_t qs[3], ks[3], vs[3], os[3];
    const float *slopes;                    // [heads] or null
    const int *prefix, *q_lens, *kv_lens;   // [batch] or null
    const int *q_docs, *kv_docs;            // [batch][..] or null (both or neither)
    int64_t qds, kds;                       // their batch strides
    int type, batch, heads, kv_heads, q_len, kv_len, dim, causal;
    float scale, cap;
};
void attention(Ctx *c, const AttnP &p, cudaStream_t s);

// Beam search's selection: the best `kout` of `kin` beams x `vocab` tokens per batch element.
struct BeamP {
    const void *logits;
    int64_t lb, lk;               // element strides of batch and beam
    const float *scores;          // [batch][kin]
    const uint8_t *finished;      // [batch][kin] or null
    float *out_scores;            // [batch][kout], as the following
    int *out_parents, *out_tokens;
    uint8_t *out_finished;        // or null
    int type, batch, kin, kout, vocab, end;
};
constexpr int kMaxBeams = 32;
void beam_select(Ctx *c, const BeamP &p, cudaStream_t s);

// States put in the order of the chosen beams: row b * kout + j of dst becomes row
// b * kin + parents[b][j] of src, `pieces` pieces of `bytes` bytes, `step` bytes apart, in rows of
// `row` bytes (src and dst alike).
struct ReorderState {
    const void *src;
    void *dst;
    int64_t pieces, bytes, step, row;
};
constexpr int kMaxStates = 64;  // of one launch
void beam_reorder(Ctx *c, const int *parents, int batch, int kin, int kout, const ReorderState *st, int n,
                  cudaStream_t s);

// CTC prefix beam search over logits [lines][steps][classes].
struct CtcP {
    const void *logits;
    int64_t ln, lt;               // element strides of line and step
    const int *lens;              // [lines] or null
    int *tokens;                  // [lines][paths][steps], -1 past a path's length
    int *lengths;                 // [lines][paths]
    float *scores;                // [lines][paths]
    int type, lines, steps, classes, width, paths, blank;
};
constexpr int kMaxWidth = 31;     // width + 1 classes of a step are one per lane of a warp
void ctc_beam(Ctx *c, const CtcP &p, cudaStream_t s);

}  // namespace k
}  // namespace wocr
