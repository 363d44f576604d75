// Entry points of the operators on device tensors (ops.h): argument checks, the stream and the
// device of a call.
#include "ops.h"

#include <algorithm>
#include <climits>
#include <cmath>

#include "elem.h"

using namespace wocr;

namespace {

// The context's device for the duration of a call; the caller's current device comes back.
struct OnDevice {
    int was = -1, now;
    explicit OnDevice(int device) : now(device) {
        WOCR_CUDA(cudaGetDevice(&was));
        if (was != now) WOCR_CUDA(cudaSetDevice(now));
    }
    ~OnDevice() {
        if (was >= 0 && was != now) cudaSetDevice(was);
    }
};

Ctx *need_ctx(wocr_ctx *ctx) {
    Ctx *c = ctx_of(ctx);
    if (!c) fail(WOCR_ERR_INVALID, "null ctx");
    return c;
}
cudaStream_t stream_of(Ctx *c, void *stream) { return stream ? (cudaStream_t)stream : c->stream; }

void check_type(int type) {
    if (type != WOCR_F32 && type != WOCR_F16 && type != WOCR_BF16)
        fail(WOCR_ERR_UNSUPPORTED, "element type " + std::to_string(type) + " (float32, float16 and bfloat16 are supported)");
}
void check_ptr(const void *p, int align, const char *what) {
    if (!p) fail(WOCR_ERR_INVALID, std::string("null ") + what);
    if ((uintptr_t)p % align) fail(WOCR_ERR_INVALID, std::string(what) + " is not aligned to its elements");
}
void check_opt(const void *p, int align, const char *what) {
    if (p) check_ptr(p, align, what);
}
// dims x strides of a tensor whose elements must not share memory (an output)
void check_apart(const int64_t *dims, const int64_t *strides, int n, const char *what) {
    // ascending strides: each dimension steps over all of the smaller ones
    int64_t d[4], s[4];
    int m = 0;
    for (int i = 0; i < n; i++)
        if (dims[i] > 1) {
            int at = m++;
            for (; at > 0 && s[at - 1] > strides[i]; at--) d[at] = d[at - 1], s[at] = s[at - 1];
            d[at] = dims[i];
            s[at] = strides[i];
        }
    int64_t reach = 1;
    for (int i = 0; i < m; i++) {
        if (s[i] < reach) fail(WOCR_ERR_INVALID, std::string(what) + ": strides put elements on one another");
        reach = (d[i] - 1) * s[i] + reach;
    }
}
// What a call of beam_reorder reads or writes of a state: pieces in rows from `lo` on, all below `hi`.
struct Reach {
    uintptr_t lo, hi;
    int64_t used, piece, step, row;  // bytes of a row from its first piece to its last, of a piece; from piece to piece, row to row
    bool write;
};
bool shares(const Reach &a, const Reach &b) {  // a.lo <= b.lo
    if (b.lo >= a.hi) return false;
    // two that interleave: rows alike with each in its own part of a row, or of every piece's step
    auto apart = [&](int64_t every, int64_t of_a, int64_t of_b) {
        const int64_t at = (int64_t)((b.lo - a.lo) % every);
        return at >= of_a && at + of_b <= every;
    };
    if (a.row != b.row) return true;
    if (apart(a.row, a.used, b.used)) return false;
    return !(a.step == b.step && a.step > 0 && a.row % a.step == 0 && apart(a.step, a.piece, b.piece));
}
// Nothing may be read or written twice of which one is a write: the states are copied in no order.
void check_shares(std::vector<Reach> &all) {
    std::sort(all.begin(), all.end(), [](const Reach &a, const Reach &b) { return a.lo < b.lo; });
    std::vector<const Reach *> open;  // those that may reach to the next
    for (const Reach &r : all) {
        open.erase(std::remove_if(open.begin(), open.end(), [&](const Reach *o) { return o->hi <= r.lo; }), open.end());
        for (const Reach *o : open)
            if ((o->write || r.write) && shares(*o, r)) fail(WOCR_ERR_INVALID, "beam_reorder: what is written overlaps a source or another destination");
        open.push_back(&r);
    }
}
void check_strides(const int64_t *s, int n, const char *what) {
    for (int i = 0; i < n; i++)
        if (s[i] < 0) fail(WOCR_ERR_INVALID, std::string(what) + ": negative stride");
}

}  // namespace

extern "C" {

int32_t wocr_attention(wocr_ctx *ctx, const wocr_attention_args *a, void *stream) {
    return guard([&] {
        if (!a) fail(WOCR_ERR_INVALID, "null arguments");
        check_type(a->type);
        if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads <= 0 || a->kv_heads <= 0)
            fail(WOCR_ERR_INVALID, "attention: negative or zero sizes");
        if (a->heads % a->kv_heads)
            fail(WOCR_ERR_SHAPE, "attention: " + std::to_string(a->heads) + " heads cannot share " + std::to_string(a->kv_heads) +
                                     " key heads");
        if (a->head_dim < 1 || a->head_dim > 256)
            fail(WOCR_ERR_UNSUPPORTED, "attention: head dimension " + std::to_string(a->head_dim) + " (1 to 256 are supported)");
        if (!std::isfinite(a->scale) || !std::isfinite(a->cap) || a->cap < 0)
            fail(WOCR_ERR_INVALID, "attention: scale and cap must be finite, the cap not negative");
        // (no queries or no keys: their ids have no address)
        if (a->q_len > 0 && a->kv_len > 0 && (a->q_docs == nullptr) != (a->kv_docs == nullptr))
            fail(WOCR_ERR_INVALID, "attention: documents need the queries' and the keys' ids");
        if (a->prefix && !a->causal) fail(WOCR_ERR_INVALID, "attention: a prefix without a causal mask");
        if ((int64_t)a->batch * a->heads > 0x7fffffff / 2 || a->q_len > 1 << 30 || a->kv_len > 1 << 30)
            fail(WOCR_ERR_UNSUPPORTED, "attention: too many heads or tokens");
        if (a->batch == 0 || a->q_len == 0) {
            need_ctx(ctx);
            return;
        }
        const int es = k::elem_size(a->type);
        check_ptr(a->q, es, "q");
        check_ptr(a->out, es, "out");
        if (a->kv_len > 0) {
            check_ptr(a->k, es, "k");
            check_ptr(a->v, es, "v");
        }
        if (a->out == a->q || a->out == a->k || a->out == a->v) fail(WOCR_ERR_INVALID, "attention: out is one of the inputs");
        check_opt(a->slopes, 4, "slopes");
        check_opt(a->prefix, 4, "prefix");
        check_opt(a->q_lens, 4, "q_lens");
        check_opt(a->kv_lens, 4, "kv_lens");
        check_opt(a->q_docs, 4, "q_docs");
        check_opt(a->kv_docs, 4, "kv_docs");
        check_strides(a->q_strides, 3, "q");
        check_strides(a->k_strides, 3, "k");
        check_strides(a->v_strides, 3, "v");
        check_strides(a->out_strides, 3, "out");
        if (a->q_docs_stride < 0 || a->kv_docs_stride < 0) fail(WOCR_ERR_INVALID, "attention: negative stride");
        const int64_t od[4] = {a->batch, a->heads, a->q_len, a->head_dim};
        const int64_t os[4] = {a->out_strides[0], a->out_strides[1], a->out_strides[2], 1};
        check_apart(od, os, 4, "out");
        k::AttnP p;
        p.q = a->q;
        p.k = a->k;
        p.v = a->v;
        p.o = a->out;
        for (int i = 0; i < 3; i++) {
            p.qs[i] = a->q_strides[i];
            p.ks[i] = a->k_strides[i];
            p.vs[i] = a->v_strides[i];
            p.os[i] = a->out_strides[i];
        }
        p.slopes = a->slopes;
        p.prefix = a->prefix;
        p.q_lens = a->q_lens;
        p.kv_lens = a->kv_lens;
        p.q_docs = a->kv_len > 0 ? a->q_docs : nullptr;  // without keys nothing is seen anyway
        p.kv_docs = a->kv_len > 0 ? a->kv_docs : nullptr;
        p.qds = a->q_docs_stride;
        p.kds = a->kv_docs_stride;
        p.type = a->type;
        p.batch = a->batch;
        p.heads = a->heads;
        p.kv_heads = a->kv_heads;
        p.q_len = a->q_len;
        p.kv_len = a->kv_len;
        p.dim = a->head_dim;
        p.causal = a->causal != 0;
        p.scale = a->scale;
        p.cap = a->cap;
        Ctx *c = need_ctx(ctx);
        OnDevice on(c->device);
        k::attention(c, p, stream_of(c, stream));
    });
}

int32_t wocr_beam_select(wocr_ctx *ctx, const void *logits, int32_t type, int32_t batch, int32_t beams, int32_t vocab,
                         int64_t batch_stride, int64_t beam_stride, const float *scores, const uint8_t *finished, int32_t end,
                         int32_t out_beams, float *out_scores, int32_t *out_parents, int32_t *out_tokens,
                         uint8_t *out_finished, void *stream) {
    return guard([&] {
        check_type(type);
        if (batch < 0 || beams < 1 || out_beams < 1 || vocab < 1) fail(WOCR_ERR_INVALID, "beam_select: negative or zero sizes");
        if (beams > k::kMaxBeams || out_beams > k::kMaxBeams)
            fail(WOCR_ERR_UNSUPPORTED, "beam_select: more than " + std::to_string(k::kMaxBeams) + " beams");
        if (vocab > 1 << 26 || batch > 1 << 26) fail(WOCR_ERR_UNSUPPORTED, "beam_select: more than 2^26 tokens or batch elements");
        if ((int64_t)beams * vocab < out_beams)
            fail(WOCR_ERR_SHAPE, "beam_select: " + std::to_string(out_beams) + " beams out of " +
                                     std::to_string((int64_t)beams * vocab) + " candidates");
        if (end >= vocab) fail(WOCR_ERR_INVALID, "beam_select: the end token is not in the vocabulary");
        if (finished && end < 0) fail(WOCR_ERR_INVALID, "beam_select: finished beams need an end token");
        if (batch_stride < 0 || beam_stride < 0) fail(WOCR_ERR_INVALID, "beam_select: negative stride");
        if (batch == 0) {
            need_ctx(ctx);
            return;
        }
        check_ptr(logits, k::elem_size(type), "logits");
        check_ptr(scores, 4, "scores");
        check_ptr(out_scores, 4, "out_scores");
        check_ptr(out_parents, 4, "out_parents");
        check_ptr(out_tokens, 4, "out_tokens");
        // a batch element's scores and flags are read before its own are written, not another's
        if (beams != out_beams && (out_scores == scores || (finished && out_finished == finished)))
            fail(WOCR_ERR_INVALID, "beam_select: in place needs as many beams out as in");
        k::BeamP p;
        p.logits = logits;
        p.lb = batch_stride;
        p.lk = beam_stride;
        p.scores = scores;
        p.finished = finished;
        p.out_scores = out_scores;
        p.out_parents = out_parents;
        p.out_tokens = out_tokens;
        p.out_finished = out_finished;
        p.type = type;
        p.batch = batch;
        p.kin = beams;
        p.kout = out_beams;
        p.vocab = vocab;
        p.end = end < 0 ? -1 : end;
        Ctx *c = need_ctx(ctx);
        OnDevice on(c->device);
        k::beam_select(c, p, stream_of(c, stream));
    });
}

int32_t wocr_beam_reorder(wocr_ctx *ctx, const int32_t *parents, int32_t batch, int32_t beams, int32_t out_beams,
                          const wocr_beam_state *states, int32_t n_states, void *stream) {
    return guard([&] {
        if (batch < 0 || beams < 1 || out_beams < 1 || n_states < 0) fail(WOCR_ERR_INVALID, "beam_reorder: negative or zero sizes");
        if (beams > k::kMaxBeams || out_beams > k::kMaxBeams)
            fail(WOCR_ERR_UNSUPPORTED, "beam_reorder: more than " + std::to_string(k::kMaxBeams) + " beams");
        if ((int64_t)batch * std::max(beams, out_beams) > INT32_MAX) fail(WOCR_ERR_UNSUPPORTED, "beam_reorder: more than 2^31 rows");
        if (n_states > 0 && !states) fail(WOCR_ERR_INVALID, "null states");
        if (batch == 0 || n_states == 0) {
            need_ctx(ctx);
            return;
        }
        check_ptr(parents, 4, "parents");
        std::vector<k::ReorderState> st((size_t)n_states);
        std::vector<Reach> all;
        all.reserve(2 * (size_t)n_states);
        for (int i = 0; i < n_states; i++) {
            const wocr_beam_state &s = states[i];
            if (s.pieces < 0 || s.piece_bytes < 0 || s.piece_stride < 0 || s.row_stride < 0)
                fail(WOCR_ERR_INVALID, "beam_reorder: negative sizes");
            const int64_t rows = (int64_t)batch * std::max(beams, out_beams), most = INT64_MAX / 4;
            if ((s.pieces > 0 && s.piece_stride > most / s.pieces) || s.piece_bytes > most || s.row_stride > most / rows)
                fail(WOCR_ERR_INVALID, "beam_reorder: sizes beyond 64 bits");
            const int64_t used = s.pieces > 0 && s.piece_bytes > 0 ? (s.pieces - 1) * s.piece_stride + s.piece_bytes : 0;
            if (used > 0) {
                check_ptr(s.src, 1, "state");
                check_ptr(s.dst, 1, "state");
                if (s.pieces > 1 && s.piece_stride < s.piece_bytes) fail(WOCR_ERR_INVALID, "beam_reorder: pieces overlap");
                if (s.row_stride < used) fail(WOCR_ERR_INVALID, "beam_reorder: rows overlap");
                auto reach = [&](const void *p, int n, bool write) {
                    const uintptr_t lo = (uintptr_t)p;
                    all.push_back({lo, lo + ((int64_t)batch * n - 1) * s.row_stride + used, used, s.piece_bytes, s.piece_stride, s.row_stride, write});
                };
                reach(s.src, beams, false);
                reach(s.dst, out_beams, true);
            }
            st[i] = {s.src, s.dst, s.pieces, s.piece_bytes, s.piece_stride, s.row_stride};
        }
        check_shares(all);
        Ctx *c = need_ctx(ctx);
        OnDevice on(c->device);
        k::beam_reorder(c, parents, batch, beams, out_beams, st.data(), n_states, stream_of(c, stream));
    });
}

int32_t wocr_ctc_beam(wocr_ctx *ctx, const void *logits, int32_t type, int32_t lines, int32_t steps, int32_t classes,
                      int64_t line_stride, int64_t step_stride, const int32_t *lens, int32_t width, int32_t blank,
                      int32_t paths, int32_t *tokens, int32_t *lengths, float *scores, void *stream) {
    return guard([&] {
        check_type(type);
        if (lines < 0 || steps < 0 || classes < 1) fail(WOCR_ERR_INVALID, "ctc_beam: negative or zero sizes");
        if (width < 1 || width > k::kMaxWidth)
            fail(WOCR_ERR_UNSUPPORTED, "ctc_beam: width " + std::to_string(width) + " (1 to " + std::to_string(k::kMaxWidth) + " are supported)");
        if (paths < 1 || paths > width) fail(WOCR_ERR_INVALID, "ctc_beam: 1 to width paths");
        if (blank < 0 || blank >= classes) fail(WOCR_ERR_INVALID, "ctc_beam: the blank is not one of the classes");
        if (classes > (1 << 27) - 2) fail(WOCR_ERR_UNSUPPORTED, "ctc_beam: more than 2^27 classes");
        if ((int64_t)lines * steps > 0x7fffffff) fail(WOCR_ERR_UNSUPPORTED, "ctc_beam: more than 2^31 steps in all");
        if (line_stride < 0 || step_stride < 0) fail(WOCR_ERR_INVALID, "ctc_beam: negative stride");
        if (lines == 0) {
            need_ctx(ctx);
            return;
        }
        if (steps > 0) {
            check_ptr(logits, k::elem_size(type), "logits");
            check_ptr(tokens, 4, "tokens");
        }
        check_opt(lens, 4, "lens");
        check_ptr(lengths, 4, "lengths");
        check_ptr(scores, 4, "scores");
        k::CtcP p;
        p.logits = logits;
        p.ln = line_stride;
        p.lt = step_stride;
        p.lens = lens;
        p.tokens = tokens;
        p.lengths = lengths;
        p.scores = scores;
        p.type = type;
        p.lines = lines;
        p.steps = steps;
        p.classes = classes;
        p.width = width;
        p.paths = paths;
        p.blank = blank;
        Ctx *c = need_ctx(ctx);
        OnDevice on(c->device);
        k::ctc_beam(c, p, stream_of(c, stream));
    });
}

}  // extern "C"
