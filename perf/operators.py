"""Operators of recognition models on one B200: what is measured, in plain form and as the library's calls.

Three operators, each with its cases:

  attention  softmax attention of line and page encoders and of decoders over a cache: ragged batches, shared
             key heads, scores capped by a tanh, a bias by distance, causal, prefix and document masks
  beam       one step of beam search: selection over beams and vocabulary, then the states of the chosen beams
             put in their new order
  ctc        CTC prefix beam search over the class scores of whole lines

`own` false runs elementary torch operations, true the library's entry points.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DEV = "cuda"
_gpu = None


def _library():
    """The library's context on the current device, opened once as a program does."""
    global _gpu
    if _gpu is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        path = os.path.join(here, "wgpu-ocr_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import wocr
        _gpu = wocr.Gpu(device=torch.cuda.current_device())
    return _gpu


def _stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------
def _attention(name, type, batch, heads, kv_heads, q_len, kv_len, dim, layout, ragged=False, cap=0.0, slopes=False,
               causal=False, prefix=0, docs=0):
    return {"name": name, "op": "attention", "type": type, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "q_len": q_len, "kv_len": kv_len, "dim": dim, "layout": layout, "ragged": ragged, "cap": cap,
            "slopes": slopes, "causal": causal, "prefix": prefix, "docs": docs}


def _beam(name, type, batch, beams, vocab, done, layers, heads, room, live, dim):
    return {"name": name, "op": "beam", "type": type, "batch": batch, "beams": beams, "vocab": vocab, "done": done,
            "layers": layers, "heads": heads, "room": room, "live": live, "dim": dim}


def _ctc(name, type, lines, steps, classes, width, paths):
    return {"name": name, "op": "ctc", "type": type, "lines": lines, "steps": steps, "classes": classes,
            "width": width, "paths": paths}


def listed():
    return [
        # the recognition neck on one batch of 320-pixel lines: 8 heads of 15 in 32 bits, cut from one projection
        _attention("neck lines", "f32", 16, 8, 8, 40, 40, 15, "packed", ragged=True),
        # the same neck on a page's widest lines, padded to the widest, near positions preferred
        _attention("neck wide lines", "f32", 64, 8, 8, 400, 400, 15, "packed", ragged=True, slopes=True),
        # an encoder over the lines of a page packed one after another: a line sees itself only
        _attention("packed lines", "bf16", 1, 16, 16, 8192, 8192, 64, "packed", docs=40),
        # a page image's tokens seen whole, its text token by token, scores capped
        _attention("image prefix capped", "f16", 4, 16, 4, 2048, 2048, 128, "split", causal=True, prefix=1024, cap=30.0),
        # a long text prompt
        _attention("long prompt", "bf16", 1, 32, 8, 8192, 8192, 128, "split", causal=True),
        # one token of a few lines over a short cache
        _attention("token short", "f16", 2, 8, 8, 1, 200, 64, "split", ragged=True, causal=True),
        # one token of many texts over long caches
        _attention("token long", "bf16", 32, 32, 8, 1, 8192, 128, "split", ragged=True, causal=True),
        # the ocrs alphabet, one line, four beams
        _beam("step small", "f32", 1, 4, 97, 0.0, 1, 8, 128, 37, 64),
        # the PP-OCR dictionary, a page's lines, eight beams with ended ones among them
        _beam("step dictionary", "bf16", 32, 8, 18709, 0.2, 2, 8, 512, 300, 64),
        # one batch of lines through the CTC head of the PP-OCR dictionary
        _ctc("lines dictionary", "f32", 16, 40, 18709, 8, 1),
        # the widest lines of a page over the ocrs alphabet, a wide search, all its answers
        _ctc("lines alphabet", "f32", 64, 256, 97, 16, 16),
        # a page's lines through the dictionary's CTC head
        _ctc("page dictionary", "f32", 64, 100, 18709, 4, 2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lines", "lines", "prompt", "prompt", "prompt", "token", "token", "beam", "beam", "ctc", "ctc"])
    if kind == "lines":  # encoders of lines: narrow heads, ragged batches
        t = _log(rng, 1, 400)
        heads = rng.randint(1, 12)
        c = _attention("", rng.choice(["f32", "f32", "f16", "bf16"]), _log(rng, 1, 64), heads, heads, t, t,
                       rng.choice([8, 15, 16, 24, 30, 32, 40, 64]), "packed", ragged=rng.random() < 0.7,
                       slopes=rng.random() < 0.4, cap=rng.choice([0.0, 0.0, 20.0]))
    elif kind == "prompt":  # encoders of pages and prompts of decoders
        kv = rng.choice([1, 2, 4])
        group = rng.choice([1, 2, 4, 7])
        t = _log(rng, 100, 8192)
        b = max(1, min(8, (8192 * 8192) // (t * t * kv * group) * 8))
        mask = rng.choice(["none", "causal", "prefix", "docs", "causal docs"])
        s = t if rng.random() < 0.6 else t + _log(rng, 1, 4000)
        c = _attention("", rng.choice(["f16", "bf16"]), rng.randint(1, b), kv * group, kv, t, s,
                       rng.choice([32, 64, 64, 72, 96, 128, 128]), "split", ragged=rng.random() < 0.4,
                       cap=rng.choice([0.0, 0.0, 15.0, 50.0]), slopes=rng.random() < 0.25,
                       causal="causal" in mask or mask == "prefix", prefix=t // 3 if mask == "prefix" else 0,
                       docs=max(2, t // 300) if "docs" in mask else 0)
    elif kind == "token":  # decoders over a cache, one token or a few
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 1, 2, 4, 5, 8])
        c = _attention("", rng.choice(["f32", "f16", "bf16"]), _log(rng, 1, 32), kv * group, kv, rng.choice([1, 1, 1, 2, 5]),
                       _log(rng, 5, 8192), rng.choice([32, 64, 80, 128]), "split", ragged=rng.random() < 0.7, causal=True,
                       cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3)
    elif kind == "beam":
        room = _log(rng, 16, 512)
        c = _beam("", rng.choice(["f32", "f16", "bf16"]), _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 10, 16]),
                  _log(rng, 30, 18709), rng.choice([0.0, 0.2]), rng.randint(1, 2), rng.choice([1, 4, 8]), room,
                  rng.randint(1, room), rng.choice([32, 40, 64]))
    else:
        width = rng.choice([1, 2, 4, 5, 8, 16])
        classes = _log(rng, 10, 18709)
        steps = _log(rng, 1, 256)
        lines = max(1, min(_log(rng, 1, 64), 5000000 // (width * classes), 120000000 // (classes * steps)))
        c = _ctc("", rng.choice(["f32", "f32", "f16", "bf16"]), lines, steps, classes, width, rng.randint(1, width))
    del c["name"]
    # none costs more than the largest listed ones
    size = "lines" if kind == "ctc" else "batch"
    while c[size] > 1 and (work(c)["bytes"] > 3e8 * (2 if kind != "ctc" else 1) or work(c)["flops"] > 2.5e11):
        c[size] = c[size] // 2
    if work(c)["flops"] > 5e11:
        c["kv_heads"], c["heads"] = 1, c["heads"] // c["kv_heads"]
    return c


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _lens(case):
    """Lengths of the sequences of a ragged batch, from the longest down to half of it."""
    b, n, least = case["batch"], case["kv_len"], 1 if case["layout"] == "packed" else min(case["q_len"], case["kv_len"])
    return [max(least, n - (n * i) // (2 * b)) for i in range(b)] if case["ragged"] else [n] * b


def _doc_len(case):
    return case["kv_len"] / case["docs"]


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    if own:
        _library()
    return {"attention": _prepare_attention, "beam": _prepare_beam, "ctc": _prepare_ctc}[case["op"]](case, g, seed)


def _randn(shape, g, type):
    return torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32).to(_TYPES[type])


def _prepare_attention(case, g, seed):
    b, h, hk, tq, tk, d = (case[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
    s = {"case": case, "scale": d ** -0.5, "lens": None, "q_lens": None, "prefix": None, "slopes": None, "q_docs": None,
         "kv_docs": None}
    if case["layout"] == "packed":  # one projection [batch, token, (q, k, v), head, dim]
        x = _randn((b, tq, 3, h, d), g, case["type"])
        s["q"], s["k"], s["v"] = (x[:, :, i].transpose(1, 2) for i in range(3))
        s["out"] = torch.zeros((b, tq, h, d), device=_DEV, dtype=_TYPES[case["type"]]).transpose(1, 2)
    else:  # queries [batch, token, head, dim], cache [batch, head, token, dim]
        s["q"] = _randn((b, tq, h, d), g, case["type"]).transpose(1, 2)
        s["k"] = _randn((b, hk, tk, d), g, case["type"])
        s["v"] = _randn((b, hk, tk, d), g, case["type"])
        s["out"] = torch.zeros((b, tq, h, d), device=_DEV, dtype=_TYPES[case["type"]]).transpose(1, 2)
    s["q"] *= 1.5  # scores of trained models spread further than those of unit normals
    if case["ragged"]:
        rng = np.random.default_rng(seed)
        s["lens"] = torch.tensor(rng.permutation(_lens(case)).astype(np.int32), device=_DEV)
        if case["layout"] == "packed":  # padded lines: rows behind a line's end are not its own
            s["q_lens"] = s["lens"]
    if case["slopes"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=_DEV, dtype=torch.float32)
    if case["prefix"]:
        rng = np.random.default_rng(seed + 1)
        s["prefix"] = torch.tensor(rng.integers(case["prefix"] // 2, case["prefix"] + 1, size=b).astype(np.int32), device=_DEV)
    if case["docs"]:
        rng = np.random.default_rng(seed + 2)
        ids = np.zeros((b, tk), np.int32)
        for i in range(b):  # lines of about the same length, one after another
            cuts = (np.arange(1, case["docs"]) + rng.uniform(-0.3, 0.3, case["docs"] - 1)) * _doc_len(case)
            ids[i] = np.searchsorted(cuts, np.arange(tk), side="right")
        s["kv_docs"] = torch.tensor(ids, device=_DEV)
        s["q_docs"] = s["kv_docs"][:, tk - tq:].contiguous()
    return s


def _prepare_beam(case, g, seed):
    b, w, v = case["batch"], case["beams"], case["vocab"]
    logits = _randn((b, w, v), g, case["type"]) * 2
    scores = -torch.rand((b, w), generator=g, device=_DEV) * 8
    rng = np.random.default_rng(seed)
    done = torch.tensor((rng.random((b, w)) < case["done"]).astype(np.uint8), device=_DEV)
    kind = torch.float32 if case["type"] == "f32" else _TYPES[case["type"]]
    shape = (b * w, case["heads"], case["room"], case["dim"])
    states = [(torch.randn(shape, generator=g, device=_DEV, dtype=kind), torch.zeros(shape, device=_DEV, dtype=kind))
              for _ in range(2 * case["layers"])]
    new = lambda t: torch.zeros((b, w), device=_DEV, dtype=t)  # noqa: E731
    return {"case": case, "logits": logits, "scores": scores, "done": done, "states": states, "end": 2, "out_scores": new(torch.float32),
            "out_parents": new(torch.int32), "out_tokens": new(torch.int32), "out_done": new(torch.uint8)}


def _prepare_ctc(case, g, seed):
    n, t, v = case["lines"], case["steps"], case["classes"]
    logits = torch.randn((n, t, v), generator=g, device=_DEV, dtype=torch.float32) * 1.5
    # a recogniser's steps: most near certain of a class, the blank more often than not, some torn between two
    rng = np.random.default_rng(seed)
    hit = torch.tensor(np.where(rng.random((n, t, 1)) < 0.5, 0, rng.integers(0, v, (n, t, 1))), device=_DEV)
    logits.scatter_add_(2, hit, torch.tensor(rng.uniform(3, 14, (n, t, 1)).astype(np.float32), device=_DEV))
    two = torch.tensor(rng.integers(0, v, (n, t, 1)), device=_DEV)
    logits.scatter_add_(2, two, torch.tensor((rng.uniform(0, 10, (n, t, 1)) * (rng.random((n, t, 1)) < 0.3)).astype(np.float32), device=_DEV))
    logits = logits.to(_TYPES[case["type"]])
    lens = [t - (t * i) // (2 * n) for i in range(n)]
    p = case["paths"]
    return {"case": case, "logits": logits, "lens": torch.tensor(rng.permutation(lens).astype(np.int32), device=_DEV),
            "tokens": torch.zeros((n, p, t), device=_DEV, dtype=torch.int32), "lengths": torch.zeros((n, p), device=_DEV, dtype=torch.int32),
            "scores": torch.zeros((n, p), device=_DEV, dtype=torch.float32)}


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    return {"attention": _run_attention, "beam": _run_beam, "ctc": _run_ctc}[state["case"]["op"]](state)


def _run_attention(s):
    if own:
        _gpu.attention(s["q"], s["k"], s["v"], s["out"], scale=s["scale"], cap=s["case"]["cap"], slopes=s["slopes"],
                       causal=s["case"]["causal"], prefix=s["prefix"], q_lens=s["q_lens"], kv_lens=s["lens"],
                       q_docs=s["q_docs"], kv_docs=s["kv_docs"], stream=_stream())
        return s["out"]
    return _plain_attention(s)


def _seen(s, b0, b1):
    """Which keys each query of batches [b0, b1) sees, [batch, 1, query, key], and their distance."""
    c = s["case"]
    tq, tk = c["q_len"], c["kv_len"]
    kv_lens = s["lens"][b0:b1].long() if s["lens"] is not None else torch.full((b1 - b0,), tk, device=_DEV)
    q_lens = s["q_lens"][b0:b1].long() if s["q_lens"] is not None else torch.full((b1 - b0,), tq, device=_DEV)
    key = torch.arange(tk, device=_DEV)[None, None, None, :]
    row = torch.arange(tq, device=_DEV)[None, None, :, None]
    at = row + (kv_lens - q_lens)[:, None, None, None]  # a query's own position among the keys
    see = (key < kv_lens[:, None, None, None]) & (row < q_lens[:, None, None, None])
    if c["causal"]:
        before = key <= at
        if s["prefix"] is not None:
            before = before | (key < s["prefix"][b0:b1, None, None, None])
        see = see & before
    if s["q_docs"] is not None:
        see = see & (s["q_docs"][b0:b1, None, :, None] == s["kv_docs"][b0:b1, None, None, :])
    return see, (at - key).abs(), row < q_lens[:, None, None, None]


def _plain_attention(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros_like(s["out"])
    step = max(1, min(c["batch"], (1 << 31) // (c["heads"] * c["q_len"] * c["kv_len"])))
    for b0 in range(0, c["batch"], step):
        b1 = min(c["batch"], b0 + step)
        see, far, _ = _seen(s, b0, b1)
        kk = k[b0:b1].float().repeat_interleave(group, 1)
        vv = v[b0:b1].float().repeat_interleave(group, 1)
        x = torch.matmul(q[b0:b1].float(), kk.transpose(2, 3)) * s["scale"]
        if c["cap"]:
            x = c["cap"] * torch.tanh(x / c["cap"])
        if s["slopes"] is not None:
            x = x - s["slopes"][None, :, None, None] * far
        x = x.masked_fill(~see, -math.inf)
        m = x.amax(3, keepdim=True)
        e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        del x
        z = e.sum(3, keepdim=True)
        o = torch.matmul(e, vv) / torch.where(z == 0, torch.ones_like(z), z)
        out[b0:b1] = o.to(out.dtype)
    return out


def _run_beam(s):
    c = s["case"]
    if own:
        _gpu.beam_select(s["logits"], s["scores"], s["out_scores"], s["out_parents"], s["out_tokens"], end=s["end"],
                         finished=s["done"], out_finished=s["out_done"], stream=_stream())
        _gpu.beam_reorder(s["out_parents"], s["states"], axis=2, live=c["live"], stream=_stream())
        return {"scores": s["out_scores"], "parents": s["out_parents"], "tokens": s["out_tokens"], "done": s["out_done"],
                "states": [d for _, d in s["states"]]}
    b, w, v = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].double()
    m = x.amax(2, keepdim=True)
    logp = x - (m + torch.log(torch.exp(x - m).sum(2, keepdim=True)))
    cand = s["scores"].double()[:, :, None] + logp
    ended = torch.full_like(cand, -math.inf)
    ended[:, :, s["end"]] = s["scores"].double()
    cand = torch.where(s["done"][:, :, None] != 0, ended, cand).reshape(b, w * v)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    best, at = best[:, :w], at[:, :w]
    parents, tokens = at // v, at % v
    done = (s["done"].long().gather(1, parents) != 0) | (tokens == s["end"])
    rows = (torch.arange(b, device=_DEV)[:, None] * w + parents).reshape(-1)
    states = []
    for src, dst in s["states"]:
        dst[:, :, :c["live"]] = src[rows, :, :c["live"]]
        states.append(dst)
    return {"scores": best.float(), "parents": parents.int(), "tokens": tokens.int(), "done": done.to(torch.uint8), "states": states}


def _run_ctc(s):
    c = s["case"]
    if own:
        _gpu.ctc_beam(s["logits"], s["tokens"], s["lengths"], s["scores"], lens=s["lens"], width=c["width"], blank=0,
                      stream=_stream())
        return {"tokens": s["tokens"], "lengths": s["lengths"], "scores": s["scores"]}
    return _plain_ctc(s)


def _logadd(a, b):
    hi, lo = torch.maximum(a, b), torch.minimum(a, b)
    return torch.where(lo == -math.inf, hi, hi + torch.log1p(torch.exp(lo - hi)))


# Log masses are compared in steps of 2^-30, so that an order never hangs on the last bits of exp and log; the
# logits are multiples of that step too (those of 32 bits below 2^-6 are rounded to it).
_STEP = 2.0 ** 30


def _plain_ctc(s):
    c = s["case"]
    n, t, v, w, p = c["lines"], c["steps"], c["classes"], c["width"], c["paths"]
    inf = -math.inf
    text = torch.full((n, w, t), -1, device=_DEV, dtype=torch.long)
    size = torch.zeros((n, w), device=_DEV, dtype=torch.long)
    pb = torch.full((n, w), inf, device=_DEV, dtype=torch.float64)  # the mass of a text that ends in a blank
    pn = pb.clone()                                                # and of one that ends in its last class
    pb[:, 0] = 0.0
    norm = torch.zeros(n, device=_DEV, dtype=torch.float64)
    for i in range(t):
        x = torch.round(s["logits"][:, i].double() * _STEP) / _STEP
        m = x.amax(1, keepdim=True)
        lse = (m + torch.log(torch.exp(x - m).sum(1, keepdim=True)))[:, 0]
        total = _logadd(pb, pn)
        last = text.gather(2, (size - 1).clamp(min=0)[:, :, None])[:, :, 0]
        last = torch.where(size > 0, last, torch.full_like(last, -1))
        xl = torch.where(last >= 0, x.gather(1, last.clamp(min=0)), torch.full_like(pb, inf))
        stay_b = total + x[:, :1]
        stay_n = pn + xl
        ext = total[:, :, None] + x[:, None, :]  # a class behind a text
        again = (last[:, :, None] == torch.arange(v, device=_DEV)) & (last >= 0)[:, :, None]
        ext = torch.where(again, (pb[:, :, None] + x[:, None, :]), ext)
        ext[:, :, 0] = inf
        # a text o that grows by a class to a text j which is held already adds to that one
        alive = total > inf
        cut = text.scatter(2, (size - 1).clamp(min=0)[:, :, None], -1)
        same = (cut[:, None] == text[:, :, None]).all(3) & (size[:, None] == size[:, :, None] + 1)
        same = same & alive[:, :, None] & alive[:, None]
        at = last.clamp(min=0)[:, None].expand(n, w, w)
        gain = ext.gather(2, at)
        stay_n = _logadd(stay_n, torch.where(same, gain, torch.full_like(gain, inf)).amax(1))
        ext.scatter_reduce_(2, at, torch.where(same, torch.full_like(gain, inf), gain), "amin")
        stay = _logadd(stay_b, stay_n)
        every = torch.cat([stay, ext.reshape(n, w * v)], 1)
        at = torch.sort(torch.round(every * _STEP), dim=1, descending=True, stable=True)[1][:, :w]
        best = every.gather(1, at)
        grown = at >= w
        origin = torch.where(grown, (at - w) // v, at)
        cls = torch.where(grown, (at - w) % v, torch.full_like(at, -1))
        new_text = text.gather(1, origin[:, :, None].expand(n, w, t)).clone()
        new_size = size.gather(1, origin)
        new_text.scatter_(2, new_size.clamp(max=t - 1)[:, :, None],
                          torch.where(grown, cls, new_text.gather(2, new_size.clamp(max=t - 1)[:, :, None])[:, :, 0])[:, :, None])
        new_size = new_size + grown.long()
        new_b = torch.where(grown, torch.full_like(best, inf), stay_b.gather(1, origin))
        new_n = torch.where(grown, best, stay_n.gather(1, origin))
        on = (i < s["lens"].long())[:, None]
        text = torch.where(on[:, :, None], new_text, text)
        size = torch.where(on, new_size, size)
        pb, pn = torch.where(on, new_b, pb), torch.where(on, new_n, pn)
        norm = torch.where(on[:, 0], norm + lse, norm)
    score = _logadd(pb, pn) - norm[:, None]
    dead = score == inf
    size = torch.where(dead, torch.zeros_like(size), size)
    text = torch.where(dead[:, :, None], torch.full_like(text, -1), text)
    return {"tokens": text[:, :p].int(), "lengths": size[:, :p].int(), "scores": score[:, :p].float()}


# ---------------------------------------------------------------------------------------
# the least work
# ---------------------------------------------------------------------------------------
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("type")]
    if case["op"] == "attention":
        b, h, hk, tq, tk, d = (case[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
        lens = _lens(case)
        rows = sum(lens) if case["layout"] == "packed" and case["ragged"] else b * tq
        pairs = 0.0
        for n in lens:
            q = n if case["layout"] == "packed" and case["ragged"] else tq
            if case["docs"]:
                full = q * min(n, _doc_len(case))
                pairs += full / 2 if case["causal"] else full
            elif case["causal"]:
                lo = n - q  # keys before the first query
                tri = q * lo + q * (q + 1) / 2
                pre = min(0.75 * case["prefix"], n)
                more = max(0.0, pre - lo)
                pairs += tri + more * (more - 1) / 2 if more > 1 else tri
            else:
                pairs += q * n
        return {"bytes": size * d * (2 * rows * h + 2 * sum(lens) * hk), "flops": 4.0 * pairs * h * d}
    if case["op"] == "beam":
        rows = case["batch"] * case["beams"]
        state = 2 * case["layers"] * rows * case["heads"] * case["live"] * case["dim"] * size
        return {"bytes": rows * case["vocab"] * size + 2 * state + rows * 18, "flops": 4.0 * rows * case["vocab"]}
    steps = sum(case["steps"] - (case["steps"] * i) // (2 * case["lines"]) for i in range(case["lines"]))
    return {"bytes": steps * case["classes"] * size + case["lines"] * case["paths"] * (case["steps"] + 2) * 4,
            "flops": 4.0 * steps * case["classes"]}


# ---------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    return {"attention": _exact_attention, "beam": _exact_beam, "ctc": _exact_ctc}[case["op"]](case, seed)


def _exact_attention(case, seed):
    pairs = case["batch"] * case["heads"] * case["q_len"] * case["kv_len"]
    if pairs * (case["dim"] + 8) > 5e11:
        return None
    s = prepare(case, seed)
    out = torch.zeros(s["out"].shape, device=_DEV, dtype=torch.float64)
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    lens, q_lens, prefix, q_docs = (host(s[k]) for k in ("lens", "q_lens", "prefix", "q_docs"))
    ratio = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        nk = int(lens[b]) if lens is not None else case["kv_len"]
        nq = int(q_lens[b]) if q_lens is not None else case["q_len"]
        pos = torch.arange(nq, device=_DEV) + (nk - nq)
        key = torch.arange(nk, device=_DEV)
        hide = torch.zeros((nq, nk), dtype=torch.bool, device=_DEV)
        if case["causal"]:
            hide |= key[None] > pos[:, None]
            if prefix is not None:
                hide[:, :int(prefix[b])] = False
        if q_docs is not None:
            hide |= s["q_docs"][b, :nq, None] != s["kv_docs"][b, None, :nk]
        for h in range(case["heads"]):
            a = s["q"][b, h, :nq].double() @ s["k"][b, h // ratio, :nk].double().T
            a *= s["scale"]
            if case["cap"]:
                a = torch.tanh(a / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                a -= s["slopes"][h].double() * (pos[:, None] - key[None]).abs()
            a[hide] = -math.inf
            lse = torch.logsumexp(a, 1)
            prob = torch.exp(a - lse[:, None])
            prob[torch.isinf(lse)] = 0.0
            out[b, h, :nq] = prob @ s["v"][b, h // ratio, :nk].double()
    return out


def _exact_beam(case, seed):
    s = prepare(case, seed)
    b, w, v = case["batch"], case["beams"], case["vocab"]
    logits = s["logits"].double().cpu().numpy()
    scores = s["scores"].double().cpu().numpy()
    done = s["done"].cpu().numpy()
    out = {"scores": np.zeros((b, w)), "parents": np.zeros((b, w), np.int32), "tokens": np.zeros((b, w), np.int32), "done": np.zeros((b, w), np.uint8)}
    for i in range(b):
        found = []  # (score, beam, token) of the best of each beam, low places first where scores are the same
        for j in range(w):
            if done[i, j]:
                found.append((scores[i, j], j, s["end"]))
                continue
            x = logits[i, j]
            top = x.max()
            norm = top + math.log(np.exp(x - top).sum())
            floor = np.partition(x, v - min(v, w))[v - min(v, w)]
            found += [(scores[i, j] + (x[k] - norm), j, int(k)) for k in np.flatnonzero(x >= floor)]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        for r, (score, j, k) in enumerate(found[:w]):
            out["scores"][i, r], out["parents"][i, r], out["tokens"][i, r] = score, j, k
            out["done"][i, r] = bool(done[i, j]) or k == s["end"]
    rows = torch.tensor((np.arange(b)[:, None] * w + out["parents"]).reshape(-1), device=_DEV)
    out["states"] = []
    for src, dst in s["states"]:
        new = torch.zeros_like(dst)
        for r in range(b * w):
            new[r, :, :case["live"]] = src[int(rows[r]), :, :case["live"]]
        out["states"].append(new)
    return out


def _exact_ctc(case, seed):
    n, t, v, w, p = case["lines"], case["steps"], case["classes"], case["width"], case["paths"]
    if n * t * (3e-4 + w * (3e-5 + v * 6e-9)) > 12:
        return None
    s = prepare(case, seed)
    lens = s["lens"].cpu().numpy()
    tokens, lengths, scores = np.full((n, p, t), -1, np.int32), np.zeros((n, p), np.int32), np.full((n, p), -math.inf)
    add = lambda a, b: max(a, b) if min(a, b) == -math.inf else max(a, b) + math.log1p(math.exp(min(a, b) - max(a, b)))  # noqa: E731
    for i in range(n):
        x_all = np.rint(s["logits"][i].double().cpu().numpy() * _STEP) / _STEP
        held = [((), 0.0, -math.inf)]  # (text, mass ending in a blank, mass ending in its last class), best first
        norm = 0.0
        for j in range(int(lens[i])):
            x = x_all[j]
            top = x.max()
            norm += top + math.log(np.exp(x - top).sum())
            order = np.argsort(-x, kind="stable")[:w + 2]
            grow = {}  # text -> [mass ending in a blank, mass ending in its last class, place among the candidates]
            for at, (text, pb, pn) in enumerate(held):
                grow[text] = [add(pb, pn) + x[0], pn + x[text[-1]] if text else -math.inf, at]
            more = []
            for at, (text, pb, pn) in enumerate(held):
                classes = set(int(k) for k in order) | {o[0][-1] for o in held if o[0]}
                for k in classes:
                    if k == 0:
                        continue
                    mass = (pb if text and text[-1] == k else add(pb, pn)) + x[k]
                    new = text + (k,)
                    if new in grow:
                        grow[new][1] = add(grow[new][1], mass)
                    else:
                        more.append((new, -math.inf, mass, w + at * v + k))
            every = [(text, m[0], m[1], m[2]) for text, m in grow.items()] + more
            every = [(text, b, q, at, add(b, q)) for text, b, q, at in every]
            every = [e for e in every if e[4] > -math.inf]
            every.sort(key=lambda e: (-round(e[4] * _STEP), e[3]))
            held = [e[:3] for e in every[:w]]
        for r, (text, pb, pn) in enumerate(held[:p]):
            tokens[i, r, :len(text)] = text
            lengths[i, r] = len(text)
            scores[i, r] = add(pb, pn) - norm
    return {"tokens": tokens, "lengths": lengths, "scores": scores}
