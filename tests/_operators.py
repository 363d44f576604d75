"""The operators from their definitions in 64 bits (torch, on the CPU), for the tests of the kernels."""
import math

import numpy as np
import torch

STEP = 2.0 ** 30  # log masses of CTC beams are compared in multiples of 1 / STEP


def attention(q, k, v, scale, cap=0.0, slopes=None, causal=False, prefix=None, q_lens=None, kv_lens=None, q_docs=None,
              kv_docs=None):
    """(out, size, rows): the outputs, per row the sum of weight |value| (what errors of weights scale with), and which
    rows are written.  Unseen keys and values are cut away before any arithmetic."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    host = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    slopes, prefix, q_lens, kv_lens, q_docs, kv_docs = map(host, (slopes, prefix, q_lens, kv_lens, q_docs, kv_docs))
    B, H, TQ, D = q.shape
    HK, TK = k.shape[1], k.shape[2]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    rows = torch.zeros((B, H, TQ), dtype=torch.bool)
    for b in range(B):
        nk = TK if kv_lens is None else min(max(int(kv_lens[b]), 0), TK)
        nq = TQ if q_lens is None else min(max(int(q_lens[b]), 0), TQ)
        rows[b, :, :nq] = True
        key = torch.arange(nk)
        for i in range(nq):
            pos = nk - nq + i
            see = torch.ones(nk, dtype=torch.bool)
            if causal:
                see &= (key <= pos) | (key < (0 if prefix is None else int(prefix[b])))
            if q_docs is not None:
                see &= (kv_docs[b, :nk] == q_docs[b, i]) & (q_docs[b, i] >= 0)
            js = key[see]
            if len(js) == 0:
                continue
            kk = k[b][:, js].repeat_interleave(H // HK, 0)
            vv = v[b][:, js].repeat_interleave(H // HK, 0)
            s = torch.einsum("hjd,hd->hj", kk, q[b, :, i]) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - slopes.double()[:, None] * (pos - js).abs()
            w = torch.softmax(s, 1)
            out[b, :, i] = torch.einsum("hj,hjd->hd", w, vv)
            size[b, :, i] = torch.einsum("hj,hjd->hd", w, vv.abs())
    return out, size, rows


def beam_select(logits, scores, kout, end=-1, finished=None):
    """(scores, parents, tokens, finished) by sorting every candidate of each batch element."""
    x = logits.detach().cpu().double().numpy()
    sc = scores.detach().cpu().double().numpy()
    B, K, V = x.shape
    big = float(np.finfo(np.float32).max)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, big))
    sc = np.where(np.isnan(sc), -np.inf, np.minimum(sc, big))
    out = np.zeros((B, kout)), np.zeros((B, kout), np.int32), np.zeros((B, kout), np.int32), np.zeros((B, kout), np.uint8)
    for b in range(B):
        cand = np.full((K, V), -np.inf)
        for j in range(K):
            if finished is not None and finished[b, j]:
                cand[j, end] = sc[b, j]
                continue
            m = x[b, j].max()
            if m > -np.inf:
                cand[j] = sc[b, j] - (m + math.log(np.exp(x[b, j] - m).sum())) + x[b, j]
        order = np.argsort(-cand.reshape(-1), kind="stable")[:kout]
        out[0][b], out[1][b], out[2][b] = cand.reshape(-1)[order], order // V, order % V
        for r, o in enumerate(order):
            fin = finished is not None and bool(finished[b, o // V])
            out[3][b, r] = fin or (o % V == end)
    return out


def _add(a, b):
    hi, lo = max(a, b), min(a, b)
    return hi if lo == -math.inf else hi + math.log1p(math.exp(lo - hi))


def ctc_beam(logits, lens, width, blank, paths):
    """(tokens, lengths, scores) by prefix beam search over texts as tuples, every class tried for every beam."""
    x_all = logits.detach().cpu().double().numpy()
    big = float(np.finfo(np.float32).max)
    x_all = np.where(np.isnan(x_all), -np.inf, np.minimum(x_all, big))
    with np.errstate(over="ignore"):
        x_all = np.where(np.abs(x_all) < 1, np.rint(x_all * STEP) / STEP, x_all)
    N, T, V = x_all.shape
    tokens, lengths, scores = np.full((N, paths, T), -1, np.int32), np.zeros((N, paths), np.int32), np.full((N, paths), -np.inf)
    for n in range(N):
        held, norm = [((), 0.0, -math.inf)], 0.0
        for t in range(T if lens is None else min(max(int(lens[n]), 0), T)):
            x = x_all[n, t]
            m = x.max()
            norm += m + math.log(np.exp(x - m).sum()) if m > -np.inf else -math.inf
            keep = {s: [_add(pb, pn) + x[blank], pn + x[s[-1]] if s else -math.inf, i] for i, (s, pb, pn) in enumerate(held)}
            more = []
            for i, (s, pb, pn) in enumerate(held):
                for c in range(V):
                    if c == blank:
                        continue
                    mass = (pb if s and s[-1] == c else _add(pb, pn)) + x[c]
                    if s + (c,) in keep:
                        keep[s + (c,)][1] = _add(keep[s + (c,)][1], mass)
                    else:
                        more.append((s + (c,), -math.inf, mass, width + i * V + c))
            every = [(s, a, b, p, _add(a, b)) for s, (a, b, p) in keep.items()] + [(s, a, b, p, b) for s, a, b, p in more]
            every = sorted((e for e in every if e[4] > -math.inf), key=lambda e: (-round(e[4] * STEP), e[3]))
            held = [e[:3] for e in every[:width]]
        for r, (s, pb, pn) in enumerate(held[:paths]):
            tokens[n, r, :len(s)] = s
            lengths[n, r] = len(s)
            scores[n, r] = _add(pb, pn) - norm
    return tokens, lengths, scores
