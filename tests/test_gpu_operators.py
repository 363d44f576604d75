"""The operators on device tensors against their definitions in 64 bits (tests/_operators.py).

Tolerances, derived before the first run.  u = finfo(type).eps / 2 is the rounding of a type, U = 2^-24 that of 32 bits.
  attention: a score is off by at most (dim + 8) U times the sum of its products' magnitudes (an fp32 dot product, its scale
    and cap), plus 4 U of the bias and 8 U of the cap's range; a weight's relative error is twice that (its own and the
    maximum's) plus 2^-20 for the exponential, and keys U for the sums; in 16 bits the weights are rounded once to the
    values' type (u, or 2^-25 absolute in fp16's subnormals) and the capped score's fast tanh is off by 2^-18 of the cap.
    The output is off by that times sum w |v|, and by its own rounding u |out| (2^-25 absolute in fp16).
  scores of beams: rounded once from 64 bits, log-sum-exps from 32-bit exponentials: 2^-24 |score| + 2^-20.
  tokens, parents, lengths: equal.
"""
import math

import numpy as np
import pytest
import torch

import _operators as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def randn(shape, type, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[type])


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attention_check(gpu, q, k, v, out=None, stream="torch", scale=None, **kw):
    """Runs the kernel and holds it to the definition; rows that are not written must keep what they held."""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    before = out.clone()
    st = torch.cuda.current_stream().cuda_stream if stream == "torch" else stream
    gpu.attention(q, k, v, out, scale=scale, stream=st, **kw)
    torch.cuda.synchronize()
    attention_compare(out, before, q, k, v, scale, **kw)
    return out


def attention_compare(out, before, q, k, v, scale, **kw):
    want, size, rows = ref.attention(q, k, v, scale, **kw)
    got = out.cpu().double()
    assert torch.equal(out.cpu()[~rows], before.cpu()[~rows])
    # unseen keys may hold anything: magnitudes over the finite ones bound those that count
    fin = lambda t: torch.nan_to_num(t.cpu().double(), 0, 0, 0)  # noqa: E731
    G = q.shape[1] // k.shape[1]
    mag = scale * float(torch.einsum("bhqd,bhkd->bhqk", fin(q).abs(), fin(k).abs().repeat_interleave(G, 1)).max()) if k.shape[2] else 0
    far = k.shape[2] + q.shape[2]
    slopes = kw.get("slopes")
    bias = float(slopes.abs().max()) * far if slopes is not None else 0.0
    cap = kw.get("cap", 0.0)
    es = (q.shape[3] + 8) * U * abs(mag) + 4 * U * bias + 8 * U * cap
    half = q.dtype != torch.float32
    u = torch.finfo(q.dtype).eps / 2
    if half:
        es += cap * 2.0 ** -18
    ew = 2 * es + 2.0 ** -20 + k.shape[2] * U + (u if half else 0)
    tol = size * ew + want.abs() * u
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (1 + k.shape[2] * fin(v).abs().max())
    tol = tol + 1e-30
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got[rows]), nan[rows])
    ok = rows[..., None].expand_as(got) & ~nan
    bad = (got - want).abs() > tol
    assert not (bad & ok).any(), f"{int((bad & ok).sum())} of {int(ok.sum())} off, worst {float(((got - want).abs() / tol)[ok].max()):.2f} of the tolerance"


def qkv(B, H, HK, TQ, TK, D, type, seed=0):
    return randn((B, H, TQ, D), type, seed, 1.5), randn((B, HK, TK, D), type, seed + 1), randn((B, HK, TK, D), type, seed + 2)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B, H, HK, TQ, TK, D", [
    (1, 1, 1, 1, 1, 1), (2, 3, 3, 5, 5, 15), (3, 8, 8, 40, 40, 15), (2, 4, 2, 33, 65, 64), (1, 2, 1, 130, 257, 128),
    (1, 6, 2, 100, 64, 72), (1, 2, 2, 129, 300, 40), (1, 1, 1, 70, 90, 256), (1, 7, 1, 257, 257, 96), (2, 2, 2, 1, 33, 31),
    (1, 2, 2, 300, 20, 16), (1, 5, 1, 260, 520, 64),
])
def test_attention(gpu, type, B, H, HK, TQ, TK, D):
    attention_check(gpu, *qkv(B, H, HK, TQ, TK, D, type))


MASKS = ["causal", "prefix", "docs", "causal docs", "lens", "causal lens", "cap", "slopes", "cap slopes causal lens", "padding docs",
         "all"]


def masks(kind, B, H, TQ, TK, seed=5):
    rng = np.random.default_rng(seed)
    kw = {}
    if "causal" in kind or kind in ("prefix", "all"):
        kw["causal"] = True
    if kind in ("prefix", "all"):
        kw["prefix"] = i32(rng.integers(-2, TK + 3, B))
    if "docs" in kind or kind == "all":
        ids = np.sort(rng.integers(0, 4, (B, TK)), 1).astype(np.int32)
        if "padding" in kind or kind == "all":
            ids[:, rng.integers(0, TK, max(1, TK // 5))] = -1
        kw["kv_docs"] = torch.tensor(ids, device="cuda")
        qd = np.stack([np.resize(ids[b][max(0, TK - TQ):], TQ) for b in range(B)])
        if "padding" in kind or kind == "all":
            qd[:, ::3] = -1
            qd[:, 1::7] = 9  # an id that no key has
        kw["q_docs"] = torch.tensor(qd.astype(np.int32), device="cuda")
    if "lens" in kind or kind == "all":
        kw["kv_lens"] = i32(np.concatenate([[0], rng.integers(1, TK + 2, B)])[:B] if B > 1 else rng.integers(1, TK + 1, B))
        kw["q_lens"] = i32(rng.integers(0, TQ + 2, B))
    if "cap" in kind or kind == "all":
        kw["cap"] = 4.0
    if "slopes" in kind or kind == "all":
        kw["slopes"] = torch.tensor(rng.uniform(-0.02, 0.5, H).astype(np.float32), device="cuda")
    return kw


@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("type, D, TQ, TK", [("f32", 15, 50, 70), ("bf16", 64, 150, 300), ("f16", 128, 280, 280), ("f16", 20, 3, 90),
                                             ("bf16", 128, 1, 700), ("f32", 64, 2, 400), ("bf16", 32, 300, 130)])
def test_attention_masks(gpu, kind, type, D, TQ, TK):
    B, H, HK = 3, 4, 2
    attention_check(gpu, *qkv(B, H, HK, TQ, TK, D, type, 11), **masks(kind, B, H, TQ, TK))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("TQ, TK, D", [(1, 200, 64), (64, 200, 15), (200, 300, 64), (260, 400, 128)])
def test_attention_leaves_what_is_masked_alone(gpu, type, TQ, TK, D):
    """NaN and infinities behind every kind of mask: behind the keys' end, a causal mask and other documents."""
    B, H = 2, 2
    q, k, v = qkv(B, H, H, TQ, TK, D, type, 21)
    kv_lens = i32([TK - 37, TK - 5])
    for b, n in enumerate(kv_lens.tolist()):
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
    attention_check(gpu, q, k, v, kv_lens=kv_lens)
    attention_check(gpu, q, k, v, kv_lens=kv_lens, causal=True)
    # a key that the later queries see and the earlier ones do not
    if TQ > 1:
        at = int(kv_lens[0]) - TQ // 2
        v[0, 0, at, D // 2] = float("nan")
        v[1, 1, at, 0] = -float("inf")
        k[1, 0, at] = float("inf")
        q[1, 0] = q[1, 0].abs()  # scores of +inf: NaN weights, in both
        attention_check(gpu, q, k, v, kv_lens=kv_lens, causal=True)
    docs = torch.zeros((B, TK), dtype=torch.int32, device="cuda")
    docs[:, 10:13] = 5
    k[:, :, 11], v[:, :, 12], v[:, :, 10, 0] = float("nan"), float("nan"), float("inf")
    attention_check(gpu, q, k, v, kv_lens=kv_lens, q_docs=torch.zeros((B, TQ), dtype=torch.int32, device="cuda"), kv_docs=docs,
                    causal=False) if TQ == 1 else attention_check(gpu, q[:, :, :3], k, v, kv_lens=kv_lens, kv_docs=docs,
                                                                  q_docs=torch.zeros((B, 3), dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("TQ", [1, 40, 200])
def test_attention_of_scores_that_are_no_number(gpu, type, TQ):
    """Capped scores: an infinite product is the cap, a NaN in sight is a NaN in the result, one behind a mask is not."""
    q, k, v = qkv(1, 2, 2, TQ, 300, 64, type, 95)
    q = q.abs() + 0.1
    k[0, 0, 150] = float("nan")
    k[0, 1, 20] = float("inf")
    docs = torch.zeros((1, 300), dtype=torch.int32, device="cuda")
    docs[0, 150] = 1
    same = torch.zeros((1, TQ), dtype=torch.int32, device="cuda")
    out = attention_check(gpu, q, k, v, cap=5.0)
    assert torch.isnan(out[0, 0]).all() and torch.isfinite(out[0, 1]).all()
    out = attention_check(gpu, q, k, v, cap=5.0, q_docs=same, kv_docs=docs)
    assert torch.isfinite(out).all()
    attention_check(gpu, q, k, v, scale=-0.2)
    attention_check(gpu, q, k[:, :, 21:150], v[:, :, 21:150], scale=0.0)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [30.0, -30.0, 1000.0, -1000.0])
def test_attention_of_large_scores(gpu, type, value):
    """Scores far from zero and far apart: the running maximum decides, nothing overflows."""
    q, k, v = qkv(1, 2, 1, 150, 200, 64, type, 31)
    q.fill_(1.0)
    k.zero_()
    k[..., 0] = torch.linspace(value, value / 2, 200, device="cuda").to(k.dtype)
    attention_check(gpu, q, k, v, scale=1.0)
    attention_check(gpu, q[:, :, :1], k, v, scale=1.0)
    attention_check(gpu, q, k.flip(2), v, scale=1.0, causal=True)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("D", [15, 64])
def test_attention_layouts(gpu, type, D):
    """Packed projections, broadcast keys, padded rows, odd offsets, an output between other values."""
    B, T, H = 2, 140, 4
    x = randn((B, T, 3, H, D), type, 41)
    q, k, v = (x[:, :, i].transpose(1, 2) for i in range(3))
    out = torch.full((B, T, H + 1, D + 3), 5.0, dtype=x.dtype, device="cuda")
    view = out[:, :, 1:, 1:D + 1].transpose(1, 2)
    attention_check(gpu, q, k, v, out=view)
    assert (out[:, :, 0] == 5).all() and (out[..., 0] == 5).all() and (out[..., D + 1:] == 5).all()
    pad = randn((B, H, T, D + 1), type, 42)
    attention_check(gpu, pad[..., 1:], k, pad[..., :D])
    one = randn((1, 1, T, D), type, 43).expand(B, H, T, D)
    attention_check(gpu, q, one, one)
    attention_check(gpu, q[:, :, :1], one, one)


def test_attention_of_nothing(gpu):
    for type in ("f16", "f32"):
        for TQ in (1, 3, 40, 200):
            q, k, v = qkv(2, 2, 2, TQ, 0, 16, type)
            out = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
            gpu.attention(q, k, v, out, stream=0)
            torch.cuda.synchronize()
            assert (out == 0).all()
    gpu.attention(q[:0], k[:0], v[:0], out[:0])
    gpu.attention(q[:, :, :0], k, v, out[:, :, :0])


@pytest.mark.parametrize("type, TQ, TK, D", [("bf16", 1, 3000, 128), ("f16", 4, 5000, 64), ("f32", 1, 4097, 32), ("bf16", 300, 2000, 64)])
def test_attention_over_long_caches(gpu, type, TQ, TK, D):
    B, H, HK = 2, 8, 2
    q, k, v = qkv(B, H, HK, TQ, TK, D, type, 51)
    attention_check(gpu, q, k, v, causal=True, kv_lens=i32([TK, TK // 2 + 1]))
    attention_check(gpu, q, k, v, causal=True, cap=20.0, slopes=torch.full((H,), 0.01, device="cuda"), kv_lens=i32([TQ, TK - 3]))


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [4, 8, 12, 40, 72, 80, 100, 128, 136])
@pytest.mark.parametrize("H, HK, TQ", [(3, 3, 1), (2, 1, 1), (6, 2, 1), (8, 1, 1), (4, 1, 5), (20, 1, 3), (70, 1, 1)])
def test_attention_of_few_rows(gpu, type, D, H, HK, TQ):
    """Every count of rows that share a key head, every way that a head's dimension ends within a thread's words."""
    q, k, v = qkv(2, H, HK, TQ, 330, D, type, 65 + D)
    attention_check(gpu, q, k, v, causal=True, kv_lens=i32([330, 77]))


@pytest.mark.parametrize("type, TQ, TK, D", [("f16", 20, 2500, 128), ("bf16", 150, 3300, 72), ("f16", 260, 1700, 64), ("bf16", 100, 900, 128)])
@pytest.mark.parametrize("kind", ["", "prefix", "docs", "causal lens", "all"])
def test_attention_with_keys_shared_out(gpu, kind, type, TQ, TK, D):
    """Few query tiles over many keys: the blocks of a cluster each take some of the key tiles (none, for short rows)."""
    B, H, HK = 2, 2, 1
    q, k, v = qkv(B, H, HK, TQ, TK, D, type, 55)
    attention_check(gpu, q, k, v, **masks(kind, B, H, TQ, TK))
    v[0, 0, TK // 3] = float("inf")
    k[1, 0, TK // 2, 0] = float("nan")
    if kind == "causal lens":
        attention_check(gpu, q, k, v, causal=True, kv_lens=i32([TK // 3, TK // 2 + TQ // 2]))


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_attention_offsets_beyond_32_bits(gpu, type):
    """A head that starts more than 2^32 elements (f16) or bytes (f32) into the cache."""
    D, TK = 64, 256
    rows = (1 << 32) // D + TK if type == "f16" else (1 << 30) // D + TK
    cache = torch.zeros((rows, D), dtype=TYPES[type], device="cuda")
    far = cache[-TK:]
    far.copy_(randn((TK, D), type, 61))
    q = randn((1, 1, 200, D), type, 62)
    stride = (rows - TK) * D
    k = torch.as_strided(cache, (2, 1, TK, D), (stride, 0, D, 1))
    attention_check(gpu, q.expand(2, 1, 200, D), k, k)
    attention_check(gpu, q[:, :, :1].expand(2, 1, 1, D), k, k)


def test_attention_streams_and_graphs(gpu):
    """On a side stream and the context's own, captured twice and replayed in turn on new values."""
    import wocr
    a, b = (qkv(2, 4, 2, 140, 300, 64, "bf16", s) for s in (71, 72))
    t1, t2 = (qkv(2, 4, 2, 1, 300, 64, "bf16", s) for s in (73, 74))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_check(gpu, *a)
    torch.cuda.synchronize()
    attention_check(gpu, *a, stream=None)
    graphs, outs = [], []
    for args in (a, t1):
        out = torch.zeros_like(args[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gpu.attention(*args, out, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        outs.append(out)
    for args, new in ((a, b), (t1, t2)):
        for x, y in zip(args, new):
            x.copy_(y)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for args, out in ((a, outs[0]), (t1, outs[1])):
        attention_compare(out, out, *args, 64 ** -0.5)
    assert torch.cuda.current_device() == gpu.device
    # an allocation that is no torch tensor
    q, k, v = a
    wrap = lambda t: wocr.DeviceArray(t.data_ptr(), "bfloat16", t.shape, t.stride())  # noqa: E731
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    gpu.attention(wrap(q), wrap(k), wrap(v), wrap(out))
    gpu.submit_wait()
    attention_compare(out, out, q, k, v, 64 ** -0.5)


def test_attention_gives_the_same_twice(gpu):
    for TQ in (1, 200):
        q, k, v = qkv(2, 8, 2, TQ, 1500, 64, "bf16", 81)
        outs = [torch.zeros_like(q) for _ in range(3)]
        for o in outs:
            gpu.attention(q, k, v, o, stream=0, causal=True)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- beam search ---------------------------------------------------------------------------
def select(gpu, logits, scores, kout, end=-1, finished=None, stream=0):
    B = logits.shape[0]
    o = [torch.zeros((B, kout), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    gpu.beam_select(logits, scores, o[0], o[1], o[2], end=end, finished=finished, out_finished=o[3], stream=stream)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in o]


def select_check(gpu, logits, scores, kout, end=-1, finished=None):
    got = select(gpu, logits, scores, kout, end, finished)
    want = ref.beam_select(logits, scores, kout, end, finished.cpu().numpy() if finished is not None else None)
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all() and (got[3] == want[3]).all()
    fin = np.isfinite(want[0])
    assert (np.isneginf(got[0]) == ~fin).all()
    assert (np.abs(got[0][fin] - want[0][fin]) <= 2.0 ** -24 * np.abs(want[0][fin]) + 2.0 ** -20).all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B, K, V, M", [(1, 1, 1, 1), (1, 1, 40, 32), (3, 4, 97, 4), (2, 32, 97, 32), (2, 8, 18709, 8), (1, 3, 151, 7),
                                        (5, 2, 5001, 3), (1, 32, 4099, 32), (300, 2, 65, 2), (1, 2, 200003, 4), (1, 32, 70001, 5)])
def test_beam_select(gpu, type, B, K, V, M):
    logits = randn((B, K, V), type, 100 + V, 2.0)
    scores = -torch.rand((B, K), generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") * 6
    select_check(gpu, logits, scores, M)
    fin = torch.tensor(np.random.default_rng(V).random((B, K)) < 0.4, device="cuda").to(torch.uint8)
    select_check(gpu, logits, scores, M, end=V // 2, finished=fin)


@pytest.mark.parametrize("B, K, V, M", [(2, 4, 97, 4), (1, 4, 9000, 8), (1, 8, 40000, 32)])
def test_beam_select_ties_and_masks(gpu, B, K, V, M):
    """Equal logits everywhere, sorted rows (all of the best in one block's slice), masked classes, first steps of a search."""
    scores = torch.zeros((B, K), device="cuda")
    flat = torch.zeros((B, K, V), device="cuda")
    select_check(gpu, flat, scores, M)
    select_check(gpu, flat.half(), scores - 3, M, end=0)
    rise = torch.arange(V, device="cuda", dtype=torch.float32).expand(B, K, V).contiguous() * 2.0 ** -10
    select_check(gpu, rise, scores, M)
    select_check(gpu, rise.flip(2).contiguous(), scores, M)
    select_check(gpu, (rise * 2.0 ** -8).bfloat16(), scores, M)
    first = scores.clone()
    first[:, 1:] = -math.inf  # one beam alive
    x = randn((B, K, V), "f32", 7)
    select_check(gpu, x, first, M)
    x[:, :, 3:] = -math.inf   # three classes left
    select_check(gpu, x, first, M)
    x[:, 0] = -math.inf       # and none of the first beam's
    select_check(gpu, x, scores, M)
    select_check(gpu, torch.full_like(x, -math.inf), scores, M)
    y = randn((B, K, V), "f32", 8)
    y[:, :, ::5] = float("nan")
    y[:, 1, 2] = torch.finfo(torch.float32).min
    select_check(gpu, y, scores, M)
    s = scores.clone()
    s[:, 0] = float("nan")
    select_check(gpu, y, s, M)
    every = torch.ones((B, K), dtype=torch.uint8, device="cuda")
    if M <= K:
        select_check(gpu, y, torch.linspace(-3, -1, K, device="cuda").expand(B, K).contiguous(), M, end=5, finished=every)


def test_beam_select_one_thread_holds_the_best(gpu):
    """Every good candidate 256 tokens from the next: one thread's, far more than its share."""
    x = torch.zeros((1, 16, 60000), device="cuda")
    x[:, :, 5::256] = torch.arange(235, device="cuda") * 2.0 ** -6 + 1
    select_check(gpu, x, torch.zeros((1, 16), device="cuda"), 32)
    x[:, :, 5::256] = 1.0
    select_check(gpu, x, torch.zeros((1, 16), device="cuda"), 32)
    # scores that drown the logits in 32 bits, not in 64
    select_check(gpu, randn((2, 4, 3000), "f32", 3, 1e-3), torch.full((2, 4), -4000.0, device="cuda"), 8)


def test_beam_select_strides_in_place_and_graph(gpu):
    B, K, V = 3, 4, 500
    wide = randn((B, K + 1, 2 * V + 3), "bf16", 9)
    logits = wide[:, 1:, 3:V + 3]
    scores = torch.linspace(-2, 0, B * K, device="cuda").reshape(B, K).contiguous()
    fin = torch.zeros((B, K), dtype=torch.uint8, device="cuda")
    fin[0, 1] = 1
    select_check(gpu, logits, scores, K, end=4, finished=fin)
    want = ref.beam_select(logits, scores, K, 4, fin.cpu().numpy())
    s, f = scores.clone(), fin.clone()
    par, tok = (torch.zeros((B, K), dtype=torch.int32, device="cuda") for _ in range(2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gpu.beam_select(logits, s, s, par, tok, end=4, finished=f, out_finished=f, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        s.copy_(scores)
        f.copy_(fin)
        g.replay()
        torch.cuda.synchronize()
        assert (par.cpu().numpy() == want[1]).all() and (tok.cpu().numpy() == want[2]).all() and (f.cpu().numpy() == want[3]).all()
        assert np.allclose(s.cpu().numpy(), want[0], rtol=2.0 ** -22, atol=2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("shape, axis, live", [((4, 9, 16), 2, 5), ((4, 9, 16), 0, None), ((3, 7, 5), 2, 7), ((3, 7, 5), 1, 2), ((33,), 0, None),
                                               ((2, 8, 3), 2, 0), ((1, 300, 64), 2, 299)])
def test_beam_reorder(gpu, dtype, shape, axis, live):
    B, N, M = 3, 4, 5
    rng = np.random.default_rng(1)
    par = rng.integers(0, N, (B, M)).astype(np.int32)
    par[1, 2], par[2, 0] = -1, N  # no such beams
    states = []
    for i in range(3):
        src = torch.randint(0, 200, (B * N,) + shape, device="cuda").to(dtype)
        dst = torch.full((B * M,) + shape, 77, device="cuda").to(dtype)
        states.append((src, dst))
    # one that starts at an odd place of a larger allocation
    raw = torch.randint(0, 200, (B * N * int(np.prod(shape)) + 1,), device="cuda").to(dtype)
    states.append((raw[1:].reshape((B * N,) + shape), torch.full((B * M,) + shape, 77, device="cuda").to(dtype)))
    want = []
    for src, dst in states:
        w = dst.clone()
        for b in range(B):
            for j in range(M):
                if 0 <= par[b, j] < N:
                    cut = (slice(None),) * (axis - 1) + (slice(0, live),) if axis and live is not None else ()
                    w[b * M + j][cut] = src[b * N + int(par[b, j])][cut]
        want.append(w)
    gpu.beam_reorder(torch.tensor(par, device="cuda"), states, axis=axis, live=live, stream=0)
    torch.cuda.synchronize()
    for (_, dst), w in zip(states, want):
        assert torch.equal(dst, w)


def test_beam_reorder_of_many(gpu):
    """More states than a launch takes, more rows than a grid's second dimension."""
    par = i32(np.random.default_rng(2).integers(0, 3, (2, 3)))
    states = [(torch.randn((6, 10 + i), device="cuda"), torch.zeros((6, 10 + i), device="cuda")) for i in range(130)]
    gpu.beam_reorder(par, states, stream=0)
    rows = (torch.arange(2, device="cuda")[:, None] * 3 + par).reshape(-1)
    for src, dst in states:
        assert torch.equal(dst, src[rows])
    B, N = 3000, 31
    par = torch.randint(0, N, (B, N), device="cuda", dtype=torch.int32)
    src = torch.randn((B * N, 3), device="cuda")
    dst = torch.zeros_like(src)
    gpu.beam_reorder(par, [(src, dst)], stream=0)
    assert torch.equal(dst, src[(torch.arange(B, device="cuda")[:, None] * N + par).reshape(-1)])


# ---- CTC -----------------------------------------------------------------------------------
def search(gpu, logits, lens, width, blank, paths, stream=0):
    n, t, _ = logits.shape
    o = (torch.full((n, paths, t), 99, dtype=torch.int32, device="cuda"), torch.full((n, paths), 99, dtype=torch.int32, device="cuda"),
         torch.zeros((n, paths), device="cuda"))
    gpu.ctc_beam(logits, *o, lens=lens, width=width, blank=blank, stream=stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in o]


def search_check(gpu, logits, width, lens=None, blank=0, paths=None):
    paths = paths or width
    got = search(gpu, logits, lens, width, blank, paths)
    search_compare(got, logits, lens, width, blank, paths)


def search_compare(got, logits, lens, width, blank, paths):
    want = ref.ctc_beam(logits, lens.cpu().numpy() if lens is not None else None, width, blank, paths)
    assert (got[1] == want[1]).all() and (got[0] == want[0]).all()
    fin = np.isfinite(want[2])
    assert (np.isneginf(got[2]) == ~fin).all()
    # a log-sum-exp per step from 32-bit exponentials, each off by less than 2^-20
    assert (np.abs(got[2][fin] - want[2][fin]) <= 2.0 ** -24 * np.abs(want[2][fin]) + logits.shape[1] * 2.0 ** -20).all()


def peaky(n, t, v, type, seed):
    """Steps near certain of a class, the blank more often than not."""
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(n, t, v)) * 1.5
    hit = np.where(rng.random((n, t)) < 0.5, 0, rng.integers(0, v, (n, t)))
    np.put_along_axis(x, hit[..., None], np.take_along_axis(x, hit[..., None], 2) + rng.uniform(1, 10, (n, t, 1)), 2)
    return torch.tensor(x.astype(np.float32), device="cuda").to(TYPES[type])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, t, v, width", [(1, 1, 1, 1), (1, 1, 2, 4), (2, 12, 3, 31), (3, 30, 12, 8), (2, 70, 40, 5), (1, 9, 300, 16),
                                            (2, 5, 2000, 31), (1, 130, 5, 3)])
def test_ctc_beam(gpu, type, n, t, v, width):
    search_check(gpu, peaky(n, t, v, type, n + t + v), width)
    lens = i32(np.random.default_rng(t).integers(0, t + 2, n))
    search_check(gpu, peaky(n, t, v, type, 5), width, lens=lens, blank=v - 1, paths=max(1, width // 2))


def test_ctc_beam_repeats_and_merges(gpu):
    """Two classes and wide beams: texts with repeated classes, reached from several others at once."""
    x = randn((4, 25, 3), "f32", 1, 0.7)
    search_check(gpu, x, 20)
    search_check(gpu, x.bfloat16(), 20)
    search_check(gpu, torch.zeros_like(x), 20)  # every alignment alike: ties all the way
    search_check(gpu, torch.zeros((2, 6, 700), device="cuda"), 12)
    search_check(gpu, randn((2, 20, 4), "bf16", 3, 4.0).round(), 15)


def test_ctc_beam_of_masked_and_odd_logits(gpu):
    x = peaky(3, 14, 50, "f32", 8)
    x[:, :, 20:] = -math.inf
    search_check(gpu, x, 8)
    x[:, :, 7] = float("nan")
    search_check(gpu, x, 8)
    x[:, :, 5] = -1e9
    x[1, 3] = 2.0 ** -9 * torch.arange(50, device="cuda")
    x[1, 4] = 2.0 ** -33 * torch.arange(50, device="cuda")
    search_check(gpu, x, 8)
    x[1, 5] = -math.inf  # a step that allows nothing
    search_check(gpu, x, 8)
    search_check(gpu, peaky(2, 14, 50, "f32", 9) * 1e4, 8)
    lens = i32([0, -3])
    search_check(gpu, peaky(2, 6, 20, "f32", 9), 3, lens=lens)
    empty = search(gpu, torch.zeros((2, 0, 5), device="cuda"), None, 3, 0, 2)
    assert (empty[1] == 0).all() and (empty[2][:, 0] == 0).all() and np.isneginf(empty[2][:, 1]).all()


@pytest.mark.parametrize("type, v", [("f32", 18709), ("bf16", 18709), ("f32", 70001), ("f16", 6000)])
def test_ctc_beam_over_dictionaries(gpu, type, v):
    x = peaky(2, 4, v, type, v)
    search_check(gpu, x, 4)
    rise = (torch.arange(v, device="cuda") * 2.0 ** -10).expand(1, 2, v).to(TYPES[type]).contiguous()
    search_check(gpu, rise, 4)
    one = torch.zeros((1, 2, v), device="cuda")
    one[:, :, 9::256] = torch.arange(len(range(9, v, 256)), device="cuda") * 2.0 ** -6 + 1  # all in one thread's hands
    search_check(gpu, one.to(TYPES[type]), 5)


def test_ctc_beam_strides_streams_and_graphs(gpu):
    """Two captured calls share nothing: replayed in turn on new logits, beside a call on another stream."""
    wide = peaky(3, 20, 45, "f32", 4)
    search_check(gpu, wide[:, ::2, 3:40], 6)
    xs = [peaky(3, 20, 30, "f32", s) for s in (1, 2)]
    outs, graphs = [], []
    for x in xs:
        o = (torch.zeros((3, 4, 20), dtype=torch.int32, device="cuda"), torch.zeros((3, 4), dtype=torch.int32, device="cuda"),
             torch.zeros((3, 4), device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gpu.ctc_beam(x, *o, width=6, stream=torch.cuda.current_stream().cuda_stream)
        outs.append(o)
        graphs.append(g)
    for s, x in zip((5, 6), xs):
        x.copy_(peaky(3, 20, 30, "f32", s))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    third = peaky(3, 20, 30, "f32", 7)
    o3 = [torch.zeros_like(t) for t in outs[0]]
    for _ in range(3):
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            gpu.ctc_beam(third, *o3, width=6, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for x, o in zip(xs + [third], outs + [o3]):
        search_compare([t.cpu().numpy() for t in o], x, None, 6, 0, 4)


# ---- together ------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_a_decoder_with_beams(gpu, type):
    """A decoder over a line's features: every step attends over the cache, selects and puts the cache in the beams' order;
    the same texts come out when each step attends over the whole of each beam's own text again."""
    B, K, H, D, V, F, STEPS = 2, 3, 4, 16, 30, 11, 6
    t = TYPES[type]
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    emb, wq, wk, wv, wo = rnd(V, H * D), rnd(H * D, H * D) / 8, rnd(H * D, H * D) / 8, rnd(H * D, H * D) / 8, rnd(H * D, V) / 2
    feats = rnd(B, F, H * D)
    S = F + STEPS
    heads = lambda x: x.reshape(x.shape[0], -1, H, D).transpose(1, 2)  # noqa: E731
    cache = [torch.full((B * K, H, S, D), float("nan"), device="cuda", dtype=t) for _ in range(4)]
    for c, w in zip(cache[:2], (wk, wv)):
        c[:, :, :F] = heads(feats @ w).to(t).repeat_interleave(K, 0)
    scores = torch.full((B, K), -math.inf, device="cuda")
    scores[:, 0] = 0
    done = torch.zeros((B, K), dtype=torch.uint8, device="cuda")
    par, tok = (torch.zeros((B, K), dtype=torch.int32, device="cuda") for _ in range(2))
    texts = [[[0]] * K for _ in range(B)]
    st = torch.cuda.current_stream().cuda_stream
    for i in range(STEPS):
        x = emb[tok.reshape(-1).long()]
        cache[0][:, :, F + i] = (x @ wk).reshape(B * K, H, D).to(t)
        cache[1][:, :, F + i] = (x @ wv).reshape(B * K, H, D).to(t)
        q = heads((x @ wq)[:, None]).to(t)
        out = torch.empty((B * K, H, 1, D), device="cuda", dtype=t)
        gpu.attention(q, cache[0], cache[1], out, causal=True, kv_lens=torch.full((B * K,), F + i + 1, dtype=torch.int32, device="cuda"), stream=st)
        logits = (out.float().reshape(B, K, H * D) @ wo).contiguous()
        # the same from the texts alone, in one causal pass over features and text
        for b in range(B):
            for j in range(K):
                if scores[b, j] == -math.inf:
                    continue
                xs = torch.cat([feats[b], emb[torch.tensor(texts[b][j], device="cuda")]])
                whole, _, _ = ref.attention(*[heads((xs @ w)[None]).to(t) for w in (wq, wk, wv)], D ** -0.5, causal=True)
                got = out[b * K + j, :, 0].cpu().double()
                assert (got - whole[0, :, -1]).abs().max() < (0.03 if type == "bf16" else 1e-5)
        want = ref.beam_select(logits, scores, K, 1, done.cpu().numpy())
        gpu.beam_select(logits, scores, scores, par, tok, end=1, finished=done, out_finished=done, stream=st)
        gpu.beam_reorder(par, [(cache[0], cache[2]), (cache[1], cache[3])], axis=2, live=F + i + 1, stream=st)
        cache = [cache[2], cache[3], cache[0], cache[1]]
        p, k = par.cpu().numpy(), tok.cpu().numpy()
        assert (p == want[1]).all() and (k == want[2]).all()
        texts = [[texts[b][p[b, j]] + [int(k[b, j])] for j in range(K)] for b in range(B)]


# ---- the graphs' own paths -----------------------------------------------------------------
def _line_batch(seed, n, w):
    return np.random.default_rng(seed).normal(size=(n, 3, 48, w)).astype(np.float32)


@pytest.mark.parametrize("n, w", [(1, 8), (3, 64), (2, 320), (1, 1600)])
def test_ndgraph_with_fused_attention(gpu, n, w):
    """The recognition neck's two attentions as one kernel each: the same logits but for sums' last bits, captured too."""
    from wocr import NdGraph, synth
    g = NdGraph(gpu, synth.pp_rec_model(classes=211), stop_before_softmax=True)
    x = _line_batch(w, n, w)
    before = g.run(x)
    assert g.fuse_attention() == 2
    fused = [g.run(x) for _ in range(3)]
    launches = g.stats()[1]
    assert g.fuse_attention(False) == 2
    plain = [g.run(x) for _ in range(3)]
    assert g.stats()[1] >= launches + 4  # a softmax and a product fewer for each, and copies of k^T and v
    for p in plain:
        assert np.array_equal(p, before)
    for f in fused:
        assert np.array_equal(f, fused[0])
        # scores off by a few 2^-24 of the attention's sums, through a block and a half of the neck
        assert np.abs(f - before).max() <= 2.0 ** -17 * max(1.0, np.abs(before).max())
    g.close()


def _graph(nodes, weights=None, ints=None, inp="x", out="y"):
    from wocr import Model, Node
    return Model([Node(o, i, [n], a) for o, i, n, a in nodes], weights or {}, ints or {}, inp, out)


def test_ndgraph_attention_of_other_shapes(gpu):
    """What looks like attention but is not the kernel's: values of another width, a softmax that others read."""
    from wocr import NdGraph
    rng = np.random.default_rng(0)
    x = rng.normal(size=(2, 3, 6, 10)).astype(np.float32)
    wide = [("Transpose", ["x"], "kt", {"perm": [0, 1, 3, 2]}), ("MatMul", ["x", "kt"], "s", {}), ("Softmax", ["s"], "p", {"axis": -1}),
            ("Concat", ["x", "x"], "v", {"axis": 3}), ("MatMul", ["p", "v"], "y", {})]
    shared = [("Transpose", ["x"], "kt", {"perm": [0, 1, 3, 2]}), ("MatMul", ["x", "kt"], "s", {}), ("Softmax", ["s"], "p", {"axis": -1}),
              ("MatMul", ["p", "x"], "o", {}), ("MatMul", ["p", "o"], "y", {})]
    for nodes, found in ((wide, 1), (shared, 0)):
        g = NdGraph(gpu, _graph(nodes))
        before = g.run(x)
        assert g.fuse_attention() == found
        for _ in range(3):
            assert np.array_equal(g.run(x), before)
        g.close()
    # and one with keys that are no transposed view
    own = [("Relu", ["x"], "q", {}), ("Transpose", ["x"], "t", {"perm": [0, 1, 3, 2]}), ("Relu", ["t"], "kt", {}),
           ("MatMul", ["q", "kt"], "s", {}), ("Softmax", ["s"], "p", {"axis": 3}), ("MatMul", ["p", "x"], "y", {})]
    g = NdGraph(gpu, _graph(own))
    before = g.run(x)
    assert g.fuse_attention() == 1
    for _ in range(3):
        assert np.abs(g.run(x) - before).max() < 1e-5
    g.close()


def test_ndgraph_beam(gpu):
    """The graph and the search in one call: the texts that the search finds in the graph's own logits."""
    import wocr
    from wocr import NdGraph, synth
    g = NdGraph(gpu, synth.pp_rec_model(classes=97), stop_before_softmax=True)
    for n, w, lens in ((2, 64, None), (3, 160, [20, 7, 0]), (2, 64, None), (2, 64, None)):
        x = _line_batch(n + w, n, w) * 3
        logits = g.run(x)
        got = g.beam(x, width=6, paths=4, lens=lens)
        want = ref.ctc_beam(torch.tensor(logits), lens, 6, 0, 4)
        assert len(got) == n
        for i in range(n):
            live = int(np.isfinite(want[2][i]).sum())
            assert len(got[i]) == live
            for j, (text, score) in enumerate(got[i]):
                assert list(text) == list(want[0][i, j, :want[1][i, j]])
                assert abs(score - want[2][i, j]) <= 2.0 ** -24 * abs(want[2][i, j]) + logits.shape[1] * 2.0 ** -20
        # a width of one and a peaked step leave the greedy text
    assert wocr.beam_text([1, 2, 500], ["", "a", "b"]) == "ab"
    for kw, code in ((dict(width=0), 2), (dict(width=32), 2), (dict(width=2, paths=3), 1), (dict(blank=97), 1), (dict(lens=[1]), 3)):
        with pytest.raises(wocr.WocrError) as e:
            g.beam(x, **kw)
        assert e.value.code == code
    assert len(g.beam(x)) == 2  # and works on
    g.close()


# ---- beam search: scores and logits far apart in size -----------------------------------------
def select_far(gpu, logits, scores, kout, end=-1, finished=None):
    """select_check, with every output filled beforehand: none may be left as it was."""
    B = logits.shape[0]
    o = [torch.full((B, kout), 111, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    gpu.beam_select(logits, scores, o[0], o[1], o[2], end=end, finished=finished, out_finished=o[3], stream=0)
    torch.cuda.synchronize()
    got = [t.cpu().numpy() for t in o]
    want = ref.beam_select(logits, scores, kout, end, finished.cpu().numpy() if finished is not None else None)
    for g, w in zip(got[1:], want[1:]):
        assert (g == w).all(), (g, w)
    fin = np.isfinite(want[0])
    assert (np.isneginf(got[0]) == ~fin).all()
    assert (np.abs(got[0][fin] - want[0][fin]) <= 2.0 ** -24 * np.abs(want[0][fin]) + 2.0 ** -20).all()


@pytest.mark.parametrize("type, least", [("f32", -1e-20), ("f32", -2.0 ** -149), ("bf16", -2.0 ** -133), ("f16", -2.0 ** -24)])
@pytest.mark.parametrize("V, M", [(97, 1), (5000, 1), (5000, 4), (30000, 8)])
def test_beam_select_of_certain_log_probabilities(gpu, type, least, V, M):
    """Log-probabilities next to zero beside scores that they do not change: candidates that tie in 64 bits go by their place."""
    x = torch.full((2, 3, V), -50.0, device="cuda").to(TYPES[type])
    x[:, :, V // 3] = least
    x[1, 1, V // 2] = 0.0
    for score in (-3.0, -200.0):
        select_far(gpu, x[:, :1].contiguous(), torch.full((2, 1), score, device="cuda"), M)
        select_far(gpu, x, torch.full((2, 3), score, device="cuda"), M)
    # a tiny constant everywhere but for a few zeros
    flat = torch.full((1, 2, V), least, device="cuda").to(TYPES[type])
    flat[:, :, [V // 5, V - 2]] = 0.0
    select_far(gpu, flat, torch.full((1, 2), -3.0, device="cuda"), M)


@pytest.mark.parametrize("dead", [-1e9, -1e12, -1e30, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("V, M", [(97, 4), (5000, 4), (30000, 12)])
def test_beam_select_of_dead_beams(gpu, dead, V, M):
    """Beams that a program scores far below all others: alone, beside ended ones, over logits and log-probabilities."""
    for seed in range(6):
        x = randn((3, 4, V), "f32", 200 + seed, 2.0)
        for y in (x, torch.log_softmax(x, 2), torch.log_softmax(x, 2) - torch.log_softmax(x, 2).amax(2, keepdim=True)):
            scores = torch.full((3, 4), dead, device="cuda")
            select_far(gpu, y, scores, M)
            scores[:, 0] = -1.5
            fin = torch.zeros((3, 4), dtype=torch.uint8, device="cuda")
            fin[:, 0] = 1  # an ended beam: one candidate, the others are of the dead ones
            select_far(gpu, y, scores, M, end=2, finished=fin)
            select_far(gpu, y, scores, M, end=2)


def test_beam_select_of_infinite_logits(gpu):
    """An infinite logit counts as the largest number: next to it all others of its beam tie."""
    x = randn((2, 1, 5000), "f32", 41)
    x[0, 0, 100] = math.inf
    x[1, 0, [3, 4000]] = math.inf
    select_far(gpu, x, torch.zeros((2, 1), device="cuda"), 4)
    y = randn((1, 3, 400), "f32", 42)
    y[0, 1, 5] = math.inf
    select_far(gpu, y, torch.zeros((1, 3), device="cuda"), 6)
    select_far(gpu, y, torch.full((1, 3), float(np.finfo(np.float32).max), device="cuda"), 6)


# ---- attention: what is seen with a weight of next to nothing ----------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("TQ, TK, D", [(1, 200, 64), (3, 700, 128), (5, 60, 15), (40, 40, 15), (64, 100, 200), (150, 300, 64), (200, 900, 128)])
@pytest.mark.parametrize("below", [20.0, 100.0, 600.0])
def test_attention_sees_values_far_below_the_best(gpu, type, TQ, TK, D, below):
    """A key in sight whose weight is e^-below: NaN and infinities among its values reach the result, as they do by the
    definition, and the rows that do not see it stay finite."""
    q, k, v = qkv(1, 4, 4, TQ, TK, D, type, 301)
    q.fill_(1.0)
    k.zero_()
    at = TK - 1 - TQ // 2
    k[:, :, at, 0] = -below
    v[0, 0, at, 3], v[0, 1, at, 0], v[0, 2, at, D - 1] = float("nan"), math.inf, -math.inf
    for kw in (dict(), dict(causal=True)):
        out = attention_check(gpu, q, k, v, scale=1.0, **kw)
        want, _, _ = ref.attention(q, k, v, 1.0, **kw)
        got = out.cpu().double()
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
        assert torch.isinf(want[0, 1, -1, 0]) and torch.isnan(want[0, 0, -1, 3]) and torch.isfinite(want[0, 3]).all()


@pytest.mark.parametrize("type, value", [("f32", 3e38), ("bf16", 3e38), ("f16", 6e4)])
@pytest.mark.parametrize("TQ, TK, D", [(1, 200, 64), (3, 700, 128), (5, 60, 15), (40, 40, 15), (64, 100, 200), (150, 300, 64), (200, 900, 128)])
def test_attention_of_values_near_the_largest(gpu, type, value, TQ, TK, D):
    """A weighted mean of finite values is finite, although the sum before the division is not."""
    q, k, v = qkv(1, 2, 2, TQ, TK, D, type, 302)
    v.fill_(value)
    v[:, 1, :, ::2] *= -1
    v[:, :, TK // 2, 1] = 0.0
    # below the largest number by more than the weights' rounding (a sum of rounded weights may exceed one by a 16-bit step)
    v *= 0.99
    out = attention_check(gpu, q, k, v, causal=True)
    assert torch.isfinite(out).all()


def infinities_compare(out, q, k, v, scale, **kw):
    """Infinite outputs exactly, and no others: a tolerance cannot fail next to an infinite value."""
    want, _, rows = ref.attention(q, k, v, scale, **kw)
    got, want = out.cpu().double()[rows], want[rows]
    assert torch.isinf(want).any()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("TQ, TK, D", [(1, 200, 64), (64, 200, 15), (200, 300, 64), (260, 400, 128), (4, 900, 128), (20, 2500, 128), (70, 90, 200)])
def test_attention_of_infinities_in_sight(gpu, type, TQ, TK, D):
    """Infinite values that some rows see and others do not, behind a causal mask and in documents: their sign and place."""
    B, H = 2, 2
    q, k, v = qkv(B, H, H, TQ, TK, D, type, 311)
    at = TK - 1 - TQ // 2
    v[0, 0, at, D - 1], v[1, 1, at, 0], v[1, 0, at, 1] = math.inf, -math.inf, math.inf
    v[1, 0, at // 2, 1] = -math.inf  # both: no number, for the rows that see both
    scale = D ** -0.5
    docs = torch.zeros((B, TK), dtype=torch.int32, device="cuda")
    docs[:, at // 2] = 1
    same = torch.zeros((B, TQ), dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(causal=True), dict(q_docs=same, kv_docs=docs), dict(cap=9.0, causal=True)):
        infinities_compare(attention_check(gpu, q, k, v, scale=scale, **kw), q, k, v, scale, **kw)


# ---- CTC: logits far from zero -------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("v, width", [(40, 5), (300, 16), (7000, 4)])
def test_ctc_beam_of_steps_that_shift_every_class(gpu, type, v, width):
    """A step whose classes are all alike says nothing, however low or high it stands: the texts and masses are those of the
    step at zero."""
    plain = peaky(3, 12, v, type, 400 + v)
    plain[:, 4] = 0.0
    plain[1, 0] = plain[2, 11] = plain[2, 7] = 0.0
    x = plain.clone()
    low = torch.finfo(x.dtype).min
    x[:, 4] = low  # a padded step
    x[1, 0], x[2, 11], x[2, 7] = math.inf, 1e30, -1e9
    lens = i32([12, 12, 10])
    search_compare(search(gpu, x, lens, width, 0, width), plain, lens, width, 0, width)


@pytest.mark.parametrize("type", ["f32", "f16"])
@pytest.mark.parametrize("v", [60, 2500, 30000])
def test_ctc_beam_of_certain_steps(gpu, type, v):
    """An infinite logit, or all classes but one masked by a very low number: the step is that class, what comes before and
    after decides the rest."""
    plain = peaky(4, 9, v, type, 500 + v)
    low = -5e4 if type == "f16" else -1e5
    for t, c in ((2, 7), (3, 0), (5, v - 1)):
        plain[:, t] = low
        plain[:, t, c] = 0.0
    x = plain.clone()
    for t, c in ((2, 7), (3, 0), (5, v - 1)):
        x[0, t] = plain[0, 6]  # any finite logits beside the infinite one
        x[0, t, c] = math.inf
        x[1, t, torch.arange(v, device="cuda") != c] = torch.finfo(x.dtype).min
        x[2, t, torch.arange(v, device="cuda") != c] = -math.inf
    search_compare(search(gpu, x, None, 4, 0, 2), plain, None, 4, 0, 2)


def test_ndgraph_attention_in_a_chain(gpu):
    """The product that ends one attention begins the next: the step is run once, in the first."""
    from wocr import NdGraph
    x = np.random.default_rng(3).normal(size=(2, 2, 5, 5)).astype(np.float32)
    chain = [("Transpose", ["x"], "t", {"perm": [0, 1, 3, 2]}), ("MatMul", ["x", "t"], "s1", {}), ("Softmax", ["s1"], "p1", {"axis": -1}),
             ("MatMul", ["p1", "x"], "s2", {}), ("Softmax", ["s2"], "p2", {"axis": -1}), ("MatMul", ["p2", "x"], "s3", {}),
             ("Softmax", ["s3"], "p3", {"axis": -1}), ("MatMul", ["p3", "x"], "y", {})]
    g = NdGraph(gpu, _graph(chain))
    before = g.run(x)
    assert g.fuse_attention() == 2  # the first and the last: the middle one shares a product with either
    for _ in range(3):
        assert np.abs(g.run(x) - before).max() < 1e-5
    g.close()


@pytest.mark.parametrize("dtype", [torch.int64, torch.float64, torch.int16, torch.float8_e4m3fn, torch.bool])
def test_beam_reorder_of_any_type(gpu, dtype):
    """States are bytes: a history of 64-bit tokens, a cache in 8 bits."""
    par = i32([[2, 0, 0], [1, 1, 2]])
    rows = (torch.arange(2, device="cuda")[:, None] * 3 + par).reshape(-1)
    src = torch.randint(-9, 9, (6, 5, 7), device="cuda").to(dtype)
    dst = torch.zeros((6, 5, 7), device="cuda").to(dtype)
    gpu.beam_reorder(par, [(src, dst)], axis=2, live=3, stream=0)
    torch.cuda.synchronize()
    as_bytes = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(as_bytes(dst[:, :, :3]), as_bytes(src[rows][:, :, :3])) and not as_bytes(dst[:, :, 3:]).any()


# ---- attention: caps far above the scores ------------------------------------------------------
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [300.0, 1e4, 1e8, 1e30])
@pytest.mark.parametrize("TQ, TK, D", [(1, 300, 64), (3, 500, 128), (40, 60, 15), (200, 400, 64), (300, 300, 128)])
def test_attention_of_wide_caps(gpu, type, cap, TQ, TK, D):
    """A cap is as exact as its scores are, however wide it is: a score's tanh is off by 8 U of the score itself, where it was
    off by 2^-22 of the cap."""
    q, k, v = qkv(1, 4, 2, TQ, TK, D, type, 601)
    for boost in (1.0, 60.0):  # the second: some scores beyond 0.6 of the least cap
        qq = (q * boost).to(q.dtype)
        scale = D ** -0.5
        out = torch.zeros_like(q)
        gpu.attention(qq, k, v, out, scale=scale, cap=cap, stream=0)
        torch.cuda.synchronize()
        want, size, _ = ref.attention(qq, k, v, scale, cap=cap)
        mag = scale * float(torch.einsum("bhqd,bhkd->bhqk", qq.cpu().double().abs(), k.cpu().double().abs().repeat_interleave(2, 1)).max())
        half = q.dtype != torch.float32
        u = torch.finfo(q.dtype).eps / 2
        es = (D + 8 + 8) * U * mag
        tol = size * (2 * es + 2.0 ** -20 + TK * U + (u if half else 0)) + want.abs() * u
        if type == "f16":
            tol = tol + 2.0 ** -25 * (1 + TK * v.cpu().double().abs().max())
        assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("TQ", [1, 3, 40, 200])
def test_attention_of_documents_without_keys(gpu, type, TQ):
    q, k, v = qkv(2, 2, 2, TQ, 0, 16, type)
    out = torch.full(q.shape, 7.0, device="cuda", dtype=q.dtype)
    docs = torch.zeros((2, TQ), dtype=torch.int32, device="cuda")
    gpu.attention(q, k, v, out, q_docs=docs, kv_docs=docs[:, :0], stream=0)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_beam_select_of_beams_that_are_all_but_certain(gpu):
    """Beams of one score, each all but certain of its token: the one whose other tokens are least likely goes first,
    although its log-sum-exp is the maximum in 32 bits."""
    for type, V in (("f32", 5), ("f32", 700), ("f32", 30000), ("bf16", 700), ("f16", 30000)):
        x = torch.full((2, 6, V), -60.0, device="cuda")
        far = torch.tensor([-19.0, -24.0, -18.0, -32.0, -28.0, -21.0], device="cuda")  # e^-19 and less: below 2^-27
        for j in range(6):
            x[:, j, (3 * j) % V] = 0.0
            x[:, j, (3 * j + 1) % V] = far[j]
            x[1, j] += 8.0 * j  # (what a row adds to every logit says nothing)
        select_far(gpu, x.to(TYPES[type]), torch.full((2, 6), -1.0, device="cuda"), 6)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("TQ, TK, D", [(1, 200, 64), (3, 700, 128), (5, 60, 15), (40, 40, 15), (64, 100, 200), (150, 300, 64), (300, 2100, 64),
                                       (200, 900, 128)])
def test_attention_of_rows_whose_every_score_is_infinite(gpu, type, TQ, TK, D):
    """Scores of -inf alone have no softmax: no number. A row that sees nothing is zero, in documents without keys too, and
    whatever lies in the keys and values that it does not see."""
    q, k, v = qkv(2, 2, 2, TQ, TK, D, type, 305)
    q[:, 0, :: 2, 1] = -math.inf
    k[:, :, :, 1] = k[:, :, :, 1].abs() + 0.5
    odd = torch.zeros(TQ, dtype=torch.bool)
    odd[::2] = True
    ids = torch.zeros((2, TK), dtype=torch.int32, device="cuda")
    ids[:, TK // 2:] = 4
    seen = torch.zeros((2, TQ), dtype=torch.int32, device="cuda")
    seen[1] = 4
    seen[:, TQ // 3:] = 2  # a document that no key is in
    seen[:, -1] = -1
    bad = v.clone()
    bad[1, :, TK // 4] = float("nan")
    for values, kw in ((v, dict()), (v, dict(causal=True)), (v, dict(causal=True, kv_lens=i32([TK, max(TQ - 1, 1)]))),
                       (bad, dict(q_docs=seen, kv_docs=ids)), (bad, dict(q_docs=seen, kv_docs=ids, causal=True))):
        out = attention_check(gpu, q, k, values, **kw)
        if not kw:
            assert torch.isnan(out[:, 0, odd]).all() and torch.isfinite(out[:, 0, ~odd]).all() and torch.isfinite(out[:, 1]).all()
