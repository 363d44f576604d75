"""The operators' argument checks, before any device is touched (no GPU needed), and the tests' own definitions."""
import numpy as np
import pytest
import torch

import wocr
from wocr import DeviceArray, _lib
from wocr.ops import DeviceOps

import _operators as ref


class _Bare(DeviceOps):
    """The Python side without a context: what passes its checks and the library's ends at the missing context."""
    h = None
    device = 0


def arr(shape, dtype="float32", strides=None, ptr=1 << 20, device=0):
    return DeviceArray(ptr, dtype, shape, strides, device)


def attn(**kw):
    b, h, hk, tq, tk, d = 2, 4, 2, 5, 7, 16
    a = dict(q=arr((b, h, tq, d)), k=arr((b, hk, tk, d), ptr=2 << 20), v=arr((b, hk, tk, d), ptr=3 << 20),
             out=arr((b, h, tq, d), ptr=4 << 20))
    a.update(kw)
    return _Bare().attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("out"), **a)


def test_what_is_right_ends_at_the_missing_context():
    for call in (lambda: attn(),
                 lambda: attn(cap=5.0, causal=True, prefix=arr((2,), "int32"), slopes=arr((4,)), kv_lens=arr((2,), "int32"),
                              q_lens=arr((2,), "int32"), q_docs=arr((2, 5), "int32"), kv_docs=arr((2, 7), "int32")),
                 lambda: attn(q=arr((0, 4, 5, 16)), k=arr((0, 2, 7, 16)), v=arr((0, 2, 7, 16)), out=arr((0, 4, 5, 16))),
                 lambda: select(), lambda: reorder(), lambda: search()):
        with pytest.raises(wocr.WocrError, match="null ctx"):
            call()


@pytest.mark.parametrize("kw, code, text", [
    (dict(k=arr((2, 3, 7, 16), ptr=2 << 20), v=arr((2, 3, 7, 16), ptr=3 << 20)), 3, "cannot share"),
    (dict(q=arr((2, 4, 5, 257)), k=arr((2, 2, 7, 257), ptr=2 << 20), v=arr((2, 2, 7, 257), ptr=3 << 20),
          out=arr((2, 4, 5, 257), ptr=4 << 20)), 2, "head dimension"),
    (dict(scale=float("inf")), 1, "finite"),
    (dict(cap=-1.0), 1, "cap"),
    (dict(cap=float("nan")), 1, "cap"),
    (dict(q_docs=arr((2, 5), "int32")), 1, "documents"),
    (dict(kv_docs=arr((2, 7), "int32")), 1, "documents"),
    (dict(prefix=arr((2,), "int32")), 1, "prefix"),
    (dict(q=arr((2, 4, 5, 16), ptr=(1 << 20) + 2)), 1, "aligned"),
    (dict(q=arr((2, 4, 5, 16), ptr=0)), 1, "null q"),
    (dict(out=arr((2, 4, 5, 16), strides=(320, 80, 0, 1), ptr=4 << 20)), 1, "one another"),
    (dict(out=arr((2, 4, 5, 16), strides=(320, 80, 8, 1), ptr=4 << 20)), 1, "one another"),
    (dict(out=arr((2, 4, 5, 16))), 1, "inputs"),
    (dict(k=arr((2, 2, 7, 16), strides=(224, 112, -16, 1), ptr=2 << 20)), 1, "negative"),
])
def test_attention_refuses(kw, code, text):
    with pytest.raises(wocr.WocrError, match=text) as e:
        attn(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("kw", [
    dict(q=arr((2, 4, 5, 16), "float16")),
    dict(q=arr((2, 4, 5, 16), "float64"), k=arr((2, 2, 7, 16), "float64"), v=arr((2, 2, 7, 16), "float64"), out=arr((2, 4, 5, 16), "float64")),
    dict(q=arr((4, 5, 16))),
    dict(out=arr((2, 4, 6, 16))),
    dict(v=arr((2, 2, 8, 16))),
    dict(q=arr((2, 4, 5, 16), strides=(640, 160, 32, 2))),
    dict(q=arr((2, 4, 5, 16), device=1)),
    dict(kv_lens=arr((3,), "int32")),
    dict(kv_lens=arr((2,), "float32")),
    dict(kv_lens=arr((2,), "int32", strides=(2,))),
    dict(slopes=arr((2,))),
    dict(q_docs=arr((2, 5), "int32", strides=(10, 2)), kv_docs=arr((2, 7), "int32")),
])
def test_attention_refuses_tensors_that_do_not_fit(kw):
    with pytest.raises(ValueError):
        attn(**kw)


def select(b=2, k=3, v=50, m=3, **kw):
    a = dict(logits=arr((b, k, v)), scores=arr((b, k)), out_scores=arr((b, m), ptr=5 << 20), out_parents=arr((b, m), "int32"),
             out_tokens=arr((b, m), "int32"))
    a.update(kw)
    return _Bare().beam_select(**a)


@pytest.mark.parametrize("kw, code, text", [
    (dict(k=33), 2, "more than 32"),
    (dict(m=33), 2, "more than 32"),
    (dict(k=1, v=2), 3, "out of"),
    (dict(end=50), 1, "end token"),
    (dict(finished=arr((2, 3), "uint8")), 1, "end token"),
    (dict(logits=arr((2, 3, 50), ptr=(1 << 20) + 1)), 1, "aligned"),
    (dict(m=2, out_scores=arr((2, 2))), 1, "in place"),
])
def test_beam_select_refuses(kw, code, text):
    with pytest.raises(wocr.WocrError, match=text) as e:
        select(**kw)
    assert e.value.code == code


@pytest.mark.parametrize("kw", [dict(scores=arr((2, 4))), dict(out_tokens=arr((2, 3), "float32")),
                                dict(logits=arr((2, 3, 50), strides=(300, 100, 2))), dict(logits=arr((2, 3, 50), "int32"), scores=None)])
def test_beam_select_refuses_tensors_that_do_not_fit(kw):
    with pytest.raises((ValueError, wocr.WocrError)):
        select(**kw)


def reorder(b=2, m=3, n=3, shape=(4, 8, 16), parents=None, dst=8 << 20, **kw):
    states = [(arr((b * n,) + shape, "float16"), arr((b * m,) + shape, "float16", ptr=dst))]
    return _Bare().beam_reorder(parents or arr((b, m), "int32"), states, **kw)


def test_beam_reorder_refuses():
    with pytest.raises(wocr.WocrError, match="overlap"):
        reorder(dst=(1 << 20) + 4096)
    with pytest.raises(wocr.WocrError, match="more than 32"):
        reorder(m=33, n=33)
    lib, state = wocr.lib(), __import__("struct").pack("2Q4q", 1 << 20, 1 << 30, 1 << 62, 16, 1 << 40, 1 << 40)
    assert lib.wocr_beam_reorder(None, 4096, 2, 3, 3, state, 1, None) == 1 and b"64 bits" in lib.wocr_last_error()
    for kw in (dict(axis=4), dict(axis=-1), dict(axis=2, live=9), dict(axis=2, live=-1)):
        with pytest.raises(ValueError):
            reorder(**kw)
    with pytest.raises(ValueError):
        _Bare().beam_reorder(arr((2, 3), "int32"), [(arr((5, 4)), arr((6, 4)))])
    with pytest.raises(ValueError):
        _Bare().beam_reorder(arr((2, 3), "int32"), [(arr((6, 4)), arr((6, 5)))])


def search(n=2, t=5, v=20, p=2, **kw):
    a = dict(logits=arr((n, t, v)), tokens=arr((n, p, t), "int32"), lengths=arr((n, p), "int32"), scores=arr((n, p)), width=4)
    a.update(kw)
    return _Bare().ctc_beam(**a)


@pytest.mark.parametrize("kw, code, text", [
    (dict(width=0), 2, "width"), (dict(width=32), 2, "width"), (dict(width=1), 1, "paths"), (dict(blank=20), 1, "blank"),
    (dict(blank=-1), 1, "blank"),
])
def test_ctc_beam_refuses(kw, code, text):
    with pytest.raises(wocr.WocrError, match=text) as e:
        search(**kw)
    assert e.value.code == code


def test_ctc_beam_refuses_tensors_that_do_not_fit():
    for kw in (dict(lens=arr((3,), "int32")), dict(tokens=arr((2, 2, 6), "int32")), dict(lengths=arr((2, 2), "int64")),
               dict(logits=arr((2, 5, 20), strides=(200, 40, 2)))):
        with pytest.raises(ValueError):
            search(**kw)


def test_null_arguments_are_status_codes():
    lib = wocr.lib()
    assert lib.wocr_attention(None, None, None) == 1
    assert lib.wocr_beam_reorder(None, None, 1, 1, 1, None, 1, None) == 1
    assert lib.wocr_ctc_beam(None, None, 7, 1, 1, 1, 1, 1, None, 1, 0, 1, None, None, None, None) == 2
    assert b"element type" in lib.wocr_last_error()


# ---- the definitions that the GPU tests hold the kernels to ------------------------------
def test_reference_search_finds_every_text():
    """Wide enough to keep every text, the search's masses are the sums over all alignments."""
    rng = np.random.default_rng(0)
    x = torch.tensor(rng.normal(size=(1, 4, 3)).astype(np.float32))
    tokens, lengths, scores = ref.ctc_beam(x, None, 31, 0, 31)
    p = np.exp(torch.log_softmax(x.double(), 2).numpy()[0])
    mass = {}
    for path in np.ndindex(3, 3, 3, 3):
        text, last = [], 0
        for c in path:
            if c != 0 and c != last:
                text.append(c)
            last = c
        mass[tuple(text)] = mass.get(tuple(text), 0.0) + np.prod([p[t, c] for t, c in enumerate(path)])
    assert len(mass) <= 31
    found = {tuple(tokens[0, r, :lengths[0, r]]): scores[0, r] for r in range(31) if scores[0, r] > -np.inf}
    assert set(found) == set(mass)
    for text, s in found.items():
        assert abs(s - np.log(mass[text])) < 1e-9


def test_reference_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((2, 3, 4, 5), generator=g) for _ in range(3))
    out, size, rows = ref.attention(q, k, v, 0.3)
    want = torch.softmax(q.double() @ k.double().transpose(2, 3) * 0.3, 3) @ v.double()
    assert rows.all() and (out - want).abs().max() < 1e-12 and (size >= out.abs()).all()


def test_beam_reorder_takes_any_type():
    """What is only copied may have any element type, alike in source and destination."""
    par = arr((2, 3), "int32")
    pair = lambda a, b: [(arr((6, 4), a), arr((6, 4), b, ptr=8 << 20))]  # noqa: E731
    for t in ("int64", "float64", "int8", "bool", "float8_e4m3fn"):
        with pytest.raises(wocr.WocrError, match="null ctx"):
            _Bare().beam_reorder(par, pair(t, t))
    for a, b in (("bool", "uint8"), ("int64", torch.int64)):
        with pytest.raises(wocr.WocrError, match="null ctx"):
            _Bare().beam_reorder(par, pair(a, b))
    for a, b in (("int64", "float64"), ("float16", "bfloat16"), ("object", "object"), ("complex64", "complex64")):
        with pytest.raises(ValueError):
            _Bare().beam_reorder(par, pair(a, b))


def test_beam_reorder_refuses_states_of_no_beams():
    """A source without rows has no beam that a parent could name."""
    with pytest.raises(ValueError, match="shape"):
        _Bare().beam_reorder(arr((2, 3), "int32"), [(arr((0, 4)), arr((6, 4), ptr=8 << 20))])
    with pytest.raises(wocr.WocrError, match="null ctx"):  # no batch elements: nothing to do
        _Bare().beam_reorder(arr((0, 3), "int32"), [(arr((0, 4)), arr((0, 4), ptr=8 << 20))])


def test_beam_reorder_refuses_states_that_share_memory():
    """One launch copies all states, in no order: what one writes, no other may read or write."""
    par = arr((2, 3), "int32")
    t = lambda mb, shape=(6, 4, 8): arr(shape, ptr=mb << 20)  # noqa: E731
    ok = pytest.raises(wocr.WocrError, match="null ctx")
    bad = pytest.raises(wocr.WocrError, match="overlap")
    with bad:  # a chain: the first's destination is the second's source
        _Bare().beam_reorder(par, [(t(1), t(2)), (t(2), t(3))])
    with bad:  # two with one destination
        _Bare().beam_reorder(par, [(t(1), t(3)), (t(2), t(3))])
    with bad:  # in part, several states apart
        _Bare().beam_reorder(par, [(t(i), t(40 + i)) for i in range(1, 20)] + [(t(20), arr((6, 4, 8), ptr=(45 << 20) + 700))])
    with ok:  # a source that two states read, any number of others
        _Bare().beam_reorder(par, [(t(1), t(2)), (t(1), t(3))] + [(t(i), t(90 + i)) for i in range(10, 80)])
    # keys and values interleaved in one allocation, row by row and head by head: the library's own call
    lib, pack = wocr.lib(), __import__("struct").pack
    call = lambda *st: (lib.wocr_beam_reorder(None, 4096, 2, 3, 3, b"".join(pack("2Q4q", *s) for s in st), len(st), None),  # noqa: E731
                        lib.wocr_last_error())
    a, b = 1 << 20, 1 << 24
    assert b"null ctx" in call((a, b, 4, 64, 64, 1024), (a + 512, b + 512, 4, 64, 64, 1024))[1]   # halves of a row
    assert b"null ctx" in call((a, b, 4, 64, 256, 1024), (a + 64, b + 64, 4, 64, 256, 1024))[1]   # quarters of a head
    assert b"null ctx" in call((a, a + 512, 4, 64, 64, 1024))[1]                                  # both halves are one state's
    assert b"overlap" in call((a, b, 4, 64, 256, 1024), (a + 64, b + 32, 4, 64, 256, 1024))[1]
    assert b"overlap" in call((a, b, 4, 64, 128, 1024), (a + 512, b + 384, 4, 64, 128, 1024))[1]
    assert b"overlap" in call((a, b, 1, 1024, 1024, 1024), (b + 5 * 1024, 1 << 26, 1, 1024, 1024, 1024))[1]  # a last row
    assert b"null ctx" in call((a, b, 1, 1024, 1024, 1024), (b + 6 * 1024, 1 << 26, 1, 1024, 1024, 1024))[1]


def test_attention_takes_empty_documents():
    """No keys or no queries: their ids have no address, as any empty tensor's."""
    docs = lambda n: arr((2, n), "int32", ptr=1 << 20 if n else 0)  # noqa: E731
    for tq, tk in ((5, 0), (0, 7), (0, 0)):
        with pytest.raises(wocr.WocrError, match="null ctx"):
            attn(q=arr((2, 4, tq, 16)), out=arr((2, 4, tq, 16), ptr=4 << 20), k=arr((2, 2, tk, 16), ptr=2 << 20),
                 v=arr((2, 2, tk, 16), ptr=3 << 20), q_docs=docs(tq), kv_docs=docs(tk))
