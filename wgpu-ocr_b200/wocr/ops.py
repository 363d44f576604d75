"""Operators on device tensors: attention, beam search's selection and reordering, CTC prefix beam search.

They take CUDA tensors of the context's device: torch tensors, or `DeviceArray`s around any other allocation.  Nothing is
copied and nothing waits: work is queued on `stream`, a cudaStream_t as an int (0: the legacy default stream, as torch's
`current_stream().cuda_stream` names it; None: the context's own stream).  Outputs are the caller's tensors.  A tensor must
stay allocated until the stream has passed the call.
"""
from __future__ import annotations

import math
import struct
from typing import Optional, Sequence, Tuple

from . import _lib as L

F32, F16, BF16, I32, U8 = 1, 10, 16, 6, 2  # ONNX TensorProto codes
_NAMES = {"float32": F32, "float16": F16, "bfloat16": BF16, "int32": I32, "uint8": U8, "bool": U8}
_codes = {}  # dtype object -> code
# bytes of an element, for what is only copied
_SIZES = {n: size for size, names in ((1, "uint8 int8 float8_e4m3fn float8_e4m3fnuz float8_e5m2 float8_e5m2fnuz float8_e8m0fnu"),
                                      (2, "int16 uint16 float16 bfloat16"), (4, "int32 uint32 float32"),
                                      (8, "int64 uint64 float64")) for n in names.split()}
_kinds = {}  # dtype object -> (name, bytes of an element)
_ARGS = struct.Struct("10Q14q8i2f")
_STATE = struct.Struct("2Q4q")
_LEGACY = 1  # cudaStreamLegacy


class DeviceArray:
    """A device allocation of the caller's as a tensor: `dtype` by name, `strides` in elements (None: dense)."""

    def __init__(self, ptr: int, dtype: str, shape: Sequence[int], strides: Optional[Sequence[int]] = None, device: int = 0):
        self.ptr, self.dtype, self.shape, self.device = int(ptr), dtype, tuple(shape), device
        if strides is None:
            dense, n = [], 1
            for d in reversed(self.shape):
                dense.append(n)
                n *= d
            strides = dense[::-1]
        self._strides = tuple(strides)

    def data_ptr(self) -> int:
        return self.ptr

    def stride(self) -> Tuple[int, ...]:
        return self._strides

    def is_contiguous(self) -> bool:
        n = 1
        for d, s in zip(reversed(self.shape), reversed(self._strides)):
            if d != 1 and s != n and 0 not in self.shape:
                return False
            n *= d
        return True

    def get_device(self) -> int:
        return self.device


def _code(x) -> int:
    code = _codes.get(x.dtype)
    if code is None:
        name = str(x.dtype).rsplit(".", 1)[-1]
        if name not in _NAMES:
            raise ValueError(f"element type {x.dtype} is not supported")
        code = _codes[x.dtype] = _NAMES[name]
    return code


def _kind(x) -> Tuple[str, int]:
    kind = _kinds.get(x.dtype)
    if kind is None:
        name = str(x.dtype).rsplit(".", 1)[-1]
        name = "uint8" if name == "bool" else name
        if name not in _SIZES:
            raise ValueError(f"element type {x.dtype} is not supported")
        kind = _kinds[x.dtype] = name, _SIZES[name]
    return kind


def _elsewhere(gpu, name: str):
    return ValueError(f"{name} is not on device {gpu.device}")


def _dense(gpu, x, name: str, code: int, shape) -> int:
    """The address of a dense tensor of one type and shape."""
    if x is None:
        raise ValueError(f"{name} is missing")
    if _code(x) != code or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"{name}: expected type {code}, contiguous, of shape {shape}, got {x.dtype} {tuple(x.shape)}")
    if x.get_device() != gpu.device:
        raise _elsewhere(gpu, name)
    return x.data_ptr()


def _state(gpu, x, kind, shape) -> int:
    """The address of a dense tensor of one type and shape that is only copied."""
    if _kind(x) != kind or x.shape != shape or not x.is_contiguous():
        raise ValueError(f"state: expected {kind[0]}, contiguous, of shape {shape}, got {x.dtype} {tuple(x.shape)}")
    if x.get_device() != gpu.device:
        raise _elsewhere(gpu, "state")
    return x.data_ptr()


def _rows(gpu, x, name: str, shape) -> Tuple[int, int]:
    """The address and row stride of an int32 [rows, n] tensor whose rows are contiguous."""
    s = x.stride()
    if _code(x) != I32 or tuple(x.shape) != shape or (shape[1] > 1 and s[1] != 1):
        raise ValueError(f"{name}: expected int32 rows of shape {shape}, got {x.dtype} {tuple(x.shape)}, strides {s}")
    if x.get_device() != gpu.device:
        raise _elsewhere(gpu, name)
    return x.data_ptr(), s[0]


def _stream(stream) -> Optional[int]:
    return None if stream is None else (stream or _LEGACY)


class DeviceOps:
    """The operators as methods of `Gpu`."""

    def attention(self, q, k, v, out, scale: Optional[float] = None, cap: float = 0.0, slopes=None, causal: bool = False,
                  prefix=None, q_lens=None, kv_lens=None, q_docs=None, kv_docs=None, stream: Optional[int] = None):
        """Softmax attention (`wocr_attention`): q, out [batch, heads, queries, dim], k, v [batch, kv_heads, keys, dim]
        of one type (float32, float16, bfloat16) and any strides but for a contiguous last dimension of 1 to 256.

        score = cap tanh(scale q.k / cap) - slopes[h] |distance|; query i of batch element b stands at position
        kv_lens[b] - q_lens[b] + i among its keys and sees those below kv_lens[b]; with `causal` up to its own position
        or below prefix[b]; with documents those whose id is its own, negative ids none.  scale None: dim ** -0.5.
        slopes float32 [heads]; prefix, q_lens, kv_lens int32 [batch]; q_docs [batch, queries], kv_docs [batch, keys]
        int32.  A query that sees nothing gets zeros; rows from q_lens[b] on are left as they were."""
        t = q.dtype
        code = _code(q)
        if (k.dtype != t and _code(k) != code) or (v.dtype != t and _code(v) != code) or (out.dtype != t and _code(out) != code):
            raise ValueError("q, k, v and out have different types")
        qs, ks = q.shape, k.shape
        if len(qs) != 4 or len(ks) != 4 or v.shape != ks or out.shape != qs or qs[0] != ks[0] or qs[3] != ks[3]:
            raise ValueError(f"attention shapes: q {tuple(qs)}, k {tuple(ks)}, v {tuple(v.shape)}, out {tuple(out.shape)}")
        b, h, tq, d = qs
        _, hk, tk, _ = ks
        q0, q1, q2, qd = q.stride()
        k0, k1, k2, kd = k.stride()
        v0, v1, v2, vd = v.stride()
        o0, o1, o2, od = out.stride()
        if d > 1 and not qd == kd == vd == od == 1:
            raise ValueError("attention: the last dimension is not contiguous")
        dev = self.device
        if not (q.get_device() == k.get_device() == v.get_device() == out.get_device() == dev):
            raise _elsewhere(self, "q, k, v or out")
        qi, qis = (0, 0) if q_docs is None else _rows(self, q_docs, "q_docs", (b, tq))
        ki, kis = (0, 0) if kv_docs is None else _rows(self, kv_docs, "kv_docs", (b, tk))
        args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                          0 if slopes is None else _dense(self, slopes, "slopes", F32, (h,)),
                          0 if prefix is None else _dense(self, prefix, "prefix", I32, (b,)),
                          0 if q_lens is None else _dense(self, q_lens, "q_lens", I32, (b,)),
                          0 if kv_lens is None else _dense(self, kv_lens, "kv_lens", I32, (b,)),
                          qi, ki, q0, q1, q2, k0, k1, k2, v0, v1, v2, o0, o1, o2, qis, kis,
                          code, b, h, hk, tq, tk, d, causal, d ** -0.5 if scale is None else scale, cap)
        st = L.lib().wocr_attention(self.h, args, _stream(stream))
        if st:
            L.check(st)

    def beam_select(self, logits, scores, out_scores, out_parents, out_tokens, end: int = -1, finished=None,
                    out_finished=None, stream: Optional[int] = None):
        """One selection of beam search (`wocr_beam_select`): logits [batch, beams, vocab] (float32, float16, bfloat16,
        last dimension contiguous), scores float32 [batch, beams]; the best candidates' scores (float32), parent beams and
        tokens (int32), [batch, out_beams] each, best first, ties to the lowest beam * vocab + token.  `finished` (uint8
        [batch, beams]) beams keep their score and give `end`; out_finished (uint8) says which of the chosen have ended."""
        if len(logits.shape) != 3 or len(out_scores.shape) != 2:
            raise ValueError("logits [batch, beams, vocab] and out_scores [batch, beams] expected")
        b, n, v = logits.shape
        m = out_scores.shape[1]
        s0, s1, s2 = logits.stride()
        if v > 1 and s2 != 1:
            raise ValueError("logits: the last dimension is not contiguous")
        if logits.get_device() != self.device:
            raise _elsewhere(self, "logits")
        inn, out = (b, n), (b, m)
        st = L.lib().wocr_beam_select(
            self.h, logits.data_ptr(), _code(logits), b, n, v, s0, s1, _dense(self, scores, "scores", F32, inn),
            None if finished is None else _dense(self, finished, "finished", U8, inn), end, m,
            _dense(self, out_scores, "out_scores", F32, out), _dense(self, out_parents, "out_parents", I32, out),
            _dense(self, out_tokens, "out_tokens", I32, out),
            None if out_finished is None else _dense(self, out_finished, "out_finished", U8, out), _stream(stream))
        if st:
            L.check(st)

    def beam_reorder(self, parents, states, axis: int = 0, live: Optional[int] = None, stream: Optional[int] = None):
        """The states of the chosen beams in their new order (`wocr_beam_reorder`): `parents` int32 [batch, out_beams] as
        beam_select gives them; `states` pairs of tensors (src [batch * beams, ...], dst [batch * out_beams, ...]) of any
        real type, dense and alike but for the first dimension.  With `axis` > 0 only the first `live` entries along it are copied (a
        cache's tokens); the rest of dst, and rows whose parent is not a beam, are left as they were."""
        if len(parents.shape) != 2:
            raise ValueError("parents [batch, beams] expected")
        b, m = parents.shape
        n, parts = None, []
        for src, dst in states:
            shape = tuple(src.shape)
            kind = _kind(src)
            if not 0 <= axis < len(shape):
                raise ValueError(f"axis {axis} of a state of shape {shape}")
            rows = shape[0] // b if b else 1
            if rows < 1 or shape[0] != rows * b or (n is not None and rows != n):
                raise ValueError(f"a state of shape {shape} for {b} x {m} parents and {n} beams")
            n = rows
            full = kind[1] * math.prod(shape[axis or 1:])  # bytes of a piece and of what of it is copied
            part = full
            if axis and live is not None:
                if not 0 <= live <= shape[axis]:
                    raise ValueError(f"live {live} of a state of shape {shape}")
                part = full // max(shape[axis], 1) * live
            pieces = math.prod(shape[1:axis])
            parts.append(_STATE.pack(_state(self, src, kind, shape), _state(self, dst, kind, (b * m,) + shape[1:]),
                                     pieces, part, full, pieces * full))
        st = L.lib().wocr_beam_reorder(self.h, _dense(self, parents, "parents", I32, (b, m)), b, n or 1, m, b"".join(parts),
                                       len(parts), _stream(stream))
        if st:
            L.check(st)

    def ctc_beam(self, logits, tokens, lengths, scores, lens=None, width: int = 8, blank: int = 0,
                 stream: Optional[int] = None):
        """CTC prefix beam search (`wocr_ctc_beam`): logits [lines, steps, classes] (float32, float16, bfloat16, last
        dimension contiguous), lens int32 [lines]; `width` (1 to 31) texts kept per step.  The best `paths` texts of each
        line: tokens int32 [lines, paths, steps] (-1 past the end), lengths int32 and scores float32 (log mass) [lines,
        paths]; paths is at most width."""
        if len(logits.shape) != 3 or len(tokens.shape) != 3:
            raise ValueError("logits [lines, steps, classes] and tokens [lines, paths, steps] expected")
        n, t, v = logits.shape
        p = tokens.shape[1]
        s0, s1, s2 = logits.stride()
        if v > 1 and s2 != 1:
            raise ValueError("logits: the last dimension is not contiguous")
        if logits.get_device() != self.device:
            raise _elsewhere(self, "logits")
        st = L.lib().wocr_ctc_beam(
            self.h, logits.data_ptr(), _code(logits), n, t, v, s0, s1,
            None if lens is None else _dense(self, lens, "lens", I32, (n,)), width, blank, p,
            _dense(self, tokens, "tokens", I32, (n, p, t)), _dense(self, lengths, "lengths", I32, (n, p)),
            _dense(self, scores, "scores", F32, (n, p)), _stream(stream))
        if st:
            L.check(st)
