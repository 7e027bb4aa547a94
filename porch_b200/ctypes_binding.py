"""csrc/python/binding.cpp in ctypes, name for name: tensor handles and the
decode-step operators, for interpreters that the compiled module was not built
for. The same results and errors; a call costs 2 to 5 us more."""

from __future__ import annotations

import operator
from ctypes import byref, c_float, c_int64, c_void_p

_tensor_type = _realise = _check = _load = None


class Handle:
    """A native tensor handle, released with the object."""

    __slots__ = ("_h", "_face")

    def __init__(self, handle):
        if handle is not None:
            handle = operator.index(handle) or None
        self._h, self._face = handle, None

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None:
            try:
                _load().pb_tensor_release(h)
                self._h = None
            except Exception:  # interpreter shutdown
                pass

    @property
    def __cuda_array_interface__(self) -> dict:
        if self._face is None:
            v = (c_int64 * 19)()
            _check(_load().pb_tensor_interface(self._h, v, 19))
            self._face = {"shape": tuple(v[3 : 3 + v[0]]), "typestr": "<f4", "data": (v[1], False), "version": 3,
                          "stream": v[2]}
        return self._face


def bind(tensor_type, realise, check, load) -> None:
    global _tensor_type, _realise, _check, _load
    if not issubclass(tensor_type, Handle):
        raise TypeError("the tensor type must derive from Handle")
    _tensor_type, _realise, _check, _load = tensor_type, realise, check, load


def connect(path) -> None:
    """ctypes has the library already."""


def _tensors(given):
    """The operands, expressions realised: held until the call has returned."""
    out = [x if isinstance(x, Handle) else _realise(x) for x in given]
    if not all(isinstance(x, Handle) for x in out):
        raise TypeError("expected a tensor")
    return out


def _call(function, count, *args):
    """function(*args, out...) with `count` tensors out."""
    out = [c_void_p() for _ in range(count)]
    _check(getattr(_load(), function)(*args, *map(byref, out)))
    return tuple(_tensor_type(x.value) for x in out)


def qk_norm_rope(*args):
    t, eps, interleaved = _tensors(args[:7]), c_float(args[7]), bool(args[8])
    return _call("pb_qk_norm_rope", 2, *[x._h for x in t], eps, interleaved)


def qk_norm_rope_backward(*args):
    t, eps, interleaved = _tensors(args[:9]), c_float(args[9]), bool(args[10])
    out = (c_void_p * 4)()
    _check(_load().pb_qk_norm_rope_backward(*[x._h for x in t], eps, interleaved, out))
    return tuple(_tensor_type(x) for x in out)


def token_logprobs(logits, tokens, top):
    t, top = _tensors([logits, tokens]), operator.index(top)
    out = (c_void_p * 5)()
    _check(_load().pb_token_logprobs(*[x._h for x in t], top, out))
    return tuple(_tensor_type(x) for x in out if x)


def token_logprobs_backward(*args):
    t = _tensors(args[:4])
    more = [None if x is None else _tensors([x])[0] for x in args[4:6]]
    return _call("pb_token_logprobs_backward", 1, *[x._h for x in t], *[x and x._h for x in more])[0]


def paged_attention(q, batch, scale):
    (q,), scale = _tensors([q]), c_float(scale)
    return _call("pb_paged_attention", 1, q._h, batch, scale)[0]


def paged_attention_scored(q, batch, scores, scale):
    (q, *scores), scale = _tensors([q] if scores is None else [q, scores]), c_float(scale)
    return _call("pb_paged_attention_scored", 2, q._h, batch, scores[0]._h if scores else None, scale)


def kv_read(batch):
    return _call("pb_kv_read", 2, batch)


def kv_evict(batch, scores, positions, budget, recent, sinks):
    scores, *positions = _tensors([scores] if positions is None else [scores, positions])
    sizes = [operator.index(x) for x in (budget, recent, sinks)]
    return _call("pb_kv_evict", 2, batch, scores._h, positions[0]._h if positions else None, *sizes)
