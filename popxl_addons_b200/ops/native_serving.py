"""CUDA implementations of the serving ops (`xl/ops/serving.py`)."""
import torch

from ..xl.opdef import native
from .native import _CODE, _c_f, _c_int, _c_ll, _c_p, _check, _count, _ok, _sig, _stream, counters
from .native_sequence import _clamped_glu, _f32, _i32, _ptr, stream_rms

_shape_logits = _sig("xl_shape_logits", *[_c_p] * 10, *[_c_int] * 7, _c_p)
_take_shaped = _sig("xl_take_shaped", *[_c_p] * 13, *[_c_int] * 11, _c_p)
_append_tokens = _sig("xl_append_tokens", _c_p, _c_p, _c_p, _c_p, _c_int, _c_int, _c_int, _c_p)


def _launched(rc, name) -> bool:
    """Whether the kernel took its arguments (-1: it does not take such ones)."""
    if rc == -1:
        return False
    _check(rc, name)
    _count(name)
    return True


@native("split_glu")
def split_glu_cuda(y, cols, lead, limit, slope, shift):
    if y.dtype not in _CODE or not y.is_cuda or not y.is_contiguous():
        return NotImplemented
    n, N = y.shape
    f = (N - cols) // 2
    joint = torch.empty((n, lead + f), dtype=y.dtype, device=y.device)
    if f:
        _check(_clamped_glu(y.data_ptr() + cols * y.element_size(), N, joint.data_ptr() + lead * y.element_size(), lead + f, n, f, limit,
                            slope, shift, _CODE[y.dtype], _stream()), "clamped_glu")
        _count("clamped_glu")
    return y[:, :cols], joint


@native("residual_rms_")
def residual_rms_cuda(x, y, *norm, mult, eps):
    return stream_rms(x, y, mult, None, None, norm[0] if norm else None, eps, y.dtype)


def _rules_ok(history, start, penalties, bias_tokens, bias_values, allowed) -> bool:
    return (_i32(history, start, bias_tokens, allowed) and _f32(penalties, bias_values)
            and all(t.is_cuda and t.is_contiguous() for t in (penalties, bias_values)))


@native("shape_logits")
def shape_logits_cuda(logits, slot, length, *rules):
    if not _ok(logits) or logits.dim() != 2 or not _i32(slot, length) or not _rules_ok(*rules):
        return NotImplemented
    (rows, V), (slots, L) = logits.shape, rules[0].shape
    out = torch.empty((rows, V), dtype=torch.float32, device=logits.device)
    rc = _shape_logits(logits.data_ptr(), out.data_ptr(), slot.data_ptr(), length.data_ptr(), *map(_ptr, rules), rows, V, slots, L,
                       rules[3].shape[1], rules[5].shape[1], _CODE[logits.dtype], _stream())
    return out if _launched(rc, "shape_logits") else NotImplemented


@native("take_shaped_")
def take_shaped_cuda(current, logits, buf, pos, length, count, *rules, valid, base, ahead, advance):
    if not _ok(logits) or logits.dim() != 2 or not _i32(current, buf, pos, length, count) or not _rules_ok(*rules):
        return NotImplemented
    rows, V = logits.shape
    if buf.dim() != 2 or not current.numel() == buf.shape[1] == rows:
        return NotImplemented
    rc = _take_shaped(logits.data_ptr(), current.data_ptr(), buf.data_ptr(), pos.data_ptr(), length.data_ptr(), count.data_ptr(),
                      *map(_ptr, rules), counters(1, logits.device, "counters greedy", 1).data_ptr(), rows, V, valid, buf.shape[0], base,
                      ahead, int(advance), rules[0].shape[1], rules[3].shape[1], rules[5].shape[1], _CODE[logits.dtype], _stream())
    return current if _launched(rc, "take_shaped") else NotImplemented


@native("append_tokens_")
def append_tokens_cuda(history, tokens, pos, count, T):
    tokens = tokens.reshape(-1)
    if not _i32(history, tokens, pos, count) or tokens.numel() != history.shape[0] * T:
        return NotImplemented
    rc = _append_tokens(history.data_ptr(), tokens.data_ptr(), pos.data_ptr(), count.data_ptr(), history.shape[0], T, history.shape[1],
                        _stream())
    return history if _launched(rc, "append_tokens") else NotImplemented
