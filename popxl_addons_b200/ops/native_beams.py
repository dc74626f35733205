"""CUDA implementations of the ops of sequences with a common beginning (`xl/ops/beams.py`)."""
import ctypes
import functools

import torch

from ..xl.opdef import native
from ..xl.ops.beams import into_and_rule
from .native import _CODE, _c_f, _c_int, _c_ll, _c_p, _count, _sig, _sms, _stream, counters, gemm_error_flag, large_scratch, workspace
from .native_sequence import _f32, _i32, _ptr
from .native_serving import _c_d, _done, _launched, _rows16

_shared_append = _sig("xl_shared_append", _c_p, _c_ll, *[_c_p] * 7, *[_c_int] * 7, _c_f, _c_int, _c_p)
_shared_general = _sig("xl_shared_attn_general", *[_c_p] * 4, _c_ll, _c_p, _c_ll, *[_c_p] * 4, *[_c_int] * 9, _c_f, _c_f, _c_int, _c_p)
_shared_portion = _sig("xl_shared_attn_portion", _c_p, _c_ll, *[_c_p] * 4, _c_ll, *[_c_p] * 4, *[_c_int] * 10, *[_c_f] * 3, _c_p, _c_p)
_shared_groups = _sig("xl_shared_attn_groups", _c_p, _c_ll, *[_c_p] * 4, _c_ll, *[_c_p] * 4, *[_c_int] * 10, *[_c_f] * 3, _c_int, _c_p, _c_p, _c_p)
_shared_groups_scratch = _sig("xl_shared_attn_groups_scratch", *[_c_int] * 5, restype=_c_ll)
_take_beams = _sig("xl_take_beams", *[_c_p] * 16, *[_c_int] * 5, _c_d, *[_c_int] * 5, _c_p)
_take_beams_parts = _sig("xl_take_beams_parts", _c_int, _c_int, _c_int)
_reorder = _sig("xl_reorder", ctypes.POINTER(_c_ll), _c_int, *[_c_p] * 3, _c_int, _c_int, _c_p)


def _on_their_device(fn):
    """A launch goes to the device of its tensors, whatever the current one is."""
    @functools.wraps(fn)
    def launch(*args, **kw):
        devices = {a.device for a in args if isinstance(a, torch.Tensor)}
        if len(devices) != 1:
            raise ValueError(f"the tensors of one call lie on {sorted(map(str, devices))}")
        dev = devices.pop()
        if dev.type != "cuda" or dev.index == torch.cuda.current_device():
            return fn(*args, **kw)
        with torch.cuda.device(dev):
            return fn(*args, **kw)
    return launch


_GROUPS_PARTS = 160 << 20  # bytes that the parts of 2^16 rows of 128 features come to


def _shared_few_rows(B, T, heads, G) -> bool:
    """Whether a portion runs on the kernel that reads shared keys once for a group and leaves parts of sums in memory, and not on the one that has
    whole tiles of a sequence's rows and no parts. Measured with 32 heads on 8 and 4 rows per token, groups against portion: 16 sequences behind 4000
    positions 1 token 42 and 106 us, 8 tokens 76 and 111, 16 tokens 136 and 114; 16 x 8 behind 2000 8 tokens 297 and 422, 16 tokens 567 and 441; 64
    behind 8000 8 tokens 204 and 800, 32 tokens 1004 and 855. Where the two cross depends on how many share how much, which only the device knows: between 9
    and 32 tokens of four rows each there are cases for either. The parts of 2^16 rows of 128 features are 136 MB."""
    return B <= 448 and (T == 1 or T * (heads // G) <= 32) and B * T * heads <= 1 << 16


@native("window_attention_shared_")
@_on_their_device
def window_attention_shared_cuda(proj, q_norm, k_norm, kc, vc, pos, count, lead, shared, joint, T, heads, window, keep_first, scale, sink, eps):
    B, G, smax, dim = kc.shape
    vdim, dt, dev = vc.shape[-1], proj.dtype, proj.device
    plain = (heads + G) * dim + G * vdim
    proj = proj if proj.stride(1) == 1 else proj.contiguous()
    if dt not in _CODE or not (dt == kc.dtype == vc.dtype == joint.dtype) or not _f32(q_norm, k_norm) or not _i32(pos, count, lead, shared):
        return NotImplemented
    if not (proj.is_cuda and joint.is_cuda and kc.is_cuda and vc.is_cuda and kc.is_contiguous() and vc.is_contiguous()) or joint.stride(1) != 1:
        return NotImplemented
    q_norm, k_norm = _rows16(q_norm), _rows16(k_norm)
    gated = proj.shape[1] > plain
    code, s, ld, ldo = _CODE[dt], _stream(), proj.stride(0), joint.stride(0)
    window, keep_first = min(window, smax), min(keep_first, smax)  # no key is further back, and the kernels count in 32 bits
    sink = float("-inf") if sink is None else sink
    norms, caches = (q_norm.data_ptr(), k_norm.data_ptr()), (kc.data_ptr(), vc.data_ptr())
    where = tuple(t.data_ptr() for t in (pos, count, lead, shared))
    sizes = (B, T, heads, G, dim, vdim, smax)

    def append(qn):
        return _shared_append(proj.data_ptr(), ld, *norms, _ptr(qn), *caches, *where[:2], *sizes, eps, code, s)

    if (dt == torch.bfloat16 and dim <= 128 and vdim <= 128 and dim % 8 == vdim % 8 == ld % 8 == ldo % 8 == 0
            and all(t.data_ptr() % 16 == 0 for t in (proj, joint, kc, vc))):
        few = _shared_few_rows(B, T, heads, G)
        # before the first launch: nothing, not even a wait for another stream, may come between that of the append and that of the groups
        scratch = large_scratch(_shared_groups_scratch(B, T, heads, vdim, _sms(dev)) * 4, dev, "shared attention", _GROUPS_PARTS) if few else None
        if not _launched(append(None), "shared_append"):
            return NotImplemented
        args = (proj.data_ptr(), ld, norms[0], *caches, joint.data_ptr(), ldo, *where, *sizes, window, keep_first, int(gated), scale, sink, eps)
        flag = gemm_error_flag(dev).data_ptr()
        if few:
            if _launched(_shared_groups(*args, _sms(dev), scratch.data_ptr(), flag, s), "shared_attn_groups"):
                _count("shared_attn_sum")
                return joint
        rc = _shared_portion(*args, flag, s)
        if rc >= 0:
            _done(rc, "shared_attn_portion")
            return joint
    qn = large_scratch(B * T * heads * dim * 4, dev, "shared queries", 1 << 30)
    if not _launched(append(qn), "shared_append"):
        return NotImplemented
    _done(_shared_general(qn.data_ptr(), *caches, proj.data_ptr() + plain * proj.element_size() if gated else None, ld, joint.data_ptr(), ldo, *where,
                          *sizes, window, keep_first, scale, sink, code, s), "shared_attn_general")
    return joint


@native("take_beams_")
@_on_their_device
def take_beams_cuda(current, parent, logits, buf, parents, step, scores, ended, length, *more, beams, end, valid, length_penalty, base, ahead,
                    advance):
    into, rule = into_and_rule(more)
    to = into or (scores, ended, length)
    if rule and not (_i32(rule[0]) and rule[1].is_cuda and rule[1].dtype == torch.float64):
        return NotImplemented
    rows = logits.shape[0]
    if not logits.is_cuda or logits.dtype not in _CODE or not _i32(current, parent, buf, parents, step, ended, length, to[1], to[2]):
        return NotImplemented
    if not _f32(scores, to[0]) or not all(t.is_cuda and t.is_contiguous() for t in (scores, to[0])):
        return NotImplemented
    logits, dev = logits.contiguous(), logits.device
    parts = _take_beams_parts(rows, beams, valid)
    scratch = workspace(rows * parts * (16 + 8 * beams), dev, "beams")
    done = counters(rows // beams + 1, dev, "counters beams")
    rc = _take_beams(logits.data_ptr(), scores.data_ptr(), ended.data_ptr(), length.data_ptr(), *map(_ptr, to), current.data_ptr(), parent.data_ptr(),
                     buf.data_ptr(), parents.data_ptr(), step.data_ptr(), scratch.data_ptr(), done.data_ptr(), *(map(_ptr, rule or (None, None))),
                     rows, logits.shape[1], valid, beams, end, length_penalty, buf.shape[0], base, ahead, int(advance), _CODE[logits.dtype], _stream())
    return current if _launched(rc, "take_beams") else NotImplemented


def _rows_of(t, axis, per):
    """What the kernel has to know of a state: see `xl_reorder`."""
    size, row = t.element_size(), t.stride(0) * t.element_size()
    if axis is None:
        return (t.data_ptr(), row, 1, 0, 1, t[0].numel() * size, 0)
    inner = 1
    for n in t.shape[axis + 1:]:
        inner *= n
    entries, outer = t.shape[axis], t[0].numel() // (t.shape[axis] * inner)
    return (t.data_ptr(), row, outer, entries * inner * size if outer > 1 else 0, entries, inner * size, per)


@native("reorder_")
@_on_their_device
def reorder_cuda(parent, begin, end, *states, beams, axes, per):
    if not _i32(parent, begin, end) or any(not (t.is_cuda and t.is_contiguous()) for t in states):
        return NotImplemented
    rows = [_rows_of(*s) for s in zip(states, axes, per)]
    if any(r[5] > 0x7fffffff for r in rows):
        return NotImplemented
    for lo in range(0, len(rows), 64):
        now = [x for r in rows[lo:lo + 64] for x in r]
        _done(_reorder((_c_ll * len(now))(*now), len(now) // 7, parent.data_ptr(), begin.data_ptr(), end.data_ptr(), parent.numel(), beams, _stream()),
              "reorder")
    return ()
