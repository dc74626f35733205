"""CUDA implementations of the serving ops (`xl/ops/serving.py`)."""
import ctypes

import torch

from ..xl import read_ahead
from ..xl.opdef import native
from .native import _CODE, _c_f, _c_int, _c_ll, _c_p, _check, _count, _ok, _sig, _sms, _stream, counters, gemm, gemm_error_flag, large_scratch
from .native_sequence import _clamped_glu, _f32, _i32, _ptr, _small, product, stream_rms

_c_d = ctypes.c_double
_shape_logits = _sig("xl_shape_logits", *[_c_p] * 10, *[_c_int] * 7, _c_p)
_take_shaped = _sig("xl_take_shaped", *[_c_p] * 13, *[_c_int] * 11, _c_p)
_append_tokens = _sig("xl_append_tokens", _c_p, _c_p, _c_p, _c_p, _c_int, _c_int, _c_int, _c_p)
_q8_append = _sig("xl_q8_append", _c_p, _c_ll, *[_c_p] * 13, *[_c_int] * 7, _c_d, _c_int, _c_p)
_q8_general = _sig("xl_q8_attn_general", *[_c_p] * 8, _c_ll, _c_p, _c_ll, _c_p, _c_p, *[_c_int] * 9, _c_f, _c_f, _c_int, _c_p)
_q8_few = _sig("xl_q8_attn_few", _c_p, _c_ll, *[_c_p] * 12, _c_ll, _c_p, _c_p, *[_c_int] * 10, _c_f, _c_f, _c_d, _c_int, _c_p, _c_p, _c_int,
               _c_p, _c_p)
_q8_append_expand = _sig("xl_q8_append_expand", _c_p, _c_ll, *[_c_p] * 5, _c_int, *[_c_p] * 3, _c_int, *[_c_p] * 8, *[_c_int] * 9, _c_d, _c_p)
_q8_tcgen05 = _sig("xl_q8_attn_tcgen05", *[_c_p] * 3, _c_int, *[_c_p] * 2, _c_int, *[_c_p] * 6, _c_ll, _c_p, _c_ll, _c_p, _c_p, *[_c_int] * 9, _c_f, _c_f, _c_p, _c_p)
_adapter_down = _sig("xl_adapter_down", *[_c_p] * 5, _c_ll, *[_c_int] * 5, _c_p)
_adapter_up = _sig("xl_adapter_up", *[_c_p] * 5, _c_ll, *[_c_int] * 6, _c_p)
_adapter_down_mma = _sig("xl_adapter_down_mma", *[_c_p] * 5, _c_ll, *[_c_int] * 5, _c_p)
_adapter_up_mma = _sig("xl_adapter_up_mma", *[_c_p] * 5, _c_ll, *[_c_int] * 5, _c_p)


def _launched(rc, name) -> bool:
    """Whether the kernel took its arguments (-1: it does not take such ones)."""
    if rc == -1:
        return False
    _check(rc, name)
    _count(name)
    return True


def _done(rc, name):
    _check(rc, name)
    _count(name)


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


def _rows16(t):
    """The same numbers in rows one after the other from a 16-byte boundary, as the kernels read them; a copy where they lie elsewhere."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rules_ok(history, start, penalties, bias_tokens, bias_values, allowed) -> bool:
    return (_i32(history, start, bias_tokens, allowed) and _f32(penalties, bias_values)
            and all(t.is_cuda and t.is_contiguous() for t in (penalties, bias_values)))


@native("shape_logits")
def shape_logits_cuda(logits, slot, length, *rules):
    logits = _rows16(logits)
    if not _ok(logits) or logits.dim() != 2 or not _i32(slot, length) or not _rules_ok(*rules):
        return NotImplemented
    (rows, V), (slots, L) = logits.shape, rules[0].shape
    out = torch.empty((rows, V), dtype=torch.float32, device=logits.device)
    rc = _shape_logits(logits.data_ptr(), out.data_ptr(), slot.data_ptr(), length.data_ptr(), *map(_ptr, rules), rows, V, slots, L,
                       rules[3].shape[1], rules[5].shape[1], _CODE[logits.dtype], _stream())
    return out if _launched(rc, "shape_logits") else NotImplemented


@native("take_shaped_")
def take_shaped_cuda(current, logits, buf, pos, length, count, *rules, valid, base, ahead, advance):
    logits = _rows16(logits)
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


def _q8_slices(units, longest, per_sm, device) -> int:
    """Into how many CTAs the keys of one unit (sequence, key head, chunk of rows) are cut, at up to `longest` keys: one wave of
    `per_sm` CTAs per SM, three 32-key items for each of a CTA's four warps (32 heads on 8 of 128: one sequence of 8000 keys 22.7, 16.5 and
    18.6 us in 8, 16 and 24 slices, 4 of 4000 17.6, 16.5 and 22.7 in 8, 12 and 16, 16 of 8000 65.7, 54.3 and 66.0 in 2, 3 and 4). Up to
    640 keys the merge costs what it saves (160 units of 600 keys: 16.6 us in 1 and 2 slices, in a window of 256 14.5 and 14.5)."""
    most = per_sm * _sms(device) // units
    if longest <= 640 or most < 2:
        return 1
    return min(most, (longest + 383) // 384, 64)


_Q8_EXPANDED = 2 << 30  # bytes that the codes of a portion may expand to at a time


def _q8_held(T: int, blocks: int, window: int, keep_first: int) -> int:
    """Blocks of codes of one sequence that a portion of T tokens may see, wherever it begins, with its own (q8_slots in attention_q8.cuh)."""
    return min(blocks, -(-keep_first // 64) + (T + window - 1) // 64 + 1) if window else blocks


def _q8_few_rows(rows: int, positions: int, dim: int, vdim: int) -> bool:
    """Whether a portion of `rows` rows per sequence and key head, against a cache of `positions`, runs on mma.sync, which cuts the keys among
    CTAs and reads codes once, and not on the tensor cores, whose keys expand first (2 sequences x 8 key heads of 128 after 6000: 16 rows
    107 us there, 35 here, 64 rows 113 and 58, 128 rows 117 and 83; 6 x 4 heads after 500: 64 rows 37 and 35, 128 rows 39 and 45).
    Features that 16 does not divide have no rows that TMA can take: on the tensor cores, which take multiples of 8, they are faster than on the
    CUDA cores for one token already (2 x 8 key heads of 40 and 24 after 6000: 4 rows 166 -> 107 us, 64 rows 1241 -> 109; 16 x 8 heads of
    72 after 8000: 4 rows 3354 -> 211; 60 x 4 heads after 100: 33 -> 27), all but a few rows against short caches (6 x 4 heads after 500: 24.6 -> 28.7)."""
    return dim % 16 == 0 and vdim % 16 == 0 and (rows <= 64 or (rows <= 128 and positions >= 4096))


def _q8_portion(at, proj, q_norm, k_norm, cache, pos, count, joint, gate, T, heads, held, window, keep_first, scale, sink, eps, s):
    """A portion of the sequences `at` on the tensor cores: append, codes of visible blocks as 16-bit numbers, attention."""
    cache, pos, count = tuple(t[at] for t in cache), pos[at], count[at]
    B, G, blocks, _, dim = cache[0].shape
    vdim, dev, rows = cache[1].shape[-1], proj.device, T + 128
    ld, ldo, row0 = proj.stride(0), joint.stride(0), at.start * T
    q = torch.empty((B, G, T, heads // G, dim), dtype=torch.float16, device=dev)
    raw_k = torch.empty((B, G, rows, dim), dtype=torch.float16, device=dev)
    raw_v = torch.empty((B, G, rows, vdim), dtype=torch.bfloat16, device=dev)
    raw_unit = torch.empty((B, G, (T + 126) // 64), dtype=torch.float32, device=dev)
    codes = large_scratch(B * G * held * 64 * (dim + vdim) * 2, dev, "q8 codes", _Q8_EXPANDED)
    kx = codes.data_ptr()
    vx = kx + B * G * held * 64 * dim * 2
    sizes = (B, T, heads, G, dim, vdim, blocks, window, keep_first)
    norms, where = (q_norm.data_ptr(), k_norm.data_ptr()), (pos.data_ptr(), count.data_ptr())
    rc = _q8_append_expand(proj.data_ptr() + row0 * ld * 2, ld, *norms, q.data_ptr(), raw_k.data_ptr(), raw_v.data_ptr(), rows, raw_unit.data_ptr(),
                           kx, vx, held, *map(_ptr, cache), *where, *sizes, eps, s)
    _done(rc, "q8_append_expand")
    _count("q8_expand")
    rc = _q8_tcgen05(q.data_ptr(), kx, vx, held, raw_k.data_ptr(), raw_v.data_ptr(), rows, raw_unit.data_ptr(), cache[2].data_ptr(),
                     cache[3].data_ptr(), *norms, gate + row0 * ld * 2 if gate else None, ld, joint.data_ptr() + row0 * ldo * 2, ldo, *where, *sizes, scale, sink,
                     gemm_error_flag(dev).data_ptr(), s)
    _done(rc, "q8_attn_tcgen05")


@native("window_attention_q8_")
def window_attention_q8_cuda(proj, q_norm, k_norm, k, v, k_scale, v_scale, k_tail, v_tail, pos, count, joint, T, heads, window,
                             keep_first, scale, sink, eps):
    B, G, blocks, _, dim = k.shape
    vdim, dt, dev = v.shape[-1], proj.dtype, proj.device
    plain = (heads + G) * dim + G * vdim
    proj = proj if proj.stride(1) == 1 else proj.contiguous()
    given, (q_norm, k_norm) = (q_norm, k_norm), (_rows16(q_norm), _rows16(k_norm))
    if not _ok(q_norm, k_norm) or not _f32(q_norm, k_norm, k_scale, v_scale) or not _i32(pos, count) or dt not in _CODE:
        return NotImplemented
    if not (dt == k_tail.dtype == v_tail.dtype == joint.dtype) or joint.stride(1) != 1 or proj.shape[0] != B * T:
        return NotImplemented
    if any(not t.is_contiguous() for t in (k, v, k_scale, v_scale, k_tail, v_tail)) or not (proj.is_cuda and k_tail.is_cuda and joint.is_cuda):
        return NotImplemented
    code, s, ld, ldo = _CODE[dt], _stream(), proj.stride(0), joint.stride(0)
    window, keep_first = min(window, blocks * 64), min(keep_first, blocks * 64)  # no key is further back, and the kernels count in 32 bits
    sink = float("-inf") if sink is None else sink
    gate = proj.data_ptr() + plain * proj.element_size() if proj.shape[1] > plain else None
    cache = tuple(t.data_ptr() for t in (k, v, k_scale, v_scale))
    sizes = (B, T, heads, G, dim, vdim, blocks, window, keep_first)

    def few(q, raw, ahead):
        rows = T * (heads // G)
        per = 8 if rows <= 8 else 16  # rows of a CTA
        units = B * G * -(-rows // per)
        if dim % 16 or vdim % 16 or units > 1 << 16:
            return False
        longest = min(blocks * 64, window + keep_first + T) if window else blocks * 64
        splits = _q8_slices(units, longest, 3 if per == 8 else 2, dev)
        done = counters(units, dev, "counters sequence", 1 << 16)
        part = torch.empty(units * splits * per * (vdim + 2), dtype=torch.float32, device=dev) if splits > 1 else None
        rc = _q8_few(proj.data_ptr(), ld, q_norm.data_ptr(), k_norm.data_ptr(), _ptr(q), _ptr(raw[0]), _ptr(raw[1]), *cache, k_tail.data_ptr(),
                     v_tail.data_ptr(), joint.data_ptr(), ldo, pos.data_ptr(), count.data_ptr(), *sizes, int(gate is not None), scale, sink,
                     eps, splits, _ptr(part), done.data_ptr(), int(ahead), gemm_error_flag(dev).data_ptr(), s)
        return _launched(rc, "q8_attn_few")

    is_few = _q8_few_rows(T * (heads // G), blocks * 64, dim, vdim)
    if T == 1 and dt == torch.bfloat16:
        # (a copy of the factors was written just now)
        ahead = given[0] is q_norm and given[1] is k_norm and read_ahead.allowed(q_norm, k_norm, k, v, k_scale, v_scale, k_tail, v_tail, pos, count)
        if few(None, (None, None), ahead):
            return joint
    aligned = all(t.data_ptr() % 16 == 0 for t in (proj, joint, k, v, k_tail, v_tail))
    held = _q8_held(T, blocks, window, keep_first)
    expanded = G * held * 64 * (dim + vdim) * 2  # bytes of one sequence
    if (dt == torch.bfloat16 and not is_few and aligned and dim <= 128 and vdim <= 128 and dim % 8 == vdim % 8 == ld % 8 == ldo % 8 == 0
            and T * heads <= 1 << 22 and expanded <= _Q8_EXPANDED):
        # as many sequences at a time as expand to what is set aside for it
        step = max(1, _Q8_EXPANDED // expanded)
        step = min(step, (1 << 30) // (G * (T + 128)) + 1, (1 << 30) // (T * heads) + 1, 65535)
        for b in range(0, B, step):
            _q8_portion(slice(b, min(B, b + step)), proj, q_norm, k_norm, (k, v, k_scale, v_scale, k_tail, v_tail), pos, count, joint, gate, T,
                        heads, held, window, keep_first, scale, sink, eps, s)
        return joint
    q = torch.empty((B, G, T, heads // G, dim), dtype=torch.float32, device=dev)
    raw = [torch.empty((B, G, T + 64, width), dtype=dt, device=dev) for width in (dim, vdim)]
    rc = _q8_append(proj.data_ptr(), ld, q_norm.data_ptr(), k_norm.data_ptr(), q.data_ptr(), raw[0].data_ptr(), raw[1].data_ptr(), *cache,
                    k_tail.data_ptr(), v_tail.data_ptr(), pos.data_ptr(), count.data_ptr(), B, T, heads, G, dim, vdim, blocks, eps, code, s)
    if not _launched(rc, "q8_append"):
        return NotImplemented
    if dt == torch.bfloat16 and is_few and few(q, raw, False):
        return joint
    rc = _q8_general(q.data_ptr(), raw[0].data_ptr(), raw[1].data_ptr(), *cache, gate, ld, joint.data_ptr(), ldo, pos.data_ptr(),
                     count.data_ptr(), B, T, heads, G, dim, vdim, blocks, window, keep_first, scale, sink, code, s)
    _done(rc, "q8_attn_general")  # the keys are in the cache: there is no other way from here
    return joint


@native("linear_adapted")
def linear_adapted_cuda(x, weight, a, b, scale, slot, T, out_dtype):
    x = _rows16(x)
    dt, dev = x.dtype, x.device
    (rows, K), N, (n, r, _) = x.shape, weight.shape[0], a.shape
    if not (dt in _CODE and dt == weight.dtype == a.dtype == b.dtype and out_dtype in (dt, torch.float32)):
        return NotImplemented
    if not x.is_cuda or not _f32(scale) or not _i32(slot) or any(not t.is_contiguous() for t in (x, a, b, scale)) or slot.numel() * T != rows:
        return NotImplemented
    if r > 128:  # the kernels hold the numbers between the two products in shared memory
        return NotImplemented
    code, s = _CODE[dt], _stream()
    low = torch.empty((rows, -(-r // 16) * 16), dtype=torch.float32, device=dev)
    down = (x.data_ptr(), a.data_ptr(), scale.data_ptr(), slot.data_ptr(), low.data_ptr(), rows, T, K, n, r, code, s)
    if not (T >= 8 and dt != torch.float32 and _launched(_adapter_down_mma(*down), "adapter_down_mma")):
        if not _launched(_adapter_down(*down), "adapter_down"):
            return NotImplemented
    # 32 bits also where the GEMM needs copies for them: the sum is rounded once
    if dt == torch.float32 or (_small(x, weight) and weight.data_ptr() % 16 == 0):
        y = product(x, weight, torch.float32)
    elif out_dtype == torch.float32:
        y = gemm(x, weight.t(), out_dtype=torch.float32)
    else:  # only for the launches of this op
        y = large_scratch(rows * N * 4, dev, "adapted", 1 << 30)[:rows * N * 4].view(torch.float32).view(rows, N)
        y = gemm(x, weight.t(), out=y)
    if y is NotImplemented:
        return NotImplemented
    if out_dtype == torch.float32:
        out = y
    else:
        out = torch.empty((rows, N), dtype=out_dtype, device=dev)
        if T >= 8 and _launched(_adapter_up_mma(low.data_ptr(), b.data_ptr(), slot.data_ptr(), y.data_ptr(), out.data_ptr(), rows, T, N, n, r, code, s),
                                "adapter_up_mma"):
            return out
    rc = _adapter_up(low.data_ptr(), b.data_ptr(), slot.data_ptr(), y.data_ptr(), out.data_ptr(), rows, T, N, n, r, code, _CODE[out_dtype], s)
    return out if _launched(rc, "adapter_up") else NotImplemented
