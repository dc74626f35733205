"""Ops of a serving step for a batch of unlike requests: attention against a cache held in 8 bits, projections with an adapter
of each request's own, and logits shaped by penalties, biases and masks before a token is chosen.

Portions, `pos` and `count` are those of the sequence ops (`sequence.py`): `batch * T` rows, sequence-major, of which the first
`count[b]` of sequence `b` are real, at positions `pos[b]` and on.

The cache (`Cache8`) holds keys and values in blocks of `CACHE8_BLOCK` tokens. A block that is complete is held as codes of 8
bits with one scale per block and head: `value = code * scale`, `scale` a 127th of the block's largest absolute value, `code` the
nearest whole number (of a block that is not finite throughout: scale NaN, codes zero). The block in progress is held as it was
computed, in the tail. A position sees its own block as it was computed and earlier blocks as the cache holds them, whatever portions
a prompt is cut into, and a code depends on nothing but the block: norms of keys are taken in 64 bits and rounded once, so that
every kernel, and the CPU, comes to the same codes.
Positions only move forward: a sequence may go back to a multiple of `CACHE8_BLOCK`, but not into a block that is complete.

No counterpart in the reference (it ships no cache or generation loop).
"""
from typing import Dict, NamedTuple, Optional, Tuple

import torch

from ..core import Tensor
from ..dtypes import bfloat16, dtype as _dtype, float16, float32, int32, int8
from ..opdef import OpDef, emit, emit1
from .decode import _store_row_ref
from .sequence import _mm, _rms

CACHE8_BLOCK = 64    # tokens that share a scale
MAX_RANK = 128       # of an adapter
MAX_BIASES = 1024    # entries of a slot's list
MAX_HISTORY = (1 << 20) - 1


class Cache8(NamedTuple):
    """Keys and values of one layer: codes `(batch, G, blocks, CACHE8_BLOCK, dim)` int8, scales `(batch, G, blocks)` fp32, tails
    `(batch, G, CACHE8_BLOCK, dim)` in the model's type."""
    k: Tensor
    v: Tensor
    k_scale: Tensor
    v_scale: Tensor
    k_tail: Tensor
    v_tail: Tensor


class Adapters(NamedTuple):
    """Low-rank adapters of one projection, `scale[i] * (x @ a[i]^T) @ b[i]^T`: `a (n, rank, K)`, `b (n, N, rank)` in the model's
    type, `scale (n,)` fp32. Smaller ranks are filled up with zeros."""
    a: Tensor
    b: Tensor
    scale: Tensor


class LogitRules(NamedTuple):
    """What shapes the logits of every slot. `history (slots, length)` int32 holds its tokens by position and `start (slots,)` how
    many of them came with the prompt; `penalties (slots, 3)` fp32: repetition, frequency, presence; `bias_tokens`, `bias_values
    (slots, n)`: what is added to single tokens (-1: no token); `allowed (slots, words)` int32: bit `i % 32` of word `i // 32` is
    set where token `i` may be chosen."""
    history: Tensor
    start: Tensor
    penalties: Tensor
    bias_tokens: Tensor
    bias_values: Tensor
    allowed: Tensor


# ---- references ------------------------------------------------------------------------------------------------------


def quantize_block(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of complete blocks `(..., CACHE8_BLOCK, width)`. Divisions are true divisions: a product with the
    reciprocal would come to other codes next to a border. A block that holds a number that is not finite: scale NaN, codes zero."""
    x = x.float()
    top = x.abs().amax((-2, -1))
    scale = torch.where(torch.isfinite(top), top / torch.full_like(top, 127.0), torch.full_like(top, float("nan")))
    code = torch.where(scale[..., None, None] > 0, (x / scale[..., None, None]).round(), torch.zeros_like(x))
    return code.clamp(-127, 127).to(torch.int8), scale


def _window_attention_q8_ref(proj, q_norm, k_norm, k, v, k_scale, v_scale, k_tail, v_tail, pos, count, joint, T, heads, window,
                             keep_first, scale, sink, eps):
    if proj.device.type == "meta":
        return torch.empty(joint.shape, dtype=joint.dtype, device="meta")
    B, G, blocks, size, dim = k.shape
    vdim, dt, dev, R = v.shape[-1], proj.dtype, proj.device, heads // G
    qk = (heads + G) * dim
    for b in range(B):
        p, n = int(pos[b]), min(int(count[b]), T)
        if n <= 0 or p < 0 or p + n > blocks * size:
            continue
        cur, first = proj.reshape(B, T, -1)[b, :n], p // size * size
        q = _rms(cur[:, :heads * dim].reshape(n, G, R, dim), q_norm, eps)
        kd = cur[:, heads * dim:qk].reshape(n, G, dim).double()
        kd = kd / torch.sqrt((kd * kd).mean(-1, keepdim=True) + eps) * k_norm.double()
        new = {"k": kd.to(dt).transpose(0, 1), "v": cur[:, qk:qk + G * vdim].reshape(n, G, vdim).transpose(0, 1)}
        raw, cached, end = {}, {}, p + n - first
        for name, codes, scales, tail in (("k", k, k_scale, k_tail), ("v", v, v_scale, v_tail)):
            raw[name] = torch.cat((tail[b, :, :p - first], new[name]), 1)  # from the start of the block in progress
            for j in range(end // size):
                codes[b, :, first // size + j], scales[b, :, first // size + j] = quantize_block(
                    raw[name][:, j * size:(j + 1) * size])
            tail[b, :, :end % size] = raw[name][:, end // size * size:]
            done = (first + end) // size
            cached[name] = (codes[b, :, :done].float() * scales[b, :, :done, None, None]).flatten(1, 2)
        gate = cur[:, qk + G * vdim:].float() if cur.shape[1] > qk + G * vdim else None
        for lo in range(first, p + n, size):  # the queries of one block
            i0, i1 = max(lo, p), min(lo + size, p + n)
            keys, vals = (torch.cat((cached[x][:, :lo], raw[x][:, lo - first:i1 - first].float()), 1) for x in "kv")
            qp, kp = torch.arange(i0, i1, device=dev)[:, None], torch.arange(0, i1, device=dev)[None]
            mask = kp <= qp
            if window:
                mask &= (qp - kp < window) | (kp < keep_first)
            s = torch.einsum("ngrd,gkd->grnk", q[i0 - p:i1 - p], keys) * scale
            known = torch.isfinite(vals)  # a value that is not finite reaches those who see it, and not by a weight of zero
            s = s.masked_fill(~known.all(-1)[:, None, None], float("nan"))
            vals = vals.masked_fill(~known, 0.0)
            s = s.masked_fill(~mask, float("-inf"))
            if sink is not None:
                s = torch.cat((s, torch.full_like(s[..., :1], sink)), dim=-1)
            o = torch.einsum("grnk,gkv->ngrv", torch.softmax(s, dim=-1)[..., :i1], vals).reshape(i1 - i0, heads * vdim)
            if gate is not None:
                o = o * torch.sigmoid(gate[i0 - p:i1 - p])
            joint.reshape(B, T, -1)[b, i0 - p:i1 - p, :heads * vdim] = o.to(joint.dtype)
    return joint


def _linear_adapted_ref(x, weight, a, b, scale, slot, T, out_dtype):
    if x.device.type == "meta":
        return torch.empty((x.shape[0], weight.shape[0]), dtype=out_dtype, device="meta")
    y = _mm(x, weight)
    for i, s in enumerate(slot.tolist()):
        if 0 <= s < a.shape[0]:
            y[i * T:(i + 1) * T] += scale[s] * _mm(_mm(x[i * T:(i + 1) * T], a[s]), b[s])
    return y.to(out_dtype)


def _split_glu_ref(y, cols, lead, limit, slope, shift):
    n, f = y.shape[0], (y.shape[1] - cols) // 2
    if y.device.type == "meta":
        return [torch.empty((n, c), dtype=y.dtype, device="meta") for c in (cols, lead + f)]
    g, u = y[:, cols:cols + f].float().clamp(max=limit), y[:, cols + f:].float().clamp(-limit, limit)
    joint = torch.zeros((n, lead + f), dtype=y.dtype, device=y.device)
    joint[:, lead:] = (g * torch.sigmoid(slope * g) * (u + shift)).to(y.dtype)
    return y[:, :cols], joint


def _residual_rms_ref(x, y, *norm, mult, eps):
    n = y.shape[0]
    if x.device.type == "meta":
        return torch.empty((n, x.shape[1]), dtype=y.dtype, device="meta") if norm else ()
    x[:n] += mult * y.float()
    return _rms(x[:n], norm[0], eps).to(y.dtype) if norm else ()


def _shaped_row(x, length, history, start, penalties, bias_tokens, bias_values, allowed):
    """One row of fp32 logits under the rules of its slot."""
    V, dev = x.numel(), x.device
    past = history[:max(0, min(int(length), history.numel()))].long()
    drawn = past[max(0, int(start)):]
    times, seen = (torch.bincount(h[(h >= 0) & (h < V)], minlength=V) for h in (drawn, past))
    repetition, frequency, presence = penalties.float()
    x = torch.where(seen > 0, torch.where(x > 0, x / repetition, x * repetition), x)
    x = torch.where(times > 0, x - frequency * times - presence, x)
    bias, listed = torch.zeros_like(x), torch.zeros(V, dtype=torch.bool, device=dev)
    for t, value in zip(bias_tokens.tolist(), bias_values):
        if 0 <= t < V:
            bias[t] += value
            listed[t] = True
    x = torch.where(listed, x + bias, x)
    at = torch.arange(V, device=dev)
    return torch.where((allowed[at // 32] >> (at % 32).int()) & 1 > 0, x, torch.full_like(x, float("-inf")))


def _shape_logits_ref(logits, slot, length, *rules):
    if logits.device.type == "meta":
        return torch.empty(logits.shape, dtype=torch.float32, device="meta")
    out = logits.float().clone()
    for i, s in enumerate(slot.tolist()):
        if 0 <= s < rules[0].shape[0]:
            out[i] = _shaped_row(out[i], length[i], *(r[s] for r in rules))
    return out


def _take_shaped_ref(current, logits, buf, pos, length, count, *rules, valid, base, ahead, advance):
    if logits.device.type == "meta":
        return current
    history, row = rules[0], buf.new_zeros(buf.shape[1])
    at = int(pos.reshape(-1)[0]) + ahead - base
    if 0 <= at < buf.shape[0]:
        row = buf[at].clone()
    for b in range(logits.shape[0]):
        if int(count[b]) <= 0:
            continue
        x = _shaped_row(logits[b, :valid].float(), length[b], *(r[b] for r in rules))
        x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)  # NaN is never chosen
        token = int((x == x.max()).int().argmax())
        current.reshape(-1)[b] = token
        row[b] = token
        if 0 <= int(length[b]) < history.shape[1]:
            history[b, int(length[b])] = token
    _store_row_ref(buf, pos + ahead, row, base)
    if advance:
        pos.add_(1)
    return current


def _append_tokens_ref(history, tokens, pos, count, T):
    if history.device.type == "meta":
        return history
    for b in range(history.shape[0]):
        p, n = int(pos[b]), min(int(count[b]), T)
        for t in range(n):
            if 0 <= p + t < history.shape[1]:
                history[b, p + t] = tokens.reshape(-1)[b * T + t]
    return history


OpDef("window_attention_q8_", impl=_window_attention_q8_ref, inplace=True)
OpDef("linear_adapted", impl=_linear_adapted_ref)
OpDef("split_glu", impl=_split_glu_ref)
OpDef("residual_rms_", impl=_residual_rms_ref)
OpDef("shape_logits", impl=_shape_logits_ref)
OpDef("take_shaped_", impl=_take_shaped_ref, inplace=True)
OpDef("append_tokens_", impl=_append_tokens_ref, inplace=True)

# ---- graph functions -------------------------------------------------------------------------------------------------


def _expect(what: str, t: Tensor, shape, dt: Optional[_dtype] = None):
    if tuple(t.shape) != tuple(shape) or (dt is not None and t.dtype != dt):
        raise ValueError(f"{what} must be {tuple(shape)}{f' {dt}' if dt is not None else ''}, not {tuple(t.shape)} {t.dtype}")


def cache8_spec(batch: int, kv_heads: int, max_seq: int, dim: int, vdim: int, dtype: _dtype) -> Dict[str, tuple]:
    """Shapes and types of the tensors of a `Cache8` that holds `max_seq` positions, by field."""
    blocks = -(-max_seq // CACHE8_BLOCK)
    lead = (batch, kv_heads)
    return {"k": ((*lead, blocks, CACHE8_BLOCK, dim), int8), "v": ((*lead, blocks, CACHE8_BLOCK, vdim), int8),
            "k_scale": ((*lead, blocks), float32), "v_scale": ((*lead, blocks), float32),
            "k_tail": ((*lead, CACHE8_BLOCK, dim), dtype), "v_tail": ((*lead, CACHE8_BLOCK, vdim), dtype)}


def window_attention_q8_(proj: Tensor, q_norm: Tensor, k_norm: Tensor, cache: Cache8, pos: Tensor, count: Tensor, joint: Tensor,
                         T: int, heads: int, scale: float, window: int = 0, keep_first: int = 0, sink: Optional[float] = None,
                         eps: float = 1e-6) -> Tensor:
    """`window_attention_` against a cache of 8 bits: `proj` rows are `[q: heads x dim | k: G x dim | v: G x vdim | gate: heads x
    vdim]` (the gate may be absent), every query and key head gets an RMS norm, keys and values join the cache, and the gated
    attention goes to the first `heads * vdim` columns of `joint`. A sequence that would not fit the cache is left out, rows past
    `count[b]` are left as they are. A key or value that is not finite has no code: the scale of its block becomes NaN, and with it the
    results, for the heads that share the key, of every later position that reads the block. Of the block's own positions those that see the
    token become NaN or infinite in at least the feature concerned; the others may, in the portion that brings it. No position that does not
    read the block is touched. On the GPU bf16 models whose features are multiples of 8 (16 for the fastest steps) up to 128, with
    projections and `joint` rows on 16-byte boundaries, run on the tensor cores; all others on the CUDA cores, many times slower."""
    if cache.k.rank != 5 or cache.v.rank != 5:
        raise ValueError("the codes of a cache are (batch, heads, blocks, tokens, features)")
    B, G, blocks, _, dim = cache.k.shape
    vdim = cache.v.shape[-1]
    for (field, (shape, dt)), t in zip(cache8_spec(B, G, blocks * CACHE8_BLOCK, dim, vdim, proj.dtype).items(), cache):
        _expect(f"cache.{field}", t, shape, dt)
    if max(dim, vdim) > 512:
        raise ValueError(f"the attention kernels take dim and vdim up to 512, not {dim} and {vdim}")
    if heads < 1 or heads % G:
        raise ValueError(f"heads ({heads}) must be a multiple of the cache's {G} heads")
    plain = (heads + G) * dim + G * vdim
    if T < 1 or proj.rank != 2 or proj.shape[0] != B * T or proj.shape[1] not in (plain, plain + heads * vdim):
        raise ValueError(f"projections of {B} sequences x {T} tokens are ({B * T}, {plain}) or, with gates, ({B * T}, "
                         f"{plain + heads * vdim}), not {tuple(proj.shape)}")
    if joint.rank != 2 or joint.shape[0] != B * T or joint.shape[1] < heads * vdim or joint.dtype != proj.dtype:
        raise ValueError(f"the joint buffer needs {B * T} rows of {heads * vdim} columns or more in {proj.dtype}")
    for what, t, n in (("q_norm", q_norm, dim), ("k_norm", k_norm, dim)):
        _expect(what, t, (n,), float32)
    _expect("pos", pos, (B,), int32)
    _expect("count", count, (B,), int32)
    if not scale > 0 or window < 0 or keep_first < 0:
        raise ValueError(f"scale ({scale}) must be positive, window ({window}) and keep_first ({keep_first}) not negative")
    return emit1("window_attention_q8_", [proj, q_norm, k_norm, *cache, pos, count, joint],
                 dict(T=int(T), heads=int(heads), window=int(window), keep_first=int(keep_first), scale=float(scale),
                      sink=None if sink is None else float(sink), eps=float(eps)))


def linear_adapted(x: Tensor, weight: Tensor, adapters: Adapters, slot: Tensor, T: int = 1, dtype: Optional[_dtype] = None) -> Tensor:
    """`x (batch * T, K) @ weight (N, K)^T` plus, for the rows of sequence `b`, the adapter `slot[b]` (int32; one that is not there
    adds nothing). Both products and their sum are accumulated in 32 bits and rounded once, to `dtype` (default: that of `x`)."""
    if x.rank != 2 or weight.rank != 2 or x.shape[1] != weight.shape[1] or x.dtype != weight.dtype:
        raise ValueError(f"cannot multiply {tuple(x.shape)} {x.dtype} by the transpose of {tuple(weight.shape)} {weight.dtype}")
    n, rank = adapters.a.shape[0], adapters.a.shape[1]
    if not 1 <= rank <= MAX_RANK:
        raise ValueError(f"adapters have between 1 and {MAX_RANK} numbers between their products, not {rank}")
    _expect("adapters.a", adapters.a, (n, rank, x.shape[1]), x.dtype)
    _expect("adapters.b", adapters.b, (n, weight.shape[0], rank), x.dtype)
    _expect("adapters.scale", adapters.scale, (n,), float32)
    if T < 1 or slot.rank != 1 or slot.dtype != int32 or x.shape[0] != slot.shape[0] * T:
        raise ValueError(f"sequences of {T} tokens with slots {tuple(slot.shape)} {slot.dtype} do not make {x.shape[0]} rows")
    return emit1("linear_adapted", [x, weight, *adapters, slot], dict(T=int(T), out_dtype=(dtype or x.dtype).as_torch()))


def split_glu(y: Tensor, cols: int, lead: int, limit: float, slope: float = 1.0, shift: float = 0.0) -> Tuple[Tensor, Tensor]:
    """The second half of `linear_split_glu`, for a product `y (n, cols + 2 F)` that is there already."""
    if y.rank != 2 or cols < 0 or lead < 0 or y.shape[1] < cols or (y.shape[1] - cols) % 2:
        raise ValueError(f"rows of {cols} columns with as many of gate and up behind them, and {lead} columns in front of the unit, do not "
                         f"make {tuple(y.shape)}")
    return tuple(emit("split_glu", [y], dict(cols=int(cols), lead=int(lead), limit=float(limit), slope=float(slope), shift=float(shift))))


def residual_rms_(x: Tensor, y: Tensor, norm: Optional[Tensor] = None, eps: float = 1e-6, mult: float = 1.0) -> Optional[Tensor]:
    """The second half of `linear_residual_rms_`: `x += mult * y` on the fp32 residual stream; with `norm`, returns the RMS norm of
    the updated rows in the type of `y`."""
    if x.rank != 2 or y.rank != 2 or x.dtype != float32 or x.shape[1] != y.shape[1] or y.shape[0] > x.shape[0]:
        raise ValueError(f"{tuple(y.shape)} cannot be added to the first rows of the residual stream {tuple(x.shape)} {x.dtype} (float32)")
    if norm is not None:
        _expect("norm", norm, (x.shape[1],), float32)
    out = emit("residual_rms_", [x, y] + ([norm] if norm is not None else []), dict(mult=float(mult), eps=float(eps)))
    return out[0] if norm is not None else None


def _check_rules(rules: LogitRules, logits: Tensor, vocab: Optional[int] = None):
    if logits.rank != 2 or logits.dtype not in (float32, float16, bfloat16):
        raise ValueError(f"logits are rows of floating-point numbers, not {tuple(logits.shape)} {logits.dtype}")
    vocab = vocab or logits.shape[1]
    for what, t, dt in zip(rules._fields, rules, (int32, int32, float32, int32, float32, int32)):
        if t.dtype != dt or t.rank != (1 if what == "start" else 2):
            raise ValueError(f"rules.{what} must be {'one row' if what == 'start' else 'rows'} of {dt}, not {tuple(t.shape)} {t.dtype}")
    if rules.history.shape[1] > MAX_HISTORY or rules.bias_tokens.shape[1] > MAX_BIASES:
        raise ValueError(f"rules hold at most {MAX_HISTORY} tokens and {MAX_BIASES} biases of a slot, not {rules.history.shape[1]} and "
                         f"{rules.bias_tokens.shape[1]}")
    slots = rules.history.shape[0]
    for what, t, tail in (("start", rules.start, ()), ("penalties", rules.penalties, (3,)), ("bias_tokens", rules.bias_tokens, rules.bias_tokens.shape[1:]),
                          ("bias_values", rules.bias_values, rules.bias_tokens.shape[1:])):
        _expect(f"rules.{what}", t, (slots, *tail))
    if rules.allowed.shape[0] != slots or rules.allowed.shape[1] * 32 < vocab:
        raise ValueError(f"rules.allowed must hold {slots} rows of {-(-vocab // 32)} words, not {tuple(rules.allowed.shape)}")


def shape_logits(logits: Tensor, slot: Tensor, length: Tensor, rules: LogitRules) -> Tensor:
    """fp32 logits `(n, vocab)` under the rules of slot `slot[i]` after its first `length[i]` tokens (a slot that is not there: as
    they are). In this order: tokens that occurred are divided by the repetition penalty where positive, else multiplied by it;
    the frequency penalty is subtracted for every time a token occurred since the prompt, the presence penalty once; biases are
    added; what is not allowed becomes minus infinity. A row that allows nothing is minus infinity throughout."""
    _check_rules(rules, logits)
    if any(t.shape != (logits.shape[0],) or t.dtype != int32 for t in (slot, length)):
        raise ValueError(f"{logits.shape[0]} rows of logits need as many slots and lengths in int32, not {tuple(slot.shape)} {slot.dtype} and "
                         f"{tuple(length.shape)} {length.dtype}")
    return emit1("shape_logits", [logits, slot, length, *rules])


def take_shaped_(current: Tensor, logits: Tensor, buf: Tensor, pos: Tensor, length: Tensor, count: Tensor, rules: LogitRules,
                 valid: Optional[int] = None, base: int = 0, ahead: int = 0, advance: bool = True) -> Tensor:
    """`take_greedy_` on shaped logits: the choice of row `b`, whose rules are those of slot `b` after `length[b]` tokens, becomes
    `current[b]`, row `pos + ahead - base` of `buf` and token `length[b]` of the history. Rows with `count[b] <= 0` are left out.
    Of equal logits the lowest index is chosen (index 0 where nothing is allowed)."""
    valid = int(valid or logits.shape[-1])
    _check_rules(rules, logits, valid)
    rows = logits.shape[0]
    if rules.history.shape[0] != rows or any(t.shape != (rows,) or t.dtype != int32 for t in (length, count)):
        raise ValueError(f"{rows} rows of logits need as many slots, lengths and counts in int32")
    if not 1 <= valid <= logits.shape[1]:
        raise ValueError(f"a choice among {valid} entries from rows of {logits.shape[1]}")
    if current.dtype != int32 or pos.dtype != int32 or buf.dtype != int32 or buf.rank != 2 or not current.nelms == buf.shape[1] == rows:
        raise ValueError(f"{rows} choices go to as many int32 numbers and rows of a buffer, not {tuple(current.shape)} and {tuple(buf.shape)}")
    if pos.nelms != 1:
        raise ValueError(f"the choices of a step have one position, not {tuple(pos.shape)}")
    return emit1("take_shaped_", [current, logits, buf, pos, length, count, *rules],
                 dict(valid=valid, base=int(base), ahead=int(ahead), advance=bool(advance)))


def append_tokens_(history: Tensor, tokens: Tensor, pos: Tensor, count: Tensor, T: int) -> Tensor:
    """The real tokens of a portion, `tokens (batch * T,)`, take their places in `history (batch, length)`; places past its end are
    dropped."""
    if T < 1 or history.rank != 2 or tokens.nelms != history.shape[0] * T:
        raise ValueError(f"{tuple(tokens.shape)} tokens are not portions of {T} for {history.shape[0]} sequences")
    if history.dtype != int32 or tokens.dtype != int32:
        raise ValueError(f"tokens are held in int32, not in {tokens.dtype} and {history.dtype}")
    for what, t in (("pos", pos), ("count", count)):
        _expect(what, t, (history.shape[0],), int32)
    return emit1("append_tokens_", [history, tokens, pos, count], dict(T=int(T)))
