"""Ops of a batch whose sequences have a beginning in common: attention over a shared prefix, and beam search's selection and reordering.

Portions, `pos` and `count` are those of the sequence ops (`sequence.py`). A sequence may leave its first positions in the cache of
another slot (its *lead*), which holds them for any number of sequences: beams of one prompt, requests behind one system prompt.

Beams are groups of `beams` consecutive slots. `take_beams_` chooses among all continuations of a group's beams. The best continuation of
a beam stays in the beam's slot and the others take the slots of beams that end there, so that `reorder_` moves only what has to move, and
no row that it reads is one that it writes.

No counterpart in the reference (it ships no cache or generation loop).
"""
from typing import NamedTuple, Optional, Sequence

import torch

from ..core import Tensor
from ..dtypes import bfloat16, float16, float32, float64, int32
from ..opdef import OpDef, emit, emit1
from .decode import _store_row_ref
from .sequence import _rms
from .serving import _expect

MAX_BEAMS = 32          # of a group
MAX_PENALTY = 32        # any number of tokens to this power, 2^992 at most, is a number in 64 bits, and sums divided by it are still unlike each other


class BeamState(NamedTuple):
    """What is known of every beam, each `(rows,)`: `scores` fp32, the sum of the logarithms of its tokens' probabilities (not finite:
    the slot holds no beam), `ended` int32 (not 0: its last token was the end) and `length` int32, its tokens so far."""
    scores: Tensor
    ended: Tensor
    length: Tensor


class BeamRule(NamedTuple):
    """What a choice of beams goes by, held on the device, so that one program serves any: `end (1,)` int32 (a number that is no token: no
    beam ends) and `length_penalty (1,)` float64 (not a number up to `MAX_PENALTY`: none)."""
    end: Tensor
    length_penalty: Tensor


class StateRows(NamedTuple):
    """A state tensor whose first axis is the slots'. `axis`: its axis of positions, of which an entry stands for `per` (None: the whole
    row belongs together)."""
    tensor: Tensor
    axis: Optional[int] = None
    per: int = 1


# ---- references ------------------------------------------------------------------------------------------------------


def shared_edge(pos: torch.Tensor, lead: torch.Tensor, shared: torch.Tensor) -> torch.Tensor:
    """How many positions of every sequence are those of its lead: no more than either of them holds before the op."""
    there = (lead >= 0) & (lead < pos.numel())
    held = pos[lead.long().clamp(0, pos.numel() - 1)]
    return torch.where(there, torch.minimum(torch.minimum(shared, pos), held).clamp(min=0), torch.zeros_like(pos))


def _window_attention_shared_ref(proj, q_norm, k_norm, kc, vc, pos, count, lead, shared, joint, T, heads, window, keep_first, scale, sink, eps):
    if proj.device.type == "meta":
        return torch.empty(joint.shape, dtype=joint.dtype, device="meta")
    B, G, smax, dim = kc.shape
    vdim, dt, dev = vc.shape[-1], proj.dtype, proj.device
    qk, edge, rows = (heads + G) * dim, shared_edge(pos, lead, shared).tolist(), proj.reshape(B, T, -1)
    places = [(int(p), min(int(n), T)) for p, n in zip(pos, count)]
    live = [b for b, (p, n) in enumerate(places) if n > 0 and 0 <= p and p + n <= smax]
    for b in live:
        p, n = places[b]
        k = rows[b, :n, heads * dim:qk].reshape(n, G, dim).double()
        kc[b, :, p:p + n] = (k / torch.sqrt((k * k).mean(-1, keepdim=True) + eps) * k_norm.double()).to(dt).transpose(0, 1)
        vc[b, :, p:p + n] = rows[b, :n, qk:qk + G * vdim].reshape(n, G, vdim).transpose(0, 1)
    for b in live:
        (p, n), e, cur = places[b], edge[b], rows[b]
        q = _rms(cur[:n, :heads * dim].reshape(n, G, heads // G, dim), q_norm, eps)
        keys, vals = (torch.cat((c[int(lead[b]), :, :e] if e else c[b, :, :0], c[b, :, e:p + n]), 1).float() for c in (kc, vc))
        qp, kp = torch.arange(p, p + n, device=dev)[:, None], torch.arange(p + n, device=dev)[None]
        mask = kp <= qp
        if window:
            mask &= (qp - kp < window) | (kp < keep_first)
        known = torch.isfinite(vals)  # a value that is not finite reaches those who see it, and not by a weight of zero
        s = torch.einsum("ngrd,gkd->grnk", q, keys) * scale
        s = s.masked_fill(~known.all(-1)[:, None, None], float("nan")).masked_fill(~mask, float("-inf"))
        if sink is not None:
            s = torch.cat((s, torch.full_like(s[..., :1], sink)), dim=-1)
        o = torch.einsum("grnk,gkv->ngrv", torch.softmax(s, dim=-1)[..., :p + n], vals.masked_fill(~known, 0.0)).reshape(n, heads * vdim)
        if cur.shape[1] > qk + G * vdim:
            o = o * torch.sigmoid(cur[:n, qk + G * vdim:].float())
        joint.reshape(B, T, -1)[b, :n, :heads * vdim] = o.to(joint.dtype)
    return joint


def place_beams(parents: Sequence[int]) -> list:
    """The slot of every continuation, in order of rank, by the slot that it continues (both counted within the group)."""
    free, taken, out = [s for s in range(len(parents)) if s not in set(parents)], set(), []
    for p in parents:
        out.append(free.pop(0) if p in taken else p)
        taken.add(p)
    return out


def into_and_rule(more) -> tuple:
    """The optional tensors of `take_beams_`: those that results go to, three or none, and the rule's, two or none."""
    n = len(more) // 3 * 3
    return more[:n], more[n:]


def _take_beams_ref(current, parent, logits, buf, parents, step, scores, ended, length, *more, beams, end, valid, length_penalty, base, ahead,
                    advance):
    if logits.device.type == "meta":
        return current
    into, rule = into_and_rule(more)
    to_scores, to_ended, to_length = into or (scores, ended, length)
    if rule:
        end, length_penalty = int(rule[0].reshape(-1)[0]), float(rule[1].reshape(-1)[0])
        end, length_penalty = end if 0 <= end < valid else -1, length_penalty if abs(length_penalty) <= MAX_PENALTY else 0.0
    at, dev = int(step.reshape(-1)[0]) + ahead - base, logits.device
    rows = [(t, t[at].clone() if 0 <= at < t.shape[0] else t.new_zeros(t.shape[1])) for t in (buf, parents)]
    for g in range(logits.shape[0] // beams):
        mine = slice(g * beams, (g + 1) * beams)
        score = scores[mine].double()
        score = torch.where(torch.isfinite(score), score, torch.full_like(score, float("-inf")))
        if not torch.isfinite(score).any():
            continue
        done = (ended[mine] != 0) & (end >= 0)
        x = logits[mine, :valid].double()
        x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
        c = score[:, None] + torch.log_softmax(x, 1)
        only = torch.where(torch.arange(valid, device=dev) == end, score[:, None], torch.full_like(c, float("-inf")))
        c = torch.where(done[:, None], only, c)
        c = torch.where(torch.isnan(c), torch.full_like(c, float("-inf")), c)
        after = length[mine] + (~done).int()
        rank = c / after.double().clamp(min=1)[:, None] ** length_penalty
        best = torch.sort(rank.reshape(-1), descending=True, stable=True).indices[:beams]
        p, token = best // valid, best % valid
        slot = g * beams + torch.tensor(place_beams(p.tolist()), device=dev)
        value, was, after = c.reshape(-1)[best].to(scores.dtype), done[p], after[p]
        current.reshape(-1)[slot], parent.reshape(-1)[slot] = token.int(), (g * beams + p).int()
        to_scores[slot], to_ended[slot], to_length[slot] = value, (was | (token == end)).int(), after
        for (_, row), new in zip(rows, (token, g * beams + p)):
            row[slot] = new.int()
    for t, row in rows:
        _store_row_ref(t, step + ahead, row, base)
    if advance:
        step.add_(1)
    return current


def _reorder_ref(parent, begin, end, *states, beams, axes, per):
    if parent.device.type == "meta":
        return ()
    B = parent.numel()
    row = torch.arange(B, device=parent.device)
    inside = (parent >= 0) & (parent < B) & (parent // beams == row // beams)
    source = torch.where(inside, parent.long(), row)
    for x, axis, n in zip(states, axes, per):
        if axis is None:
            x.copy_(x[source].clone())
            continue
        i = torch.arange(x.shape[axis], device=x.device)
        lo, hi = begin.clamp(min=0) // n, (end.clamp(min=0).long() + n - 1) // n
        takes = (i >= lo[:, None]) & (i < hi[:, None]) & (end > begin)[:, None]
        takes = takes.reshape(B, *[1] * (axis - 1), -1, *[1] * (x.dim() - axis - 1))
        x.copy_(torch.where(takes, x[source], x))
    return ()


OpDef("window_attention_shared_", impl=_window_attention_shared_ref, inplace=True)
OpDef("take_beams_", impl=_take_beams_ref, inplace=True)
OpDef("reorder_", impl=_reorder_ref)

# ---- graph functions -------------------------------------------------------------------------------------------------


def window_attention_shared_(proj: Tensor, q_norm: Tensor, k_norm: Tensor, k_cache: Tensor, v_cache: Tensor, pos: Tensor, count: Tensor,
                             lead: Tensor, shared: Tensor, joint: Tensor, T: int, heads: int, scale: float, window: int = 0,
                             keep_first: int = 0, sink: Optional[float] = None, eps: float = 1e-6) -> Tensor:
    """`window_attention_` where the first `shared[b]` positions of sequence `b` are those of slot `lead[b]` (both int32; a lead that is not
    there: none), and the others its own. Nobody shares more than both hold before the op: `min(shared[b], pos[b], pos[lead[b]])`
    positions, which have to be in the lead's own cache. New keys and values go to the sequence's own; norms of keys are taken in 64 bits and rounded
    to 32 and then to the model's type, queries are not rounded to the model's type. A sequence that would not fit the cache is
    left out, rows past `count[b]` are left as they are. A value that is not finite makes those results non-finite (at least in the feature
    concerned) that read its position, and may do so for the other results of a sequence's portion of which some read it; portions that do not are
    not touched.
    On the GPU bf16 models of features up to 128 in multiples of 8 run on the tensor cores, where the keys that a group of sequences shares
    are read once for all of it; all others on the CUDA cores, many times slower."""
    if k_cache.rank != 4 or v_cache.rank != 4:
        raise ValueError("a cache is (batch, heads, positions, features)")
    B, G, smax, dim = k_cache.shape
    vdim = v_cache.shape[-1]
    _expect("k_cache", k_cache, (B, G, smax, dim), proj.dtype)
    _expect("v_cache", v_cache, (B, G, smax, vdim), proj.dtype)
    if k_cache is v_cache:
        raise ValueError("keys and values cannot be held in one tensor")
    if joint is proj:
        raise ValueError("the results cannot lie on top of the projections, which are read until the last one is written")
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
    for what, t in (("pos", pos), ("count", count), ("lead", lead), ("shared", shared)):
        _expect(what, t, (B,), int32)
    if not scale > 0 or window < 0 or keep_first < 0:
        raise ValueError(f"scale ({scale}) must be positive, window ({window}) and keep_first ({keep_first}) not negative")
    return emit1("window_attention_shared_", [proj, q_norm, k_norm, k_cache, v_cache, pos, count, lead, shared, joint],
                 dict(T=int(T), heads=int(heads), window=int(window), keep_first=int(keep_first), scale=float(scale),
                      sink=None if sink is None else float(sink), eps=float(eps)))


def take_beams_(current: Tensor, parent: Tensor, logits: Tensor, buf: Tensor, parents: Tensor, step: Tensor, state: BeamState, beams: int,
                end: Optional[int] = None, valid: Optional[int] = None, length_penalty: float = 0.0, into: Optional[BeamState] = None,
                base: int = 0, ahead: int = 0, advance: bool = True, rule: Optional[BeamRule] = None) -> Tensor:
    """One step of beam search. Row `i` of `logits (rows, vocab)` continues beam `i` of group `i // beams` by every token below `valid`, at
    the sum `scores[i] + log_softmax(logits[i])`; a beam that has ended only by `end`, at the sum that it has. The `beams` continuations of
    a group with the largest `sum / tokens ** length_penalty` are its next beams: token `current[s]` of slot `s` continues slot
    `parent[s]`, and both become row `step + ahead - base` of `buf` and `parents (n, rows)` (ignored when out of range). Of equal ones the
    lowest slot and then the lowest token is taken. The best continuation of a beam keeps its slot, the others take the free ones, in
    order of rank. Sums are compared in 64 bits (on the GPU those of a row are formed from exponentials in 32, and again in 64 where the choice
    hangs on it) and kept in 32, in `into` (default: `state` itself). Without `end` no beam ends, whatever `ended` holds. `rule`: `end` and
    `length_penalty` are those that the device holds. NaN among logits counts as minus infinity; where too few continuations are finite those
    at minus infinity follow. A group without a finite score is left as it is, and its rows, like those of beams that have ended, are not read. With
    `advance`, `step` moves on by one."""
    rows, valid = (logits.shape[0] if logits.rank == 2 else 0), int(logits.shape[-1] if valid is None else valid)
    if logits.rank != 2 or logits.dtype not in (float32, float16, bfloat16):
        raise ValueError(f"logits are rows of floating-point numbers, not {tuple(logits.shape)} {logits.dtype}")
    if not 1 <= beams <= MAX_BEAMS or rows < 1 or rows % beams:
        raise ValueError(f"{rows} rows are not groups of {beams} beams (1 to {MAX_BEAMS})")
    if not 1 <= valid <= logits.shape[1] or valid * beams > 0x7fffffff:
        raise ValueError(f"a choice among {valid} entries from rows of {logits.shape[1]}")
    if end is not None and not 0 <= end < valid:
        raise ValueError(f"the end is a token below {valid}, not {end}")
    if not abs(length_penalty) <= MAX_PENALTY:
        raise ValueError(f"a length penalty is a number up to {MAX_PENALTY}, not {length_penalty}")
    if rule is not None:
        if end is not None or length_penalty:
            raise ValueError("a choice goes by a rule that the device holds, or by an end and a length penalty given here")
        _expect("rule.end", rule.end, (1,), int32)
        _expect("rule.length_penalty", rule.length_penalty, (1,), float64)
    for what, s in (("state", state), ("into", into)):
        for field, t, dt in zip(BeamState._fields, s or (), (float32, int32, int32)):
            _expect(f"{what}.{field}", t, (rows,), dt)
    for what, t in (("current", current), ("parent", parent)):
        _expect(what, t, (rows,), int32)
    if any(t.rank != 2 or t.shape[1] != rows or t.dtype != int32 for t in (buf, parents)) or buf.shape != parents.shape:
        raise ValueError(f"the choices of {rows} beams are kept in rows of two int32 buffers, not {tuple(buf.shape)} and {tuple(parents.shape)}")
    written = [current, parent, buf, parents, step, *(into or state), *(rule or ())[:1]]
    if len({id(t) for t in written}) < len(written):
        raise ValueError("the results of a choice go to tensors of their own")
    if step.dtype != int32 or step.nelms != 1:
        raise ValueError(f"the choices of a step have one position in int32, not {tuple(step.shape)} {step.dtype}")
    return emit1("take_beams_", [current, parent, logits, buf, parents, step, *state, *(into or ()), *(rule or ())],
                 dict(beams=int(beams), end=-1 if end is None else int(end), valid=valid, length_penalty=float(length_penalty), base=int(base),
                      ahead=int(ahead), advance=bool(advance)))


def reorder_(states: Sequence[StateRows], parent: Tensor, begin: Tensor, end: Tensor, beams: int) -> None:
    """Positions `begin[b]` to `end[b] - 1` of row `b` of every state become those of row `parent[b]` (all int32), as all rows were before
    the op; states without positions are taken whole. Rows are groups of `beams` consecutive ones, and a row whose parent is not of its
    own group is left as it is. An entry that stands for several positions is taken whole if one of them is meant."""
    states = list(states)
    if not states:
        return
    B = parent.shape[0] if parent.rank == 1 else 0
    if not 1 <= beams <= MAX_BEAMS or B < 1 or B % beams:
        raise ValueError(f"{tuple(parent.shape)} parents are not groups of {beams} rows (1 to {MAX_BEAMS})")
    for what, t in (("parent", parent), ("begin", begin), ("end", end)):
        _expect(what, t, (B,), int32)
    for s in states:
        if s.tensor.rank < 1 or s.tensor.shape[0] != B or 0 in s.tensor.shape:
            raise ValueError(f"a state of {B} rows cannot be {tuple(s.tensor.shape)}")
        if s.axis is not None and not (1 <= s.axis < s.tensor.rank and s.per >= 1):
            raise ValueError(f"positions of {tuple(s.tensor.shape)} cannot lie along axis {s.axis}, {s.per} to an entry")
        if s.tensor in (parent, begin, end) or sum(s.tensor is o.tensor for o in states) > 1:
            raise ValueError(f"{s.tensor} is given twice")
    emit("reorder_", [parent, begin, end, *(s.tensor for s in states)],
         dict(beams=int(beams), axes=tuple(s.axis for s in states), per=tuple(int(s.per) for s in states)))
