"""Operators of a batch whose sequences have a beginning in common, each as a user's program calls it and in a plain form.

* `attention`: sliding-window attention of a portion of tokens where the first positions of a sequence lie in the cache of another one:
  beams of a prompt, requests behind one system prompt.
* `beams`: beam search's selection over all beams and tokens of a prompt. The best continuation of a beam keeps the beam's slot, others
  take the slots of beams that end here.
* `reorder`: what the beams hold follows the selection.

Plain forms are elementary torch operations in 32 bits (norms of keys and the selection's sums, whose rounding decides on what is stored or
chosen, in 64), rounded once at the end. `exact` has the same results in 64 bits, sequence by sequence.
"""
import math

import torch

own = False  # whether `run` makes the calls of the framework

EPS = 1e-6
SINK = 0.0


# ---------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------


def _attention(groups, per, T, heads, kv_heads, dim, vdim, prefix, tokens, window=0, keep=4, dtype="bfloat16", ragged=True):
    """`groups` prefixes of about `prefix` positions, `per` sequences behind each, with about `tokens` of their own."""
    return dict(kind="attention", groups=groups, per=per, T=T, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, prefix=prefix, tokens=tokens,
                window=window, keep=keep if window else 0, dtype=dtype, ragged=ragged)


def _beams(groups, beams, vocab, dtype="float32", penalty=0.0, first=False):
    return dict(kind="beams", groups=groups, beams=beams, vocab=vocab, dtype=dtype, penalty=penalty, first=first)


def _reorder(groups, beams, layers, kv_heads, dim, prompt, tokens, room, cache="model", dtype="bfloat16"):
    return dict(kind="reorder", groups=groups, beams=beams, layers=layers, kv_heads=kv_heads, dim=dim, prompt=prompt, tokens=tokens, room=room,
                cache=cache, dtype=dtype)


def listed():
    return [
        # four beams of one short prompt: latency
        dict(_attention(1, 4, 1, 16, 4, 128, 128, 200, 17, ragged=False), name="attn_single"),
        # eight beams for each of sixteen documents
        dict(_attention(16, 8, 1, 32, 8, 128, 128, 2000, 130), name="attn_beams"),
        # requests behind one long system prompt
        dict(_attention(1, 64, 1, 32, 8, 128, 128, 8000, 700), name="attn_system"),
        # the prompts of requests behind a system prompt, in one portion
        dict(_attention(1, 16, 250, 32, 8, 128, 128, 4000, 0), name="attn_portion"),
        # beams of a 32-bit model, a window next to the first tokens
        dict(_attention(2, 4, 1, 8, 2, 128, 128, 215, 40, 128, dtype="float32"), name="attn_float32"),
        # one prompt's beams
        dict(_beams(1, 4, 32000), name="beams_single"),
        # a large batch, some beams ended, hypotheses ranked by a length penalty
        dict(_beams(48, 8, 50400, penalty=0.8), name="beams_batch"),
        # logits in the model's type, many beams
        dict(_beams(16, 16, 32000, dtype="bfloat16"), name="beams_wide"),
        # one prompt's beams in the caches of four layers
        dict(_reorder(1, 4, 4, 4, 128, 200, 17, 512), name="reorder_single"),
        # a large batch, eight layers
        dict(_reorder(32, 8, 8, 8, 128, 200, 230, 512), name="reorder_batch"),
        # caches in 8 bits
        dict(_reorder(16, 4, 6, 8, 128, 300, 700, 1024, cache="int8"), name="reorder_int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["attention", "attention", "attention", "beams", "beams", "reorder", "reorder"])
    if kind == "attention":
        dim, vdim = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 80), (40, 24)])
        kv_heads, each = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8])
        window = rng.choice([0, 0, _log(rng, 32, 4096)])
        if rng.random() < 0.15:
            return _attention(_log(rng, 1, 3), _log(rng, 2, 4), rng.choice([1, 1, _log(rng, 2, 48)]), kv_heads * each, kv_heads, dim, vdim,
                              _log(rng, 4, 600), rng.randint(1, 60), window, rng.randint(0, 8), "float32")
        if rng.random() < 0.65:
            groups = _log(rng, 1, 16)
            return _attention(groups, _log(rng, 2, 96 // groups if groups > 4 else 64), 1, kv_heads * each, kv_heads, dim, vdim, _log(rng, 4, 8000),
                              _log(rng, 1, 1000), window, rng.randint(0, 70), ragged=rng.random() < 0.7)
        return _attention(_log(rng, 1, 3), _log(rng, 2, 12), _log(rng, 2, 500), kv_heads * each, kv_heads, dim, vdim, _log(rng, 4, 4000),
                          rng.choice([0, _log(rng, 1, 500)]), window, rng.randint(0, 70), ragged=rng.random() < 0.7)
    if kind == "beams":
        return _beams(_log(rng, 1, 48), rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24]), _log(rng, 1000, 50400), rng.choice(["float32", "float32", "bfloat16"]),
                      rng.choice([0.0, 0.0, 0.6, 1.0]), rng.random() < 0.2)
    room = _log(rng, 64, 1500)
    prompt = rng.randint(1, room // 2)
    return _reorder(_log(rng, 1, 32), rng.choice([2, 3, 4, 5, 8, 12, 16, 24]), rng.randint(1, 8), rng.choice([1, 2, 4, 8]), rng.choice([128, 64, 40, 24]), prompt,
                    rng.randint(1, room - prompt), room, rng.choice(["model", "model", "int8"]), rng.choice(["bfloat16", "bfloat16", "float32"]))


def _plain_size(case):
    """Numbers that the plain form of the attention holds at a time."""
    L = case["prefix"] + case["tokens"] + case["T"]
    return case["groups"] * case["per"] * L * (case["kv_heads"] * (case["dim"] + case["vdim"]) + case["heads"] * case["T"])


def _held_bytes(case):
    return case["groups"] * case["beams"] * case["layers"] * 2 * case["kv_heads"] * case["room"] * case["dim"]


def draw(rng):
    top = {c["name"]: c for c in listed()}
    largest = {"beams": work(top["beams_batch"])["bytes"], "reorder": work(top["reorder_batch"])["bytes"]}
    while True:
        case = _draw_once(rng)
        w = work(case)
        if case["kind"] == "attention":
            most = work(top["attn_portion"] if case["T"] > 1 else top["attn_system"])
            if w["flops"] > most["flops"] or _plain_size(case) > _plain_size(top["attn_portion"]):
                continue
        elif w["bytes"] > largest[case["kind"]] or case["kind"] == "reorder" and _held_bytes(case) > _held_bytes(top["reorder_batch"]):
            continue
        return case


# ---------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------


def _size(case):
    return {"float32": 4, "bfloat16": 2}[case["dtype"]]


def _places(case):
    """By sequence: whose cache holds its first positions, how many of them, its position, its real tokens in the portion."""
    lead, shared, pos, count = [], [], [], []
    for g in range(case["groups"]):
        p = case["prefix"] - (g * 7919) % max(1, case["prefix"] // 4) * case["ragged"]
        for i in range(case["per"]):
            b = g * case["per"] + i
            lead.append(g * case["per"])
            # now and then a sequence that left the prefix a little earlier
            shared.append(max(1, p - (b * 31) % max(1, p // 8)) if case["ragged"] and i % 5 == 4 else p)
            pos.append(p + case["tokens"] - (b * 131) % max(1, case["tokens"] // 2) * case["ragged"])
            count.append(case["T"] - (b * 131) % max(1, case["T"] // 8) * case["ragged"] if case["T"] > 1 else int(not case["ragged"] or b % 16 != 13))
    return lead, [min(s, p, pos[l]) for s, p, l in zip(shared, pos, lead)], pos, count


def _room(case):
    return (max(_places(case)[2]) + case["T"] + 63) // 64 * 64


def _visible(i, window, keep, lo, hi):
    """Keys that position i sees among [lo, hi)."""
    hi = min(hi, i + 1)
    first = max(0, i - window + 1) if window else 0
    return max(0, hi - max(lo, first)) + max(0, min(hi, keep, first) - lo)


def _survivors(case, seed):
    """Slots that the beams of every slot come from: those that go on keep their slot."""
    g = torch.Generator().manual_seed(seed)
    K = case["beams"]
    parents = []
    for group in range(case["groups"]):
        alive = torch.rand(K, generator=g) < 0.6
        alive[int(torch.randint(K, (1,), generator=g))] = True
        live = torch.nonzero(alive).flatten()
        pick = live[torch.randint(len(live), (K,), generator=g)]
        parents += (torch.where(alive, torch.arange(K), pick) + group * K).tolist()
    return parents


def _lengths(case):
    """Positions of the beams of every prompt before the step."""
    return [case["prompt"] + case["tokens"] - (g * 131) % max(1, case["tokens"] // 2) for g in range(case["groups"])]


def work(case):
    e = _size(case)
    if case["kind"] == "attention":
        H, G, d, v, w, keep = (case[k] for k in ("heads", "kv_heads", "dim", "vdim", "window", "keep"))
        lead, shared, pos, count = _places(case)
        pairs, rows, keys, seen = 0, 0, 0, {}
        for b, (p, n) in enumerate(zip(pos, count)):
            rows += n
            pairs += sum(_visible(i, w, keep, 0, i + 1) for i in range(p, p + n))
            if n:  # keys of the prefix are read once for all, the sequence's own ones by itself
                kept, first = min(keep, shared[b]), max(0, p - w + 1) if w else 0
                lo, hi, k = seen.get(lead[b], (1 << 30, 0, 0))
                seen[lead[b]] = (min(lo, first), max(hi, shared[b]), max(k, kept))
                keys += max(0, p - max(first, shared[b])) + max(0, min(keep, first) - shared[b])
        keys += sum(max(0, hi - lo) + min(k, lo, hi) for lo, hi, k in seen.values())
        return {"bytes": rows * e * ((H + G) * d + (G + 2 * H) * v) + (keys + rows) * G * (d + v) * e, "flops": 2 * (d + v) * pairs * H}
    if case["kind"] == "beams":
        rows = case["groups"] * (1 if case["first"] else case["beams"])
        return {"bytes": rows * (case["vocab"] * e + 32), "flops": 4 * rows * case["vocab"]}
    moved = read = 0
    parents, K = _survivors(case, 1), case["beams"]
    for g, n in enumerate(_lengths(case)):
        p = [(b, q) for b, q in enumerate(parents[g * K:(g + 1) * K], g * K) if b != q]
        moved += len(p) * (n - case["prompt"])
        read += len({q for _, q in p}) * (n - case["prompt"])
    per = 2 * case["layers"] * case["kv_heads"] * case["dim"]
    return {"bytes": (moved + read) * per * (1 if case["cache"] == "int8" else e), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------


class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def __call__(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=self.g) * std + mean

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)

    def rows(self, *shape, dtype):
        """Large tensors in their own type, a sequence at a time."""
        out = torch.empty(shape, dtype=dtype, device="cuda")
        for row in out:
            row.copy_(self(*shape[1:]))
        return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _attention_inputs(case, seed):
    n, dt = _Draws(seed), getattr(torch, case["dtype"])
    T, H, G, d, v = (case[k] for k in ("T", "heads", "kv_heads", "dim", "vdim"))
    B, room = case["groups"] * case["per"], _room(case)
    lead, shared, pos, count = _places(case)
    return {"proj": n(B * T, (H + G) * d + (G + H) * v).to(dt), "q_norm": n(d, std=0.2, mean=1.6), "k_norm": n(d, std=0.2, mean=1.2),
            "k": n.rows(B, G, room, d, dtype=dt), "v": n.rows(B, G, room, v, dtype=dt), "pos": _i32(pos), "count": _i32(count),
            "lead": _i32(lead), "shared": _i32(shared), "joint": n(B * T, H * v).to(dt)}


def _beams_inputs(case, seed):
    n, K = _Draws(seed), case["beams"]
    rows = case["groups"] * K
    slot = torch.arange(rows, device="cuda") % K
    scores = -30.0 * n.uniform(case["groups"]).repeat_interleave(K) - 4.0 * n.uniform(rows)
    ended = (n.uniform(rows) < 0.1).int()
    length = torch.full((rows,), 23, dtype=torch.int32, device="cuda") - ended * (1 + slot.int() % 7)
    if case["first"]:  # a prompt has just been read: one beam stands for all
        scores, ended, length = torch.where(slot == 0, 0.0, -math.inf), ended * 0, length * 0
    return {"logits": n(rows, case["vocab"], std=2.5).to(getattr(torch, case["dtype"])), "scores": scores, "ended": ended, "length": length,
            "scores_next": scores * 0, "ended_next": ended * 0, "length_next": length * 0, "current": _i32([0] * rows),
            "parent": _i32([0] * rows), "generated": torch.zeros((8, rows), dtype=torch.int32, device="cuda"),
            "parents": torch.zeros((8, rows), dtype=torch.int32, device="cuda"), "step": _i32([3])}


END = 2  # the token that ends a beam


def _reorder_inputs(case, seed):
    n, dt = _Draws(seed), getattr(torch, case["dtype"])
    B, G, d, room = case["groups"] * case["beams"], case["kv_heads"], case["dim"], case["room"]
    out = {}
    for i in range(case["layers"]):
        for name in "kv":
            if case["cache"] == "int8":
                blocks = -(-room // 64)
                out[f"{name}{i}"] = torch.randint(-127, 128, (B, G, blocks, 64, d), dtype=torch.int8, device="cuda", generator=n.g)
                out[f"{name}_scale{i}"], out[f"{name}_tail{i}"] = 0.01 + n.uniform(B, G, blocks), n(B, G, 64, d).to(dt)
            else:
                out[f"{name}{i}"] = n.rows(B, G, room, d, dtype=dt)
    K = case["beams"]
    out.update(parent=_i32(_survivors(case, seed)), begin=_i32([case["prompt"]] * B), end=_i32([x for x in _lengths(case) for _ in range(K)]))
    return out


_INPUTS = {"attention": _attention_inputs, "beams": _beams_inputs, "reorder": _reorder_inputs}


def prepare(case, seed):
    t = _INPUTS[case["kind"]](case, seed)
    s = {"case": case, "in": t}
    if case["kind"] == "attention":  # the positions that the plain form looks at
        s["extent"] = max(_places(case)[2]) + case["T"]
    if own:
        s.update(_program(case, t))
        s["in"] = s["held"]
    return s


def _positions(case, name):
    """The axis of positions of a state (None: it has none), and how many of them an entry stands for."""
    return (None, 1) if "tail" in name else (2, 64 if case["cache"] == "int8" else 1)


_READ = {"attention": {"proj", "q_norm", "k_norm", "pos", "count", "lead", "shared"}, "beams": {"logits", "scores", "ended", "length"},
         "reorder": {"parent", "begin", "end"}}


def _program(case, t):
    """A session that holds the tensors, and a program of one pass through the operator."""
    import numpy as np
    from popxl_addons_b200 import xl
    from popxl_addons_b200.xl import ops

    ir = xl.Ir()
    with ir.main_graph:
        held = {k: xl.variable(xl.LazyInit(tuple(x.shape), np.float32, "zeros"), xl.dtype.as_dtype(x.dtype), k) for k, x in t.items()}
    session = xl.Session(ir, "cuda")
    for k, x in t.items():
        session.device_tensor(held[k]).copy_(x)
    program = xl.Program(ir, "pass")
    with program:
        use = {k: program.use(v, by_ref=k not in _READ[case["kind"]]) for k, v in held.items()}
        if case["kind"] == "attention":
            ops.window_attention_shared_(use["proj"], use["q_norm"], use["k_norm"], use["k"], use["v"], use["pos"], use["count"], use["lead"],
                                         use["shared"], use["joint"], case["T"], case["heads"], case["dim"] ** -0.5, case["window"], case["keep"],
                                         SINK, EPS)
        elif case["kind"] == "beams":
            ops.take_beams_(use["current"], use["parent"], use["logits"], use["generated"], use["parents"], use["step"],
                            ops.BeamState(use["scores"], use["ended"], use["length"]), case["beams"], end=END, length_penalty=case["penalty"],
                            into=ops.BeamState(use["scores_next"], use["ended_next"], use["length_next"]), advance=False)
        else:
            ops.reorder_([ops.StateRows(use[k], *_positions(case, k)) for k in _states(use)], use["parent"], use["begin"], use["end"], case["beams"])
    return {"session": session, "program": program, "held": {k: session.device_tensor(v) for k, v in held.items()}}


def _states(t):
    return [k for k in t if k not in _READ["reorder"]]


# ---------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------


def run(state):
    case, t = state["case"], state["in"]
    if own:
        state["session"].run_program(state["program"], fetch=False, copy=False)
    elif case["kind"] == "attention":
        _attention_plain(case, t, state["extent"])
    else:
        {"beams": _beams_plain, "reorder": _reorder_plain}[case["kind"]](case, t)
    if case["kind"] == "attention":
        return {k: t[k] for k in ("joint", "k", "v")}
    if case["kind"] == "beams":
        return {k: t[k] for k in ("current", "parent", "generated", "parents", "scores_next", "ended_next", "length_next")}
    return {k: t[k] for k in _states(t)}


def _unit(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _attention_plain(case, t, extent):
    T, H, G, d, v = (case[k] for k in ("T", "heads", "kv_heads", "dim", "vdim"))
    B, R, dt, dev = case["groups"] * case["per"], H // G, t["joint"].dtype, t["joint"].device
    proj, pos, count = t["proj"].reshape(B, T, -1), t["pos"].long(), t["count"].long()
    qk = (H + G) * d
    q = _unit(proj[..., :H * d].float().reshape(B, T, G, R, d), t["q_norm"])
    b, real = torch.arange(B, device=dev)[:, None], torch.arange(T, device=dev) < count[:, None]
    at = pos[:, None] + torch.arange(T, device=dev)                                                       # (B, T)
    new = {"k": _unit(proj[..., H * d:qk].double().reshape(B, T, G, d), t["k_norm"].double()).to(dt),
           "v": proj[..., qk:qk + G * v].reshape(B, T, G, v)}
    t["k"][b, :, at] = torch.where(real[..., None, None], new["k"], t["k"][b, :, at])
    t["v"][b, :, at] = torch.where(real[..., None, None], new["v"], t["v"][b, :, at])
    lead = t["lead"].long()
    edge = torch.minimum(torch.minimum(t["shared"].long(), pos), pos[lead])[:, None]
    j = torch.arange(extent, device=dev)
    rows = torch.where(j < edge, lead[:, None], b)                                                        # (B, extent): whose cache
    keys = t["k"][rows, :, j].transpose(1, 2).float()                                                     # (B, G, extent, d)
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, G, R * T, d), keys.transpose(-1, -2)).reshape(B, G, R, T, -1) * d ** -0.5
    del keys
    seen = j <= at[..., None]
    if case["window"]:
        seen = seen & ((at[..., None] - j < case["window"]) | (j < case["keep"]))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=SINK)
    s.sub_(top).exp_()
    total = s.sum(-1) + torch.exp(SINK - top[..., 0])
    o = torch.matmul(s.reshape(B, G, R * T, -1), t["v"][rows, :, j].transpose(1, 2).float()).reshape(B, G, R, T, v) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, H * v) * torch.sigmoid(proj[..., qk + G * v:].float())
    joint = t["joint"].reshape(B, T, -1)
    joint.copy_(torch.where(real[..., None], o.to(dt), joint))


def _beams_plain(case, t):
    n, K, V = case["groups"], case["beams"], case["vocab"]
    dev, rows = t["logits"].device, n * K
    ended = t["ended"][:, None] > 0
    token = torch.arange(V, device=dev)
    x = t["logits"].double()
    top = x.amax(1, keepdim=True)
    c = t["scores"].double()[:, None] + (x - top - torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    c = torch.where(ended, torch.where(token == END, t["scores"].double()[:, None], -math.inf), c)
    after = t["length"] + 1 - t["ended"]
    c = torch.where(torch.isnan(c), -math.inf, c)
    rank = (c / after.double().clamp(min=1)[:, None] ** case["penalty"]).reshape(n, K * V)
    at = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :K]                             # in order of rank
    parent, chosen, score = at // V, at % V, c.reshape(n, -1).gather(1, at)
    # the best continuation of a beam takes its slot, the others take free slots in order
    i = torch.arange(K, device=dev)
    again = ((parent[:, :, None] == parent[:, None]) & (i[:, None] > i)).any(-1)                          # an earlier one has the same parent
    free = (parent[:, None] != i[:, None]).all(-1)                                                        # (groups, slots)
    spare = torch.sort(torch.where(free, i, K + i), dim=1).values                                         # free slots in front
    slot = torch.where(again, spare.gather(1, (again.long().cumsum(1) - 1).clamp(min=0)), parent)
    base = torch.arange(n, device=dev)[:, None] * K
    to = (base + slot).flatten()
    parent, chosen = (base + parent).flatten(), chosen.flatten()
    was = t["ended"][parent] > 0
    t["current"][to] = chosen.int()
    t["parent"][to] = parent.int()
    t["scores_next"][to] = score.flatten().float()
    t["ended_next"][to] = (was | (chosen == END)).int()
    t["length_next"][to] = after[parent]
    t["generated"][t["step"].long()] = t["current"]
    t["parents"][t["step"].long()] = t["parent"]


def _reordered(case, t, name, x):
    axis, per = _positions(case, name)
    if axis is None:
        return x.copy_(x[t["parent"].long()])
    i = torch.arange(x.shape[2], device=x.device)
    takes = (i >= (t["begin"] // per)[:, None]) & (i < ((t["end"] + per - 1) // per)[:, None]) & (t["end"] > t["begin"])[:, None]
    takes = takes.reshape(takes.shape[0], 1, -1, *[1] * (x.dim() - 3))
    return x.copy_(torch.where(takes, x[t["parent"].long()], x))


def _reorder_plain(case, t):
    return [_reordered(case, t, k, t[k]) for k in _states(t)]


# ---------------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------


def _attention_exact(case, t):
    T, H, G, d, v = (case[k] for k in ("T", "heads", "kv_heads", "dim", "vdim"))
    R, dt = H // G, t["joint"].dtype
    lead, shared, pos, count = _places(case)
    joint = t["joint"].double().reshape(len(pos), T, H * v)
    before = {x: [t[x][l, :, :e].double() for l, e in zip(lead, shared)] for x in "kv"}
    for b, (p, n) in enumerate(zip(pos, count)):
        if n == 0:
            continue
        q, k, val, gate = t["proj"][b * T:b * T + n].double().split((H * d, G * d, G * v, H * v), 1)
        q = q.reshape(n, H, d) * (q.reshape(n, H, d).square().mean(-1, keepdim=True) + EPS).rsqrt() * t["q_norm"].double()
        k = k.reshape(n, G, d) * (k.reshape(n, G, d).square().mean(-1, keepdim=True) + EPS).rsqrt() * t["k_norm"].double()
        t["k"][b, :, p:p + n] = k.to(dt).transpose(0, 1)
        t["v"][b, :, p:p + n] = val.reshape(n, G, v).transpose(0, 1).to(dt)
        keys, vals = (torch.cat((before[x][b], t[x][b, :, shared[b]:p + n].double()), 1) for x in "kv")
        s = torch.einsum("igrd,gjd->grij", q.reshape(n, G, R, d), keys) * d ** -0.5
        i, j = torch.arange(p, p + n, device=s.device)[:, None], torch.arange(p + n, device=s.device)
        ok = j <= i
        if case["window"]:
            ok = ok & ((i - j < case["window"]) | (j < case["keep"]))
        s = torch.cat((s.masked_fill(~ok, -math.inf), torch.full_like(s[..., :1], SINK)), -1)
        o = torch.einsum("grij,gjv->igrv", torch.softmax(s, -1)[..., :-1], vals).reshape(n, H * v)
        joint[b, :n] = o * torch.sigmoid(gate)
    return {"joint": joint.reshape(-1, H * v), "k": t["k"].double(), "v": t["v"].double()}


def _beams_exact(case, t):
    K, V = case["beams"], case["vocab"]
    for g in range(case["groups"]):
        found = []  # (rank, flat index, sum)
        for k in range(K):
            row = g * K + k
            score, length, ended = float(t["scores"][row]), int(t["length"][row]), int(t["ended"][row])
            if ended:
                found.append((score / max(length, 1) ** case["penalty"], k * V + END, score))
                continue
            if score == -math.inf:
                continue
            c = score + torch.log_softmax(t["logits"][row].double(), 0)
            best = torch.sort(c, descending=True, stable=True)
            found += [(float(x) / max(length + 1, 1) ** case["penalty"], k * V + int(i), float(x)) for x, i in zip(best.values[:K], best.indices[:K])]
        found = sorted(found, key=lambda f: (-f[0], f[1]))[:K]
        free, taken = [s for s in range(K) if s not in {i // V for _, i, _ in found}], set()
        for _, i, c in found:
            p, token = i // V, i % V
            slot = free.pop(0) if p in taken else p
            taken.add(p)
            to, row = g * K + slot, g * K + p
            t["current"][to], t["parent"][to], t["scores_next"][to] = token, row, c
            t["ended_next"][to] = int(t["ended"][row] > 0 or token == END)
            t["length_next"][to] = t["length"][row] + 1 - t["ended"][row]
    t["generated"][3], t["parents"][3] = t["current"], t["parent"]
    return {k: t[k] for k in ("current", "parent", "generated", "parents", "scores_next", "ended_next", "length_next")}


def _reorder_exact(case, t):
    parent, K = t["parent"].tolist(), case["beams"]
    out = {}
    for name in _states(t):
        out[name] = t[name].clone()
        for b, p in enumerate(parent):
            axis, per = _positions(case, name)
            lo, hi = case["prompt"] // per, -(-_lengths(case)[b // K] // per)
            if axis is None:
                out[name][b] = t[name][p]
            else:
                out[name][b, :, lo:hi] = t[name][p, :, lo:hi]
    return out


def exact(case, seed):
    return {"attention": _attention_exact, "beams": _beams_exact, "reorder": _reorder_exact}[case["kind"]](case, _INPUTS[case["kind"]](case, seed))
