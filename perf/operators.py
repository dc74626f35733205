"""Operators of a serving step for a batch of unlike requests, each as a user's program calls it and in a plain form.

* `attention`: sliding-window attention of a portion of tokens against a cache held in 8 bits, with a scale for each block of 64
  tokens and head. A position sees the tokens of its own block as they were computed and those of earlier blocks as the cache
  holds them, so results do not depend on how a prompt is cut into portions.
* `adapted`: a projection that all requests share, and beside it a low-rank adapter of each request's own.
* `shape`, `choose`: penalties for repeated tokens, biases and grammar masks on logits; the shaped logits for a caller that
  samples, or the greedy choice that becomes the current token and a row of the history.

Plain forms are elementary torch operations in 32 bits (norms of keys, whose rounding decides on codes, in 64), rounded once at
the end. `exact` has the same results in 64 bits, sequence by sequence.
"""
import math

import torch

own = False  # whether `run` makes the calls of the framework

BLOCK = 64   # tokens of a cache block with one scale
EPS = 1e-6
SINK = 0.0


# ---------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------


def _attention(batch, T, heads, kv_heads, dim, vdim, pos, window=0, keep=4, dtype="bfloat16", ragged=True, complete=False):
    return dict(kind="attention", batch=batch, T=T, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, pos=pos, window=window,
                keep=keep if window else 0, dtype=dtype, ragged=ragged, complete=complete)


def _adapted(batch, T, K, N, adapters, rank, dtype="bfloat16"):
    return dict(kind="adapted", batch=batch, T=T, K=K, N=N, adapters=adapters, rank=rank, dtype=dtype)


def _logits(kind, rows, slots, vocab, history, biases, dtype="float32"):
    return dict(kind=kind, rows=rows, slots=slots, vocab=vocab, history=history, biases=biases, dtype=dtype)


def listed():
    return [
        # one user whose program samples on the host: latency of a single token on a short history
        dict(_attention(1, 1, 16, 4, 128, 128, 33, 256), name="attn_single"),
        # a batch of documents in progress, no window: reading the cache is all there is
        dict(_attention(16, 1, 32, 8, 128, 128, 8000), name="attn_long"),
        # more users than one tile holds, a short window, and every sequence fills a block with this token
        dict(_attention(40, 1, 16, 4, 128, 128, 2000, 256, complete=True), name="attn_window"),
        # documents of several thousand tokens in one portion, windows next to the first tokens
        dict(_attention(2, 4096, 32, 8, 128, 128, 0, 1024, ragged=False), name="attn_prompt"),
        # the next portion of long documents: an odd length, after what the cache holds already
        dict(_attention(2, 515, 32, 8, 128, 128, 6000), name="attn_portion"),
        # a 32-bit model
        dict(_attention(4, 1, 8, 2, 128, 128, 215, 8192, dtype="float32"), name="attn_float32"),
        # one user with an adapter: the smallest product
        dict(_adapted(1, 1, 2048, 2048, 4, 8), name="adapted_single"),
        # 40 users of 32 adapters, the joint input projection of a layer
        dict(_adapted(40, 1, 4096, 32256, 32, 16), name="adapted_batch"),
        # prompts of unlike requests, the joint input projection of a layer
        dict(_adapted(4, 1024, 4096, 32256, 8, 16), name="adapted_prompts"),
        # one user whose program samples on the host
        dict(_logits("shape", 1, 1, 32000, 48, 8), name="shape_single"),
        # logits of several places of every request
        dict(_logits("shape", 96, 16, 50400, 2048, 64), name="shape_places"),
        # a decoding step of a large batch, logits in the model's type
        dict(_logits("choose", 48, 48, 50400, 2048, 32, dtype="bfloat16"), name="choose_batch"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["attention", "attention", "attention", "adapted", "adapted", "shape", "choose"])
    if kind == "attention":
        dim, vdim = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 80), (40, 24)])
        kv_heads, groups = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8, 16])
        window = rng.choice([0, 0, _log(rng, 32, 4096)])
        dtype = "float32" if rng.random() < 0.15 else "bfloat16"
        if dtype == "float32":
            return _attention(_log(rng, 1, 4), rng.choice([1, 1, _log(rng, 2, 64)]), kv_heads * groups, kv_heads, dim, vdim,
                              _log(rng, 1, 1000), window, rng.randint(0, 8), dtype)
        if rng.random() < 0.6:
            return _attention(_log(rng, 1, 48), 1, kv_heads * groups, kv_heads, dim, vdim, _log(rng, 1, 12000), window,
                              rng.randint(0, 70), ragged=rng.random() < 0.8, complete=rng.random() < 0.25)
        return _attention(_log(rng, 1, 6), _log(rng, 2, 3000), kv_heads * groups, kv_heads, dim, vdim,
                          rng.choice([0, _log(rng, 1, 6000)]), window, rng.randint(0, 70), ragged=rng.random() < 0.8)
    if kind == "adapted":
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        one = rng.random() < 0.6
        if dtype == "float32":
            return _adapted(_log(rng, 1, 8), 1 if one else _log(rng, 2, 64), 8 * _log(rng, 32, 256), 2 * _log(rng, 64, 2048),
                            _log(rng, 1, 16), 4 * rng.randint(1, 8), dtype)
        return _adapted(_log(rng, 1, 64 if one else 6), 1 if one else _log(rng, 2, 1000), 8 * _log(rng, 32, 640),
                        2 * _log(rng, 128, 16384), _log(rng, 1, 64), rng.choice([4, 8, 16, 24, 32, 64]), dtype)
    slots = _log(rng, 1, 64)
    return _logits(kind, slots if kind == "choose" else _log(rng, 1, 96), slots, _log(rng, 1000, 50400), _log(rng, 8, 8192),
                   rng.choice([0, _log(rng, 1, 256)]), rng.choice(["float32", "bfloat16"]))


def _scores(case):
    """Entries of the plain form's score matrices."""
    last = max(_positions(case)) + case["T"]
    return case["batch"] * case["heads"] * case["T"] * (last + case["T"] + 3 * BLOCK)


def draw(rng):
    top = {c["name"]: c for c in listed()}
    heaviest = {"attention": work(top["attn_prompt"]), "adapted": work(top["adapted_prompts"]), "shape": work(top["shape_places"]),
                "choose": work(top["shape_places"])}
    while True:
        case = _draw_once(rng)
        w, most = work(case), heaviest[case["kind"]]
        if w["flops"] > most["flops"] or w["bytes"] > max(most["bytes"], work(top["attn_long"])["bytes"]):
            continue
        if case["kind"] == "attention" and _scores(case) > _scores(top["attn_prompt"]):
            continue
        return case


# ---------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------


def _size(case):
    return {"float32": 4, "bfloat16": 2}[case["dtype"]]


def _positions(case):
    """Tokens that every sequence holds before the pass."""
    out = []
    for b in range(case["batch"]):
        p = case["pos"] - (b * 7919) % max(1, case["pos"] // 4) * case["ragged"]
        if case["T"] == 1:
            p = p // BLOCK * BLOCK + BLOCK - 1 if case["complete"] else p - (p % BLOCK == BLOCK - 1)
        out.append(p)
    return out


def _counts(case):
    """Real tokens of every sequence in the portion; the rest of its rows is padding."""
    return [case["T"] - (b * 131) % max(1, case["T"] // 8) for b in range(case["batch"])]


def _blocks(case):
    return (max(_positions(case)) + case["T"]) // BLOCK + 1


def _visible(i, window, keep):
    """Keys that position i sees."""
    return i + 1 if not window or i < window else window + min(keep, i - window + 1)


def _slots(case):
    """The adapter of every sequence; -1: none."""
    return [(b * 5 + 1) % (case["adapters"] + 1) - 1 if case["adapters"] > 1 else 0 for b in range(case["batch"])]


def _held(case):
    """Tokens in the history of every slot, and how many of them came with the prompt."""
    held = [case["history"] - (s * 7919) % max(1, case["history"] // 2) for s in range(case["slots"])]
    return held, [n // 2 for n in held]


def work(case):
    e = _size(case)
    if case["kind"] == "attention":
        H, G, d, v = (case[k] for k in ("heads", "kv_heads", "dim", "vdim"))
        flops = reads = rows = 0
        for p, n in zip(_positions(case), _counts(case)):
            pairs = sum(_visible(i, case["window"], case["keep"]) for i in range(p, p + n))
            flops += 2 * (d + v) * pairs * H
            rows += n
            old = p // BLOCK * BLOCK  # tokens that the cache holds in 8 bits before the pass, of which the window shows some
            seen = old if not case["window"] else min(old, max(0, old - (p - case["window"] + 1)) + case["keep"])
            reads += G * (seen * (d + v) + -(-seen // BLOCK) * 8 + p % BLOCK * (d + v) * e)
            reads += G * ((p + n) // BLOCK - p // BLOCK) * (BLOCK * (d + v) + 8)  # blocks that the pass completes
            reads += G * min(n, (p + n) % BLOCK) * (d + v) * e
        return {"bytes": rows * e * ((H + G) * d + (G + 2 * H) * v) + reads, "flops": flops}
    if case["kind"] == "adapted":
        rows, K, N, r = case["batch"] * case["T"], case["K"], case["N"], case["rank"]
        used = len({s for s in _slots(case) if s >= 0})
        return {"bytes": e * (rows * (K + N) + N * K + used * r * (K + N)), "flops": 2 * rows * (N * K + r * (K + N))}
    n, V = case["rows"], case["vocab"]
    held = sum(_held(case)[0][i % case["slots"]] for i in range(n))
    rules = min(n, case["slots"]) * (V / 8 + 8 * case["biases"]) + 4 * held * min(1, case["slots"] / n)
    return {"bytes": n * V * (e + (4 if case["kind"] == "shape" else 0)) + rules, "flops": 6 * n * V}


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


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _attention_inputs(case, seed):
    n, dt = _Draws(seed), getattr(torch, case["dtype"])
    B, T, H, G, d, v = (case[k] for k in ("batch", "T", "heads", "kv_heads", "dim", "vdim"))
    blocks = _blocks(case)
    out = {"proj": n(B * T, (H + G) * d + (G + H) * v).to(dt), "q_norm": n(d, std=0.2, mean=1.6), "k_norm": n(d, std=0.2, mean=1.2)}
    for name, width, std in (("k", d, 1.2), ("v", v, 1.0)):
        x = n(B, G, blocks, BLOCK, width, std=std) * torch.exp(n(B, G, blocks, 1, 1, std=0.2))
        scale = x.abs().amax((-2, -1)) / 127
        out[name] = (x / scale[..., None, None]).round().clamp(-127, 127).to(torch.int8)
        out[name + "_scale"] = scale
        out[name + "_tail"] = n(B, G, BLOCK, width, std=std).to(dt)
    out["pos"], out["count"] = _i32(_positions(case)), _i32(_counts(case))
    out["joint"] = n(B * T, H * v).to(dt)
    return out


def _adapted_inputs(case, seed):
    n, dt = _Draws(seed), getattr(torch, case["dtype"])
    B, T, K, N, a, r = (case[k] for k in ("batch", "T", "K", "N", "adapters", "rank"))
    return {"x": n(B * T, K).to(dt), "weight": n(N, K, std=K ** -0.5).to(dt), "a": n(a, r, K, std=K ** -0.5).to(dt),
            "b": n(a, N, r, std=0.5 * r ** -0.5).to(dt), "scale": 0.5 + n.uniform(a), "slot": _i32(_slots(case))}


def _logits_inputs(case, seed):
    n, dt = _Draws(seed), getattr(torch, case["dtype"])
    rows, S, V, L, K = (case[k] for k in ("rows", "slots", "vocab", "history", "biases"))
    held, start = _held(case)
    words = -(-V // 32)
    # what grammars allow: everything, half of all tokens, a few of them; in a large batch one slot is left with nothing
    share = torch.tensor([(2.0, 0.5, 20.0 / V, 2.0)[s % 4] if s != 13 else -1.0 for s in range(S)], device="cuda")
    bits = (n.uniform(S, words, 32) < share[:, None, None]).long()
    word = (bits << torch.arange(32, device="cuda")).sum(-1)
    out = {"logits": n(rows, V, std=2.5).to(dt), "length": None, "history": (V ** n.uniform(S, L + 1) - 1).to(torch.int32).clamp(0, V - 1),
           "start": _i32(start), "allowed": torch.where(word > 0x7fffffff, word - (1 << 32), word).to(torch.int32),
           "penalties": torch.stack((1.0 + 0.5 * n.uniform(S), 0.5 * n.uniform(S), n.uniform(S)), 1)}
    # repetition, frequency, presence; a slot in three has none of them
    plain = torch.arange(S, device="cuda") % 3 == 2
    out["penalties"] = torch.where(plain[:, None], torch.tensor([1.0, 0.0, 0.0], device="cuda"), out["penalties"])
    K1 = max(1, K)  # a list always has room for one entry; -1: not in use
    out["bias_tokens"] = torch.topk(n.uniform(S, V), K1).indices.to(torch.int32)
    out["bias_tokens"][:, K - K // 4:] = -1
    out["bias_values"] = n(S, K1, std=3.0)
    if case["kind"] == "shape":  # places of the slots in turn, the later ones further along
        out["slot"] = _i32([i % S for i in range(rows)])
        out["length"] = _i32([max(1, held[i % S] - (rows - 1 - i) // S) for i in range(rows)])
        return out
    out["length"], out["count"] = _i32(held), _i32([1] * S)
    out["current"], out["step"] = _i32([0] * S), _i32([3])
    out["generated"] = torch.zeros((8, S), dtype=torch.int32, device="cuda")
    return out


def prepare(case, seed):
    t = {"attention": _attention_inputs, "adapted": _adapted_inputs}.get(case["kind"], _logits_inputs)(case, seed)
    s = {"case": case, "in": t}
    if case["kind"] == "attention" and (case["complete"] or case["T"] > 1):
        # cache blocks that the pass may complete: (sequences, 1) and their numbers
        s["which"] = (torch.arange(case["batch"], device="cuda")[:, None],
                      t["pos"].long()[:, None] // BLOCK + torch.arange(case["T"] // BLOCK + 1, device="cuda"))
    if own:
        s.update(_program(case, t))
        s["in"] = s["held"]
    return s


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
    program, stream = xl.Program(ir, "pass"), None
    written = {"k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "joint", "current", "generated", "step", "history"}
    with program:
        use = {k: program.use(v, by_ref=k in written) for k, v in held.items()}
        if case["kind"] == "attention":
            cache = ops.Cache8(*(use[k] for k in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")))
            ops.window_attention_q8_(use["proj"], use["q_norm"], use["k_norm"], cache, use["pos"], use["count"], use["joint"],
                                     case["T"], case["heads"], case["dim"] ** -0.5, case["window"], case["keep"], SINK, EPS)
        elif case["kind"] == "adapted":
            y = ops.linear_adapted(use["x"], use["weight"], ops.Adapters(use["a"], use["b"], use["scale"]), use["slot"], case["T"])
        else:
            rules = ops.LogitRules(*(use[k] for k in ("history", "start", "penalties", "bias_tokens", "bias_values", "allowed")))
            if case["kind"] == "shape":
                y = ops.shape_logits(use["logits"], use["slot"], use["length"], rules)
            else:
                ops.take_shaped_(use["current"], use["logits"], use["generated"], use["step"], use["length"], use["count"], rules,
                                 advance=False)
        if case["kind"] in ("adapted", "shape"):
            stream = xl.d2h_stream(y.shape, y.dtype, "result")
            ops.host_store(stream, y)
    return {"session": session, "program": program, "stream": stream, "held": {k: session.device_tensor(v) for k, v in held.items()}}


# ---------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------


def run(state):
    case, t = state["case"], state["in"]
    if own:  # outputs that are not held in the session's variables are the program's own buffers
        out = state["session"].run_program(state["program"], fetch=False, copy=False)
        y = out[state["stream"]][0, 0] if state["stream"] is not None else None
    else:
        y = {"attention": _attention_plain, "adapted": _adapted_plain, "shape": _shape_plain, "choose": _choose_plain}[case["kind"]](case, t)
    if case["kind"] == "choose":
        return {k: t[k] for k in ("current", "generated", "history")}
    if case["kind"] != "attention":
        return y
    res = {k: t[k] for k in ("joint", "k_tail", "v_tail")}
    if "which" in state:  # the values that the blocks stand for
        b, j = state["which"]
        for k in "kv":
            res[k] = (t[k][b, :, j] * t[k + "_scale"][b, :, j][..., None, None]).to(t["joint"].dtype)
    return res


def _unit(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _attention_plain(case, t):
    B, T, H, G, d, v = (case[k] for k in ("batch", "T", "heads", "kv_heads", "dim", "vdim"))
    R, dt, dev = H // G, t["joint"].dtype, t["joint"].device
    proj, pos, count = t["proj"].reshape(B, T, -1), t["pos"].long(), t["count"].long()
    qk = (H + G) * d
    q = _unit(proj[..., :H * d].float().reshape(B, T, G, R, d), t["q_norm"])
    new = {"k": _unit(proj[..., H * d:qk].double().reshape(B, T, G, d), t["k_norm"].double()).to(dt),
           "v": proj[..., qk:qk + G * v].reshape(B, T, G, v)}
    first = pos // BLOCK * BLOCK           # position of the first row of `raw`: the block in progress
    fill, end = pos - first, pos - first + count
    row = torch.arange(T // BLOCK * BLOCK + 2 * BLOCK, device=dev)
    b = torch.arange(B, device=dev)[:, None]
    j = torch.arange(T // BLOCK + 1, device=dev)
    which, full = (b, first[:, None] // BLOCK + j), (end[:, None] >= (j + 1) * BLOCK)
    raw, cached = {}, {}
    for name in "kv":
        from_tail = t[name + "_tail"].transpose(1, 2)[b, row.clamp(max=BLOCK - 1)]
        from_new = new[name][b, (row - fill[:, None]).clamp(0, T - 1)]
        x = torch.where((row < fill[:, None])[..., None, None], from_tail, from_new).transpose(1, 2)      # (B, G, rows, width)
        x = torch.where((row < end[:, None])[:, None, :, None], x, torch.zeros_like(x))
        raw[name] = x.float()
        piece = raw[name][:, :, :len(j) * BLOCK].reshape(B, G, len(j), BLOCK, -1)
        top = piece.abs().amax((-2, -1))
        scale = top / torch.full_like(top, 127.0)
        code = torch.where(scale[..., None, None] > 0, (piece / scale[..., None, None]).round().clamp(-127, 127), torch.zeros_like(piece))
        codes, scales, tail = t[name], t[name + "_scale"], t[name + "_tail"]
        codes[which[0], :, which[1]] = torch.where(full[..., None, None, None], code.transpose(1, 2).to(torch.int8), codes[which[0], :, which[1]])
        scales[which[0], :, which[1]] = torch.where(full[..., None], scale.transpose(1, 2), scales[which[0], :, which[1]])
        left = torch.arange(BLOCK, device=dev)
        kept = x.transpose(1, 2)[b, end[:, None] // BLOCK * BLOCK + left].transpose(1, 2)
        tail.copy_(torch.where((left < end[:, None] % BLOCK)[:, None, :, None], kept, tail))
        cached[name] = (codes.float() * scales[..., None, None]).flatten(2, 3)
    scores, seen = [], []
    qp = (pos[:, None] + torch.arange(T, device=dev))[:, :, None]                                         # (B, T, 1)
    for keys, kp in ((cached["k"], torch.arange(cached["k"].shape[2], device=dev).expand(B, 1, -1)), (raw["k"], (first[:, None] + row)[:, None])):
        mask = kp // BLOCK < qp // BLOCK if keys is cached["k"] else (kp // BLOCK == qp // BLOCK) & (kp <= qp)
        if case["window"]:
            mask = mask & ((qp - kp < case["window"]) | (kp < case["keep"]))
        scores.append(torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, G, R * T, d), keys.transpose(-1, -2)).reshape(B, G, R, T, -1) * d ** -0.5)
        seen.append(mask)
    s = torch.cat(scores, -1)
    del scores
    s.masked_fill_(~torch.cat(seen, -1)[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=SINK)
    s.sub_(top).exp_()
    total = s.sum(-1) + torch.exp(SINK - top[..., 0])
    o = torch.matmul(s.reshape(B, G, R * T, -1), torch.cat((cached["v"], raw["v"]), 2)).reshape(B, G, R, T, v) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, H * v) * torch.sigmoid(proj[..., qk + G * v:].float())
    joint = t["joint"].reshape(B, T, -1)
    joint.copy_(torch.where((torch.arange(T, device=dev) < count[:, None])[..., None], o.to(dt), joint))


def _adapted_plain(case, t):
    B, T = case["batch"], case["T"]
    x, slot = t["x"].float(), t["slot"].long()
    low = torch.matmul(x.reshape(B, T, -1), t["a"].float()[slot.clamp(min=0)].transpose(1, 2))
    delta = torch.matmul(low, t["b"].float()[slot.clamp(min=0)].transpose(1, 2))
    delta = delta * torch.where(slot >= 0, t["scale"][slot.clamp(min=0)], torch.zeros_like(t["scale"][:1]))[:, None, None]
    return (torch.matmul(x, t["weight"].float().t()) + delta.reshape(B * T, -1)).to(t["x"].dtype)


def _shaped(t, slot, length, V):
    x, dev = t["logits"].float(), t["logits"].device
    rows = x.shape[0]
    history, at = t["history"].long()[slot], torch.arange(t["history"].shape[1], device=dev)
    held, drawn = at < length[:, None], (at < length[:, None]) & (at >= t["start"][slot][:, None])
    zero = torch.zeros((rows, V), device=dev)
    seen = zero.scatter_add(1, history, held.float()) > 0
    times = zero.scatter_add(1, history, drawn.float())
    repetition, frequency, presence = t["penalties"][slot][:, :, None].unbind(1)
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * times
    x = x - presence * (times > 0).float()
    token, value = t["bias_tokens"].long()[slot], t["bias_values"][slot]
    x = x + zero.scatter_add(1, token.clamp(min=0), torch.where(token >= 0, value, torch.zeros_like(value)))
    bits = t["allowed"][slot][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32) & 1
    return torch.where(bits.reshape(rows, -1)[:, :V] > 0, x, torch.full_like(x, -math.inf))


def _shape_plain(case, t):
    return _shaped(t, t["slot"].long(), t["length"], case["vocab"])


def _choose_plain(case, t):
    n = case["rows"]
    slot = torch.arange(n, device=t["logits"].device)
    x = _shaped(t, slot, t["length"], case["vocab"])
    # the lowest index among the largest
    ids = torch.arange(case["vocab"], device=x.device, dtype=torch.int32).expand(n, -1)
    token = torch.where(x == x.amax(1, keepdim=True), ids, torch.full_like(ids, case["vocab"])).amin(1)
    t["current"].copy_(token)
    t["generated"][t["step"].long()] = token
    t["history"][slot, t["length"].long()] = token


# ---------------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------


def _stored(block):
    """What a completed block `(G, 64, width)` stands for: whole steps of a 127th of its largest value per head."""
    top = block.float().abs().amax((1, 2), keepdim=True)
    step = top / torch.full_like(top, 127.0)
    code = torch.where(step > 0, torch.round(block.float() / step), torch.zeros_like(block.float()))
    return code.double() * step.double()


def _attention_exact(case, t):
    B, T, H, G, d, v = (case[k] for k in ("batch", "T", "heads", "kv_heads", "dim", "vdim"))
    R, dt = H // G, t["joint"].dtype
    joint = t["joint"].double().reshape(B, T, H * v)
    tails = {k: t[k + "_tail"].double() for k in "kv"}
    spans = case["T"] // BLOCK + 1
    values = {k: [] for k in "kv"}
    for b in range(B):
        p, n = _positions(case)[b], _counts(case)[b]
        rows = t["proj"][b * T:b * T + n].double()
        q, k, val, gate = rows.split((H * d, G * d, G * v, H * v), 1)
        q = (q.reshape(n, H, d) * (q.reshape(n, H, d).square().mean(-1, keepdim=True) + EPS).rsqrt() * t["q_norm"].double())
        k = (k.reshape(n, G, d) * (k.reshape(n, G, d).square().mean(-1, keepdim=True) + EPS).rsqrt() * t["k_norm"].double())
        fresh = {"k": k.to(dt).double().transpose(0, 1), "v": val.reshape(n, G, v).transpose(0, 1)}
        held, now = {}, {}
        for name in "kv":
            held[name] = t[name][b].double() * t[name + "_scale"][b].double()[..., None, None]             # (G, blocks, 64, width)
            now[name] = torch.cat((tails[name][b][:, :p % BLOCK], fresh[name]), 1)                         # from the block in progress on
        for lo in range(p // BLOCK * BLOCK, p + n, BLOCK):  # the queries of one block
            i0, i1 = max(lo, p), min(lo + BLOCK, p + n)
            at = lo - p // BLOCK * BLOCK
            keys, vals = (torch.cat((held[x][:, :lo // BLOCK].flatten(1, 2), now[x][:, at:at + i1 - lo]), 1) for x in "kv")
            s = torch.einsum("igrd,gjd->grij", q[i0 - p:i1 - p].reshape(-1, G, R, d), keys) * d ** -0.5
            i, j = (torch.arange(x, y, device=s.device) for x, y in ((i0, i1), (0, i1)))
            ok = j <= i[:, None]
            if case["window"]:
                ok &= (i[:, None] - j < case["window"]) | (j < case["keep"])
            s = torch.cat((s.masked_fill(~ok, -math.inf), torch.full_like(s[..., :1], SINK)), -1)
            o = torch.einsum("grij,gjv->igrv", torch.softmax(s, -1)[..., :-1], vals).reshape(i1 - i0, H * v)
            joint[b, i0 - p:i1 - p] = o * torch.sigmoid(gate[i0 - p:i1 - p])
            for x in "kv":
                if i1 == lo + BLOCK:
                    held[x][:, lo // BLOCK] = _stored(now[x][:, at:at + BLOCK])
                elif i1 == p + n:
                    tails[x][b, :, :i1 - lo] = now[x][:, at:at + i1 - lo]
        for x in "kv":
            values[x].append(held[x][:, p // BLOCK:p // BLOCK + spans].transpose(0, 1))
    out = {"joint": joint.reshape(B * T, -1), "k_tail": tails["k"], "v_tail": tails["v"]}
    if case["complete"] or T > 1:
        out.update({k: torch.stack(x) for k, x in values.items()})
    return out


def _adapted_exact(case, t):
    T = case["T"]
    y = t["x"].double() @ t["weight"].double().t()
    for b, s in enumerate(_slots(case)):
        if s >= 0:
            part = t["x"][b * T:(b + 1) * T].double() @ t["a"][s].double().t()
            y[b * T:(b + 1) * T] += t["scale"][s].double() * (part @ t["b"][s].double().t())
    return y


def _shaped_exact(case, t, row, slot, length):
    V, x = case["vocab"], t["logits"][row].double()
    past, first = t["history"][slot, :length].long(), int(t["start"][slot])
    all_of, drawn = torch.bincount(past, minlength=V), torch.bincount(past[first:], minlength=V)
    repetition, frequency, presence = t["penalties"][slot].double()
    x = torch.where(all_of > 0, torch.where(x > 0, x / repetition, x * repetition), x) - frequency * drawn - presence * (drawn > 0)
    used = t["bias_tokens"][slot] >= 0
    x[t["bias_tokens"][slot][used].long()] += t["bias_values"][slot][used].double()
    word = t["allowed"][slot].long() & 0xffffffff
    at = torch.arange(V, device=x.device)
    return torch.where((word[at // 32] >> at % 32) % 2 > 0, x, torch.full_like(x, -math.inf))


def exact(case, seed):
    t = {"attention": _attention_inputs, "adapted": _adapted_inputs}.get(case["kind"], _logits_inputs)(case, seed)
    if case["kind"] == "attention":
        return _attention_exact(case, t)
    if case["kind"] == "adapted":
        return _adapted_exact(case, t)
    length = t["length"].tolist()
    if case["kind"] == "shape":
        return torch.stack([_shaped_exact(case, t, i, i % case["slots"], length[i]) for i in range(case["rows"])])
    token = torch.stack([_shaped_exact(case, t, i, i, length[i]).argmax() for i in range(case["rows"])]).to(torch.int32)
    t["generated"][int(t["step"])] = token
    t["history"][torch.arange(case["rows"], device=token.device), t["length"].long()] = token
    return {"current": token, "generated": t["generated"], "history": t["history"]}
