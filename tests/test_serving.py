"""Batches of unlike requests through `SequenceGenerator`: caches of 8 bits, adapters, shaped logits, one by one and together,
against plain float64 implementations. CPU backend, and marked `gpu` the kernels in 32-bit and bf16."""
import numpy as np
import pytest
import torch

import plain_serving as plain
import plain_zirunex as plain_model
import zirunex_cases as C
from popxl_addons_b200.models.sequence_generator import LogitShaping, SequenceGenerator
from popxl_addons_b200.models.zirunex import Zirunex, ZirunexConfig
from test_zirunex import backend, run  # noqa: F401  (fixture and helper)

# sizes of every kernel: tensor cores, mma.sync and the general one, with and without windows, shared weights, no feed-forward
MODEL = C.config([C.layer(C.attention(heads=4, kv_heads=2, dim=64, vdim=64, size=70, keep=3), 64),
                  C.layer(C.attention(heads=3, kv_heads=1, dim=24, vdim=16, size=0), 0),
                  C.layer(C.attention(heads=4, kv_heads=2, dim=64, vdim=64, size=70, keep=3), 64, weights_of=0),
                  C.layer(C.attention(heads=8, kv_heads=1, dim=32, vdim=80, size=9, keep=40), 40)], width=64, vocab=96)


def generator(backend, ckpt, batch=3, cfg=MODEL, options=None, **kw):  # noqa: F811
    device, dtype = backend
    kw.setdefault("max_seq", 220)
    return SequenceGenerator(Zirunex(ZirunexConfig.from_dict(cfg), dtype, **(options or {})), batch=batch, device=device, **kw).load_checkpoint(ckpt)


def attention_of_8_bits(h, w, mix, eps):
    """What `plain_zirunex.window_attention` is for a cache of 8 bits, with keys held in fp64 until they become codes."""
    m = mix.get("mask") or {}
    rows = torch.cat([h @ w[k].T for k in ("q", "k", "v", "g")], 1)
    out, _, _ = plain.q8_attention(rows, w["q.norm"], w["k.norm"], mix["heads"], mix["kv_heads"], mix["dim"], mix["vdim"], m.get("size") or 0,
                                   m.get("keep_first") or 0, mix["scale"], 0.0, eps, torch.float64)
    return out @ w["o"].T


def test_cache_of_8_bits(backend, monkeypatch):  # noqa: F811
    """Logits of every position, cut in many ways, against the plain model with such a cache. Where products are 32-bit a key is off
    by some 2^-20 and lands on the other side of a border between two codes in one of some thousand cases: single steps of 1/127 of
    a block's largest value among 64 features, less than 1 % of a score and 2e-3 of the logits. Without codes the logits differ by
    more than that."""
    ckpt, tokens = C.checkpoint(MODEL, 4), C.prompt(MODEL, 150)
    unquantised = C.oracle_logits(MODEL, ckpt, tokens)
    monkeypatch.setattr(plain_model, "window_attention", attention_of_8_bits)
    want = C.oracle_logits(MODEL, ckpt, tokens)
    assert 2e-3 < C.error(unquantised, want) < 0.1
    gen = generator(backend, ckpt, options={"cache": "int8"})
    tol = max(2e-3, C.TOLERANCE[backend[1]])
    for cuts in ([150], [1], [3, 5, 17, 2, 1, 19, 64, 8, 31], [128, 22]):
        assert C.error(run(gen, tokens, cuts), want) < tol, cuts


def adapter_tensors(seed, ranks):
    """An adapter for some matrices of the model: `ranks` by checkpoint name."""
    g, shapes = torch.Generator().manual_seed(seed), Zirunex(ZirunexConfig.from_dict(MODEL)).checkpoint_tensors()
    out = {}
    for name, r in ranks.items():
        n, k = shapes[name]
        out[name + ".a"] = (torch.randn(r, k, generator=g) * k ** -0.5).to(torch.bfloat16)
        out[name + ".b"] = (torch.randn(n, r, generator=g) * 0.5 * r ** -0.5).to(torch.bfloat16)
    return out


ADAPTERS = [({"l0.mix.q": 4, "l0.mix.v": 4, "l0.mlp.gate": 2, "l0.mix.o": 3, "l0.mlp.down": 4}, 1.5),
            ({"l1.mix.q": 8, "l1.mix.k": 1, "l3.mlp.up": 5, "l3.mix.g": 5, "l1.mix.o": 8}, 0.5)]


def merged(ckpt, index):
    """The checkpoint with an adapter's products added to its matrices."""
    out = {k: v.double() for k, v in ckpt.items()}
    ranks, scale = ADAPTERS[index]
    t = adapter_tensors(index, ranks)
    for name in ranks:
        out[name] = out[name] + scale * (t[name + ".b"].double() @ t[name + ".a"].double())
    return out


def load_adapters(gen):
    for i, (ranks, scale) in enumerate(ADAPTERS):
        gen.load_adapter(i, adapter_tensors(i, ranks), scale)
    return gen


def test_adapters_of_unlike_requests(backend):  # noqa: F811
    """Three requests in one batch, with either adapter and with none, in portions of unequal lengths and token by token: each gets the
    logits of the model into whose matrices its adapter has been merged. A slot that had an adapter has none for the next request."""
    ckpt, tokens = C.checkpoint(MODEL, 5), C.prompt(MODEL, 90)
    want = {a: plain_model.forward(MODEL, merged(ckpt, a) if a is not None else {k: v.double() for k, v in ckpt.items()}, tokens).numpy()
            for a in (0, 1, None)}
    assert C.error(want[0], want[None]) > 0.1 and C.error(want[1], want[None]) > 0.1
    gen = load_adapters(generator(backend, ckpt, options={"adapters": 2, "adapter_rank": 12}))
    for order in ((0, 1, None), (None, 0, 1), (1, None, None)):
        for k, a in enumerate(order):
            gen.admit(k, adapter=a)
        got = {k: [] for k in range(3)}
        for at, n in ((0, 80), (80, 1), (81, 1), (82, 8)):
            part = {k: tokens[at:at + n] for k in range(3)}
            for k, x in gen.step(part, {k: range(n) for k in range(3)}).items():
                got[k].append(x)
        for k, a in enumerate(order):
            gen.release(k)
            assert C.error(np.concatenate(got[k]), want[a]) < C.TOLERANCE[backend[1]], (order, k)


SHAPINGS = [LogitShaping(), LogitShaping(repetition=1.7), LogitShaping(1.2, 0.6, 0.9, biases={5: 2.5, 7: -9.0}),
            LogitShaping(biases={3: 4.0}, allowed=[3, 4, 5, 8, 13, 21, 34, 55, 89]), LogitShaping(frequency=-0.5, presence=0.2)]


def shaped_row(x, history, prompt, s, vocab):
    allowed = [s.allowed is None or v in s.allowed for v in range(vocab)]
    return plain.shaped(x, list(history), prompt, (s.repetition, s.frequency, s.presence), list((s.biases or {}).items()), allowed).numpy()


def test_shaped_generation(backend):  # noqa: F811
    """The tokens that a caller would choose from the logits by the formulas, for requests with rules of their own in one batch and
    more prompts than slots. bf16 tokens are compared only where the best two logits are further apart than rounding."""
    ckpt, vocab, new = C.checkpoint(MODEL, 6), MODEL["vocab"], 12
    prompts = [list(C.prompt(MODEL, n)) for n in (9, 1, 30, 17, 64)]
    gen = generator(backend, ckpt, batch=2, max_new_tokens=16, shaping=True)
    out = gen.generate(prompts, new, SHAPINGS)
    plain_out = gen.generate(prompts, new)
    assert any(list(a) != list(b) for a, b in zip(out, plain_out))
    ref = generator(backend, ckpt, batch=2, max_new_tokens=16)
    assert [list(x) for x in ref.generate(prompts, new)] == [list(x) for x in plain_out]  # rules that change nothing
    exact = backend[1] == "float32"
    for p, s, got in zip(prompts, SHAPINGS, out):
        history = list(p)
        for i, token in enumerate(got):
            ref.admit("r")
            row = ref.step({"r": history}, {"r": [len(history) - 1]})["r"][0]
            ref.release("r")
            want = shaped_row(row, history, len(p), s, vocab)
            best = np.sort(want)[-2:]
            if exact or best[1] - best[0] > 0.05 * np.abs(row).max():
                assert int(token) == int(want.argmax()), (s, i)
            history.append(int(token))


def test_shaped_logits_of_steps(backend):  # noqa: F811
    """A caller that samples itself: the shaped logits of several places of a portion, the mask changed between steps."""
    ckpt, vocab = C.checkpoint(MODEL, 6), MODEL["vocab"]
    gen = generator(backend, ckpt, shaping=True, max_biases=4)
    tokens = list(C.prompt(MODEL, 40))
    for k, s in enumerate(SHAPINGS[1:4]):
        gen.admit(k, shaping=s, prompt=10)
    at = 0
    for n in (25, 1, 14):
        if at:
            gen.set_allowed(1, [1, 2, 90])
        part, places = {k: tokens[at:at + n] for k in range(3)}, {k: [n - 1, 0] for k in range(3)}
        got, slots = gen.step(part, places, shaped=True), dict(gen.slots)
        for k, s in enumerate(SHAPINGS[1:4]):
            other = generator(backend, ckpt)
            other.admit(k)
            rows = other.step({k: tokens[:at + n]}, {k: [at + n - 1, at]})[k]
            rule = LogitShaping(s.repetition, s.frequency, s.presence, s.biases, [1, 2, 90]) if at and k == 1 else s
            for row, x, place in zip(rows, got[k], (n - 1, 0)):
                want = shaped_row(row, tokens[:at + place + 1], 10, rule, vocab)
                fine = np.isfinite(want)
                assert np.array_equal(fine, np.isfinite(x))
                assert np.abs(x[fine] - want[fine]).max() < 2 * C.TOLERANCE[backend[1]] * np.abs(row).max()
        assert slots == gen.slots
        at += n


def test_everything_together(backend):  # noqa: F811
    """Unlike requests with 8-bit caches, adapters and rules: each in a batch as it is alone."""
    ckpt, options = C.checkpoint(MODEL, 7), {"cache": "int8", "adapters": 2, "adapter_rank": 12}
    prompts = [list(C.prompt(MODEL, n)) for n in (70, 3, 129)]
    adapters, shapings = [1, None, 0], [SHAPINGS[2], SHAPINGS[3], None]
    gen = load_adapters(generator(backend, ckpt, options=options, shaping=True, max_new_tokens=16))
    together = gen.generate(prompts, 10, shapings, adapters)
    again = gen.generate(prompts, 10, shapings, adapters)
    assert [list(x) for x in together] == [list(x) for x in again]
    if backend[1] == "float32":
        for p, a, s, got in zip(prompts, adapters, shapings, together):
            assert list(gen.generate([p], 10, [s], [a])[0]) == list(got)
    assert gen.slots == {} and len(gen._free) == 3


def test_refusals(tmp_path):
    ckpt = C.checkpoint(MODEL, 7)
    gen = generator(("cpu", "float32"), ckpt, batch=1, shaping=True, max_biases=2)
    for bad in (LogitShaping(repetition=0.0), LogitShaping(frequency=float("nan")), LogitShaping(biases={1: 1.0, 2: 1.0, 3: 1.0}),
                LogitShaping(biases={96: 1.0}), LogitShaping(allowed=[]), LogitShaping(allowed=[96]), LogitShaping(allowed=np.zeros(96, bool))):
        with pytest.raises(ValueError):
            gen.admit("r", shaping=bad)
        assert not gen.slots and len(gen._free) == 1
    with pytest.raises(ValueError, match="adapter 0 of 0"):
        gen.admit("r", adapter=0)
    with pytest.raises(ValueError, match="without adapters"):
        gen.load_adapter(0, {})
    with pytest.raises(ValueError, match="as many shapings"):
        gen.generate([[1], [2]], 1, [None])
    plain_gen = generator(("cpu", "float32"), ckpt, batch=1)
    with pytest.raises(ValueError, match="shaping=True"):
        plain_gen.admit("r", shaping=LogitShaping())
    with pytest.raises(ValueError, match="shaping=True"):
        plain_gen.step({}, shaped=True)
    with pytest.raises(ValueError, match="held as"):
        generator(("cpu", "float32"), ckpt, options={"cache": "fp4"})
    with pytest.raises(ValueError, match="rank"):
        generator(("cpu", "float32"), ckpt, options={"adapters": 1, "adapter_rank": 129})
    gen = generator(("cpu", "float32"), ckpt, options={"adapters": 1, "adapter_rank": 4})
    t = adapter_tensors(0, {"l0.mix.q": 3, "l0.mix.k": 2})
    with pytest.raises(ValueError, match="rank of 5 together"):
        gen.load_adapter(0, t)
    with pytest.raises(ValueError, match="both halves"):
        gen.load_adapter(0, {"l0.mix.q.a": t["l0.mix.q.a"]})
    with pytest.raises(ValueError, match="unexpected adapter tensors"):
        gen.load_adapter(0, {"l2.mix.q.a": t["l0.mix.q.a"]})
    with pytest.raises(ValueError, match="the adapter of 'l0.mix.k' is"):
        gen.load_adapter(0, {"l0.mix.k.a": t["l0.mix.k.a"][:, 1:], "l0.mix.k.b": t["l0.mix.k.b"]})


def test_command_line(tmp_path, capsys):
    """A cache of 8 bits and penalties from the command line."""
    from popxl_addons_b200.generate import main

    C.write_model(tmp_path, MODEL, C.checkpoint(MODEL, 8))
    args = ["--model", str(tmp_path), "--prompt", "5 17 3", "--max-new-tokens", "40", "--dtype", "float32", "--device", "cpu"]
    for more in (["--cache", "int8"], ["--repetition-penalty", "1.5", "--frequency-penalty", "1000"]):
        assert main(args + more) == 0
        out = capsys.readouterr().out.split()
        assert len(out) == 40
    assert len(set(out)) == 40  # a token that was chosen once is not chosen again
