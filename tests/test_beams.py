"""Beam search and shared prefixes through `SequenceGenerator`, against plain float64 models. CPU backend, and marked `gpu` the kernels in
32 bits and bf16."""

import numpy as np
import pytest
import torch

import dunelix_cases as D
import zirunex_cases as C
from popxl_addons_b200.models.dunelix import Dunelix, DunelixConfig
from popxl_addons_b200.models.sequence_generator import LogitShaping, SequenceGenerator
from popxl_addons_b200.models.zirunex import Zirunex, ZirunexConfig
from test_serving import MODEL
from test_zirunex import backend, run  # noqa: F401  (fixture and helper)


def generator(backend, ckpt, batch=3, cfg=MODEL, options=None, **kw):  # noqa: F811
    device, dtype = backend
    kw.setdefault("max_seq", 220)
    return SequenceGenerator(Zirunex(ZirunexConfig.from_dict(cfg), dtype, **(options or {})), batch=batch, device=device, **kw).load_checkpoint(ckpt)


def log_probs(logits):
    return torch.log_softmax(torch.as_tensor(logits).double(), -1)


def replay(gen, prompt, tokens, shaping=None):
    """The sum of a continuation by the generator's own logits, one request by itself."""
    seq = list(prompt) + [int(t) for t in tokens]
    gen.admit("one", None, shaping, len(prompt))
    want = list(range(len(prompt) - 1, len(seq) - 1))
    out = log_probs(gen.step({"one": seq[:-1]}, {"one": want}, shaped=shaping is not None)["one"])
    gen.release("one")
    return sum(float(out[i, t]) for i, t in enumerate(tokens))


def plain_search(oracle, prompt, n_new, K, end, penalty):
    """Beam search over a function of the tokens so far, in float64: `[(tokens, sum)]`, the best first."""
    beams = [((), 0.0, False)]
    for _ in range(n_new):
        found = []
        for k, (tokens, total, done) in enumerate(beams):
            if done:
                found.append((tokens, total, True))
                continue
            lp = oracle(list(prompt) + list(tokens))
            found += [(tokens + (v,), total + float(lp[v]), v == end) for v in range(len(lp))]
        beams = sorted(found, key=lambda b: -b[1] / max(1, len(b[0])) ** penalty)[:K]
    return beams


TOL = {"float32": 2e-3, "bfloat16": 0.2}  # of a sum of some ten logarithms, each off by the tolerance of a logit


@pytest.mark.parametrize("options", [{}, {"shared_prefixes": True}, {"cache": "int8"}], ids=["copied", "shared", "int8"])
def test_beams_of_unequal_prompts(backend, options):  # noqa: F811
    """Every sum is what the model gives the continuation by itself; the best ones are those of a plain search (32 bits, where rounding decides
    nothing); more prompts than there are groups; portions shorter than prompts."""
    ckpt = C.checkpoint(MODEL, 4)
    prompts = [C.prompt(MODEL, n, seed=n) for n in (5, 71, 1)]
    gen = generator(backend, ckpt, batch=8, options=options, beams=4, max_portion=32, max_new_tokens=9)
    alone = generator(backend, ckpt, batch=1, options={k: v for k, v in options.items() if k == "cache"})
    for end, penalty in ((None, 0.0), (7, 0.7)):
        out = gen.generate_beams(prompts, 9, end, penalty)
        assert len(out) == 3 and not gen.slots and len(gen._free) == 8
        for prompt, beams in zip(prompts, out):
            assert len(beams) == 4 and len({tuple(b.tokens) for b in beams}) == 4
            ranks = [b.score / len(b.tokens) ** penalty for b in beams]
            assert ranks == sorted(ranks, reverse=True)
            for b in beams:
                assert len(b.tokens) == 9 or b.tokens[-1] == end
                assert end is None or end not in b.tokens[:-1]
                assert abs(replay(alone, prompt, b.tokens) - b.score) < TOL[backend[1]]
        if backend[1] == "float32" and "cache" not in options:
            def oracle(seq):
                return log_probs(C.oracle_logits(MODEL, ckpt, seq)[-1])

            want = plain_search(oracle, prompts[0], 9, 4, end, penalty)
            assert [tuple(b.tokens) for b in out[0]] == [w[0] for w in want]
            assert all(abs(b.score - w[1]) < TOL["float32"] for b, w in zip(out[0], want))


def test_one_beam_is_the_greedy_choice(backend):  # noqa: F811
    ckpt, prompts = C.checkpoint(MODEL, 5), [C.prompt(MODEL, 20, seed=1), C.prompt(MODEL, 3, seed=2)]
    greedy = generator(backend, ckpt, batch=2).generate(prompts, 8)
    for options in ({}, {"shared_prefixes": True}):
        out = generator(backend, ckpt, batch=2, options=options, beams=1).generate_beams(prompts, 8)
        if options == {}:
            assert all(np.array_equal(a, b[0].tokens) for a, b in zip(greedy, out))
        else:  # another kernel: the choice may differ where two logits are closer than its rounding
            assert all(a[0] == b[0].tokens[0] for a, b in zip(greedy, out))


def test_beams_of_shaped_logits_and_adapters(backend):  # noqa: F811
    """Penalties follow the beam's own tokens, masks its slot's rules, adapters its request."""
    ckpt, prompt = C.checkpoint(MODEL, 6), C.prompt(MODEL, 40, seed=3)
    shaping = LogitShaping(1.3, 0.2, 0.1, {5: 1.5}, list(range(3, 60)))
    for options in ({}, {"shared_prefixes": True}):
        gen = generator(backend, ckpt, batch=6, options=options, beams=3, shaping=True)
        alone = generator(backend, ckpt, batch=1, shaping=True)
        out = gen.generate_beams([prompt, prompt], 7, shaping=[shaping, None])
        for b in out[0]:
            assert all(3 <= t < 60 for t in b.tokens)
            assert abs(replay(alone, prompt, b.tokens, shaping) - b.score) < TOL[backend[1]]
        for b in out[1]:
            assert abs(replay(alone, prompt, b.tokens) - b.score) < TOL[backend[1]]


def test_beams_of_recurrent_models(backend):  # noqa: F811
    """States without positions and caches of two maps follow their beams."""
    device, dtype = backend
    cfg = next(iter(D.CASES.values()))
    ckpt = D.checkpoint(cfg)

    def make(batch, **kw):
        return SequenceGenerator(Dunelix(DunelixConfig.from_dict(cfg), dtype), batch=batch, max_seq=64, device=device, **kw).load_checkpoint(ckpt)

    prompts = [D.prompt(cfg, 9, seed=1), D.prompt(cfg, 2, seed=2)]
    out, alone = make(6, beams=3).generate_beams(prompts, 6), make(1)
    for prompt, beams in zip(prompts, out):
        assert len({tuple(b.tokens) for b in beams}) == 3
        for b in beams:
            assert abs(replay(alone, prompt, b.tokens) - b.score) < TOL[dtype]


def test_requests_behind_one_prefix(backend):  # noqa: F811
    """Logits of requests that share a system prompt are those of whole sequences; the holder may go on, be released first, and its slot comes back
    when nobody shares it any more; a request shares on what it shares itself."""
    ckpt = C.checkpoint(MODEL, 7)
    system, tails = C.prompt(MODEL, 90, seed=1), [C.prompt(MODEL, n, seed=10 + n) for n in (4, 17, 1)]
    gen = generator(backend, ckpt, batch=5, options={"shared_prefixes": True})
    gen.admit("system")
    gen.step({"system": system})
    gen.admit("a", prefix_of="system")
    gen.admit("b", prefix_of="system", prefix=61)
    gen.admit("c", prefix_of="a", prefix=90)
    whole = {"a": list(system) + list(tails[0]), "b": list(system[:61]) + list(tails[1]), "c": list(system) + list(tails[2])}
    held = {"a": 90, "b": 61, "c": 90}
    more = C.prompt(MODEL, 30, seed=5)
    got = gen.step({**{r: s[held[r]:] for r, s in whole.items()}, "system": more}, {r: range(len(s) - held[r]) for r, s in whole.items()})
    tol = C.TOLERANCE[backend[1]]
    for r, s in whole.items():
        assert C.error(got[r], C.oracle_logits(MODEL, ckpt, s)[held[r]:]) < tol, r
    gen.release("system")
    assert len(gen._free) == 1
    step = {r: [s[-1]] for r, s in whole.items()}
    got = gen.step(step, {r: [0] for r in step})  # single tokens, the holder gone
    for r, s in whole.items():
        assert C.error(got[r], C.oracle_logits(MODEL, ckpt, s + [s[-1]])[-1:]) < tol, r
    for r in ("a", "b", "c"):
        gen.release(r)
    assert sorted(gen._free) == [0, 1, 2, 3, 4] and not gen._kept
    gen.admit("again")
    assert C.error(gen.step({"again": system}, {"again": range(90)})["again"], C.oracle_logits(MODEL, ckpt, system)) < tol


def test_refusals():
    ckpt = C.checkpoint(MODEL, 1)
    cpu = ("cpu", "float32")
    with pytest.raises(ValueError, match="beams"):
        generator(cpu, ckpt, batch=3, beams=2)
    with pytest.raises(ValueError, match="shared"):
        generator(cpu, ckpt, options={"cache": "int8", "shared_prefixes": True})
    gen = generator(cpu, ckpt, batch=2)
    with pytest.raises(ValueError, match="without beams"):
        gen.generate_beams([[1]], 2)
    gen.admit("x")
    with pytest.raises(ValueError, match="without shared"):
        gen.admit("y", prefix_of="x")
    gen = generator(cpu, ckpt, batch=4, options={"shared_prefixes": True}, beams=2, max_new_tokens=5)
    for kw in (dict(max_new_tokens=6), dict(max_new_tokens=0), dict(max_new_tokens=2, end=96), dict(max_new_tokens=2, shaping=[None, None])):
        with pytest.raises(ValueError):
            gen.generate_beams([[1, 2]], **kw)
    with pytest.raises(ValueError):
        gen.generate_beams([[]], 2)
    gen.admit("x")
    with pytest.raises(RuntimeError):
        gen.generate_beams([[1]], 2)
    gen.step({"x": [1, 2, 3]})
    for kw in (dict(prefix_of="nobody"), dict(prefix_of="x", prefix=4), dict(prefix_of="x", prefix=-1)):
        with pytest.raises(ValueError):
            gen.admit("y", **kw)
    gen.admit("y", prefix_of="x", prefix=2)
    gen.step({"y": [4, 5]})
    with pytest.raises(ValueError, match="itself"):
        gen.admit("z", prefix_of="y")
    assert len(gen._free) == 2
