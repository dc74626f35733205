"""Beams and shared prefixes of requests that bring adapters, shaped logits and an early end. CPU backend, and marked `gpu` the kernels."""
import numpy as np
import pytest

import plain_zirunex as plain_model
import zirunex_cases as C
from popxl_addons_b200.models.sequence_generator import LogitShaping
from test_beams import TOL, generator, log_probs
from test_serving import MODEL, load_adapters, merged
from test_zirunex import backend  # noqa: F401  (fixture)

ADAPTED = {"adapters": 2, "adapter_rank": 12}


@pytest.mark.parametrize("options", [{}, {"shared_prefixes": True}], ids=["copied", "shared"])
def test_beams_of_unlike_adapters(backend, options):  # noqa: F811
    """Every sum is that of the continuation by itself with the prompt's adapter; with another one (32 bits) some beam's is not."""
    ckpt, prompt = C.checkpoint(MODEL, 5), C.prompt(MODEL, 40, seed=3)
    gen = load_adapters(generator(backend, ckpt, batch=9, options={**ADAPTED, **options}, beams=3))
    alone = load_adapters(generator(backend, ckpt, batch=1, options=ADAPTED))
    adapters = [0, None, 1]
    out = gen.generate_beams([prompt] * 3, 6, adapters=adapters)
    for a, beams in zip(adapters, out):
        assert len({tuple(b.tokens) for b in beams}) == 3
        off = {other: 0.0 for other in adapters}
        for b in beams:
            seq, sums = list(prompt) + [int(t) for t in b.tokens], {}
            for other in adapters:
                alone.admit("one", adapter=other)
                lp = log_probs(alone.step({"one": seq[:-1]}, {"one": range(39, 45)})["one"])
                alone.release("one")
                sums[other] = sum(float(lp[i, t]) for i, t in enumerate(b.tokens))
            off = {other: max(off[other], abs(s - b.score)) for other, s in sums.items()}
        assert off.pop(a) < TOL[backend[1]]
        assert backend[1] != "float32" or min(off.values()) > 2 * TOL["float32"]


def test_prefixes_of_adapted_requests(backend):  # noqa: F811
    """Positions that an adapter's products made are shared by requests with the same adapter only."""
    ckpt, tokens = C.checkpoint(MODEL, 5), C.prompt(MODEL, 90)
    gen = load_adapters(generator(backend, ckpt, batch=4, options={**ADAPTED, "shared_prefixes": True}))
    gen.admit("a", adapter=1)
    gen.step({"a": tokens[:70]})
    for other in (0, None):
        with pytest.raises(ValueError, match="another adapter"):
            gen.admit("b", adapter=other, prefix_of="a")
    assert len(gen._free) == 3 and set(gen.slots) == {"a"}
    gen.admit("b", adapter=1, prefix_of="a", prefix=64)
    got = gen.step({"b": tokens[64:]}, {"b": range(26)})["b"]
    assert C.error(got, plain_model.forward(MODEL, merged(ckpt, 1), tokens).numpy()[64:]) < C.TOLERANCE[backend[1]]


def test_prefixes_of_shaped_requests(backend):  # noqa: F811
    """Tokens of shared positions count among a request's own, by its own rules, whatever the rules of the request that read them."""
    ckpt, tokens = C.checkpoint(MODEL, 6), C.prompt(MODEL, 60, seed=4)
    rules = LogitShaping(1.6, 0.4, 0.3, {5: 1.5}, list(range(1, 90)))
    gen = generator(backend, ckpt, batch=3, options={"shared_prefixes": True}, shaping=True)
    gen.admit("a", shaping=LogitShaping(repetition=1.1), prompt=50)
    gen.step({"a": tokens[:50]})
    for prompt in (10, 50):
        gen.admit("b", shaping=rules, prompt=prompt, prefix_of="a", prefix=45)
        gen.admit("whole", shaping=rules, prompt=prompt)
        got = gen.step({"b": tokens[45:], "whole": tokens}, {"b": range(15), "whole": range(45, 60)}, shaped=True)
        low = got["whole"] < -1e30  # tokens that are not allowed
        assert np.array_equal(low, got["b"] < -1e30) and low.any()
        assert C.error(np.where(low, 0, got["b"]), np.where(low, 0, got["whole"])) < C.TOLERANCE[backend[1]]
        plainly = gen.step({"whole": [1]}, {"whole": [0]})["whole"]
        assert np.isfinite(plainly).all()
        gen.release("b")
        gen.release("whole")


def test_beams_that_have_all_ended(backend, monkeypatch):  # noqa: F811
    """Steps end when no beam goes on, which is looked at every 16 of them; results are those of the tokens until then."""
    ckpt, prompts, end = C.checkpoint(MODEL, 6), [C.prompt(MODEL, n, seed=n) for n in (12, 5)], 7
    likely = LogitShaping(biases={end: 12.0})
    gen = generator(backend, ckpt, batch=6, beams=3, shaping=True, max_new_tokens=60)
    ran, run = [], gen.session.run_program
    monkeypatch.setattr(gen.session, "run_program", lambda p, *a, **kw: ran.append(p) or run(p, *a, **kw))
    out = gen.generate_beams(prompts, 60, end, 0.6, shaping=likely)
    assert len(ran) == 16 and all(b.tokens[-1] == end and len(b.tokens) < 16 for beams in out for b in beams)
    short = gen.generate_beams(prompts, 16, end, 0.6, shaping=likely)
    for a, b in zip(out, short):
        assert [x.score for x in a] == [x.score for x in b] and all(np.array_equal(x.tokens, y.tokens) for x, y in zip(a, b))
    del ran[:]
    gen.generate_beams(prompts, 20, None, 0.6, shaping=likely)
    assert len(ran) == 20  # nothing ends
