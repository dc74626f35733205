"""What the ops and the generator of sequences with a common beginning refuse, beside what the tests of each of them have."""
import math

import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from test_beams_ops import backend, check_beams  # noqa: F401  (fixture and helper)


def var(shape, dt=xl.int32):
    return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)


@pytest.fixture
def graph():
    ir = xl.Ir()
    with ir.main_graph:
        yield ir


def choose(n=8, **kw):
    """A call of `take_beams_` with tensors of its own, but for those given."""
    kw = dict(current=var((n,)), parent=var((n,)), logits=var((n, 50), xl.float32), buf=var((5, n)), parents=var((5, n)), step=var((1,)),
              state=ops.BeamState(var((n,), xl.float32), var((n,)), var((n,))), beams=min(n, 4)) | kw
    return ops.take_beams_(**kw)


def test_a_choice_among_no_entries(graph):
    choose(valid=50)
    with pytest.raises(ValueError, match="choice among 0 entries"):
        choose(valid=0)


def test_results_on_top_of_the_step(graph):
    """One beam: its token and the number of the step have the same shape, and whether the step is read first is up to the kernel."""
    choose(1)
    for name in ("current", "parent", "buf", "parents"):
        step = var((1, 1)) if name.startswith("b") or name == "parents" else var((1,))
        with pytest.raises(ValueError, match="of their own"):
            choose(1, **{"step": step, name: step}, **({"parents": var((1, 1))} if name == "buf" else {"buf": var((1, 1))} if name == "parents" else {}))


def test_attention_on_top_of_its_projections(graph):
    def call(proj, joint):
        k, v = var((3, 2, 30, 16), xl.float32), var((3, 2, 30, 24), xl.float32)
        return ops.window_attention_shared_(proj, var((16,), xl.float32), var((16,), xl.float32), k, v, *(var((3,)) for _ in range(4)), joint, 1, 4, 0.5)

    proj = var((3, 240), xl.float32)
    call(proj, var((3, 240), xl.float32))
    with pytest.raises(ValueError, match="on top of the projections"):
        call(proj, proj)


@pytest.mark.parametrize("penalty", [ops.MAX_PENALTY, -ops.MAX_PENALTY])
def test_the_largest_length_penalties(backend, penalty):  # noqa: F811
    """Sums of unlike beams stay unlike when divided by the largest number of tokens to the largest power."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(4, 200, generator=g).to(backend[1])
    for tokens in (1, 1500, 0x7ffffff0):
        length = torch.full((4,), tokens, dtype=torch.int32)
        assert math.isfinite(float(tokens + 1) ** penalty)
        check_beams(backend, logits, torch.tensor([-1.0, -1.25, -2.0, -0.5]), torch.zeros(4, dtype=torch.int32), length, 4, 3, 200, float(penalty))


def test_length_penalties_whose_powers_overflow(graph):
    choose(length_penalty=float(ops.MAX_PENALTY))
    for penalty in (100.0, -100.0, 32.5):  # 2000 tokens to the power of 100 are infinite, and all sums divided by it zero
        with pytest.raises(ValueError, match="length penalty"):
            choose(length_penalty=penalty)


def test_a_prefix_of_nobody():
    import zirunex_cases as C
    from test_beams import MODEL, generator

    gen = generator(("cpu", "float32"), C.checkpoint(MODEL, 1), options={"shared_prefixes": True})
    gen.admit("x")
    gen.step({"x": [1, 2, 3]})
    with pytest.raises(ValueError, match="no request"):
        gen.admit("y", prefix=2)
    assert gen.slots == {"x": 0} and len(gen._free) == 2
