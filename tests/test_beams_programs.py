"""One program for beams of any end and length penalty."""
import numpy as np
import pytest
import torch

import zirunex_cases as C
from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from test_beams import MODEL, generator
from test_beams_ops import backend as types  # noqa: F401  (fixture)
from test_beams_ops import beams_case
from test_dunelix_ops import i32, op
from test_zirunex import backend  # noqa: F401  (fixture)


def test_programs_do_not_add_up(backend):  # noqa: F811
    """Every call brings numbers of its own; the programs are those of the first call, and results those of a generator that has only seen them."""
    ckpt, prompts = C.checkpoint(MODEL, 4), [C.prompt(MODEL, n, seed=n) for n in (5, 3)]
    gen = generator(backend, ckpt, batch=6, beams=3, max_new_tokens=6)
    gen.generate_beams(prompts, 6)
    programs = set(gen._programs)
    for end, penalty in ((7, 0.7), (2, 0.31), (None, 0.7), (7, -0.5)):
        got = gen.generate_beams(prompts, 6, end, penalty)
        assert set(gen._programs) == programs
        want = generator(backend, ckpt, batch=6, beams=3, max_new_tokens=6).generate_beams(prompts, 6, end, penalty)
        for a, b in zip(got, want):
            assert [x.score for x in a] == [x.score for x in b] and all(np.array_equal(x.tokens, y.tokens) for x, y in zip(a, b))


@pytest.mark.parametrize("end,penalty", [(2, 0.0), (-1, 0.7), (None, -1.25), (1000, 0.5), (5, float("nan")), (5, 40.0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules_that_the_device_holds(types, end, penalty, in_place):  # noqa: F811
    """The same as with numbers given to the call; a number that is no token is no end, one that is no penalty none."""
    dev, (groups, K, V) = types[0], (5, 4, 999)
    logits, scores, ended, length = (x.to(dev) for x in beams_case(types, groups, K, V, V, 3))
    out = []
    for ruled in (True, False):
        state, n = [x.clone() for x in (scores, ended, length)], groups * K
        into = [] if in_place else [torch.full_like(x, -9) for x in state]
        results = [i32(types, *[-7] * n) for _ in range(2)] + [torch.full((3, n), -7, dtype=torch.int32, device=dev) for _ in range(2)]
        number = -1 if end is None else end
        given = dict(end=-1, length_penalty=0.0) if ruled else dict(end=number if 0 <= number < V else -1, length_penalty=penalty if abs(penalty) <= 32 else 0.0)
        rule = [i32(types, number), torch.tensor([penalty], dtype=torch.float64, device=dev)] if ruled else []
        op("take_beams_", types, results[0], results[1], logits, *results[2:], i32(types, 1), *state, *into, *rule, beams=K, valid=V, base=0, ahead=0, advance=True, **given)
        out.append([*results, *state, *into])
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(*out))


def test_refusals_of_rules():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def call(rule, **kw):
            state = ops.BeamState(var((8,), xl.float32), var((8,)), var((8,)))
            return ops.take_beams_(var((8,)), var((8,)), var((8, 50), xl.float32), var((5, 8)), var((5, 8)), kw.pop("step", None) or var((1,)), state, 4, rule=rule, **kw)

        rule = ops.BeamRule(var((1,)), var((1,), xl.float64))
        call(rule)
        for bad, kw in ((rule, dict(end=3)), (rule, dict(length_penalty=0.5)), (rule, dict(step=rule.end)), (ops.BeamRule(var((2,)), rule[1]), {}),
                        (ops.BeamRule(rule.end, var((1,), xl.float32)), {})):
            with pytest.raises(ValueError):
                call(bad, **kw)
    gen = generator(("cpu", "float32"), C.checkpoint(MODEL, 1), batch=2, beams=2, max_new_tokens=3)
    for penalty in (float("nan"), 33.0):
        with pytest.raises(ValueError, match="length penalty"):
            gen.generate_beams([[1, 2]], 2, length_penalty=penalty)
    assert not gen.slots
