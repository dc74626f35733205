"""Shaped logits and the choice from them against the plain oracle. Rows of odd lengths, so that rows start off 16-byte boundaries;
masks that leave one token and none; tokens that occur often, twice in a bias list, and outside the vocabulary. CPU backend, and
marked `gpu` the kernels."""
import math

import pytest
import torch

import plain_serving as plain
from test_dunelix_ops import backend, i32, op, rnd  # noqa: F401  (fixture and helpers)
from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from popxl_addons_b200.xl.opdef import OPS

# every one of at most five roundings (quotient or product, product, two differences, a sum of at most three biases) is off by at
# most 2^-24 of a number below 64: 8 * 2^-24 * 64
TOLERANCE = 8 * 64 * 2.0 ** -24


def bits_of(allowed):
    """`(slots, vocab)` truth values -> words."""
    S, V = allowed.shape
    padded = torch.zeros(S, -(-V // 32) * 32, dtype=torch.int64)
    padded[:, :V] = allowed
    word = (padded.reshape(S, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(word > 0x7fffffff, word - (1 << 32), word).to(torch.int32)


def rules(S, V, L, K, seed=0):
    """Host tensors of the rules, and the truth values of the masks. Slot 0 has no penalties, slot 1 allows a single token, slot 2
    nothing at all; tokens are drawn from few, so that some occur often; some lie outside the vocabulary."""
    g = torch.Generator().manual_seed(seed)
    history = torch.randint(-1, max(2, V // 3), (S, L), generator=g)
    history[:, ::5] = V - 1  # the last entry of a row
    history[:, 1::7] = V + 3
    allowed = torch.rand(S, V, generator=g) < 0.7
    if S > 1:
        allowed[1] = False
        allowed[1, V // 2] = True
    if S > 2:
        allowed[2] = False
    penalties = torch.stack((1 + torch.rand(S, generator=g), torch.rand(S, generator=g), torch.rand(S, generator=g)), 1)
    penalties[0] = torch.tensor([1.0, 0.0, 0.0])
    tokens = torch.randint(-1, V + 1, (S, K), generator=g)
    if K > 4:
        tokens[:, 3] = tokens[:, 0]  # listed twice
        tokens[:, 4] = V - 1
    values = torch.randn(S, K, generator=g)
    start = torch.randint(0, L + 1, (S,), generator=g)
    return [history.int(), start.int(), penalties, tokens.int(), values, bits_of(allowed)], allowed


def want(logits, s, length, r, allowed):
    return plain.shaped(logits, r[0][s][:length].tolist(), int(r[1][s]), r[2][s], list(zip(r[3][s].tolist(), r[4][s])), allowed[s])


def same(got, ref, tol=TOLERANCE):
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(ref))
    fine = torch.isfinite(ref)
    assert (got[fine] - ref[fine]).abs().max().item() <= tol if fine.any() else True


@pytest.mark.parametrize("rows,S,V,L,K", [(1, 1, 7, 1, 0), (3, 2, 33, 5, 1), (5, 4, 1021, 64, 6), (4, 3, 8192, 300, 40),
                                          (2, 3, 50257, 2000, 300), (130, 3, 100, 9, 5), (1, 1, 300001, 40, 3)])
def test_shaped_logits(backend, rows, S, V, L, K):  # noqa: F811
    if backend[0] == "cpu" and V > 10000 and rows > 2:
        pytest.skip("covered by the smaller ones")
    r, allowed = rules(S, V, L, K)
    g = torch.Generator().manual_seed(5)
    logits = (torch.randn(rows, V, generator=g) * 4).to(backend[1])
    slot = torch.arange(rows) % (S + 1) - int(rows > 3)  # some rows have no slot
    length = torch.randint(0, L + 1, (rows,), generator=g)
    got = op("shape_logits", backend, logits.to(backend[0]), slot.int().to(backend[0]), length.int().to(backend[0]),
             *[x.to(backend[0]) for x in r])
    assert got.dtype == torch.float32
    for i in range(rows):
        s = int(slot[i])
        ref = want(logits[i], s, int(length[i]), r, allowed) if 0 <= s < S else logits[i].double()
        same(got[i], ref)
    # the kernels round as the reference does
    cpu = OPS["shape_logits"].impl(logits, slot.int(), length.int(), *r)
    if K < 3:  # sums of biases may be taken in another order
        assert torch.equal(got.cpu(), cpu)


@pytest.mark.parametrize("S,V,L,K,valid", [(1, 7, 1, 1, 7), (4, 130, 20, 6, 129), (6, 5003, 100, 10, 5003), (3, 50400, 900, 64, 50257),
                                           (70, 1000, 12, 0, 1000)])
def test_choice_from_shaped_logits(backend, S, V, L, K, valid):  # noqa: F811
    dev = backend[0]
    r, allowed = rules(S, V, L, K, seed=3)
    g = torch.Generator().manual_seed(6)
    # few distinct values: ties, of which the lowest index wins; beyond `valid` there is nothing to choose
    logits = torch.randint(-6, 7, (S, V), generator=g).to(backend[1])
    logits[:, valid:] = 1000.0
    length = torch.randint(0, L, (S,), generator=g)
    length[-1] = L  # a full history: the choice has no place in it
    count = torch.ones(S, dtype=torch.int32)
    if S > 3:
        count[3] = 0
    d = [x.to(dev) for x in r]
    current, buf, pos = torch.full((S,), -7, dtype=torch.int32, device=dev), torch.full((3, S), -7, dtype=torch.int32, device=dev), i32(backend, 5)
    op("take_shaped_", backend, current, logits.to(dev), buf, pos, length.int().to(dev), count.to(dev), *d, valid=valid, base=5, ahead=1,
       advance=True)
    ref = OPS["shape_logits"].impl(logits[:, :valid], torch.arange(S, dtype=torch.int32), length.int(), *r)
    token = [int((x == x.max()).int().argmax()) for x in ref]
    history = r[0].clone()
    for s in range(S):
        if count[s] > 0:
            same(ref[s], want(logits[s, :valid], s, int(length[s]), r, allowed[:, :valid]))
            if length[s] < L:
                history[s, length[s]] = token[s]
        else:
            token[s] = -7
    assert current.tolist() == token
    assert buf[1].tolist() == token and (buf[[0, 2]] == -7).all()
    assert torch.equal(d[0].cpu(), history)
    assert pos.tolist() == [6]
    if S > 2:
        assert token[1] == V // 2 and token[2] == 0  # the single token that is allowed; nothing allowed
    # the row is out of range: only the buffer is left alone; the position stays without `advance`
    op("take_shaped_", backend, current, logits.to(dev), buf, pos, length.int().to(dev), count.to(dev), *d, valid=valid, base=0, ahead=0,
       advance=False)
    assert pos.tolist() == [6] and (buf[[0, 2]] == -7).all()


def test_infinite_and_undefined_logits(backend):  # noqa: F811
    """What is not allowed may hold anything; NaN is never chosen; the lowest value of the type is a value like others."""
    V, dev = 40, backend[0]
    r, _ = rules(2, V, 3, 1)
    allowed = torch.ones(2, V, dtype=torch.bool)
    allowed[:, :3] = False
    r[5] = bits_of(allowed)
    r[0][:], r[3][:], r[2][:] = 30, -1, torch.tensor([1.5, 0.0, 0.0])
    logits = torch.full((2, V), torch.finfo(backend[1]).min).to(backend[1])
    logits[:, 0], logits[:, 1], logits[:, 2], logits[0, 5], logits[0, 6] = math.nan, math.inf, 3.0, math.nan, 1.0
    logits[1, 7] = -math.inf
    d = [x.to(dev) for x in r]
    got = op("shape_logits", backend, logits.to(dev), i32(backend, 0, 1), i32(backend, 1, 1), *d).cpu()
    assert (got[:, :3] == -math.inf).all() and math.isnan(got[0, 5]) and got[0, 6] == 1.0 and got[1, 7] == -math.inf
    assert got[0, 4] == float(logits[0, 4]) and got[0, 30] == -math.inf  # seen: 1.5 times as low, below what 32 bits hold
    current, buf = i32(backend, -7, -7), torch.zeros(1, 2, dtype=torch.int32, device=dev)
    op("take_shaped_", backend, current, logits.to(dev), buf, i32(backend, 0), i32(backend, 1, 1), i32(backend, 1, 1), *d, valid=V, base=0,
       ahead=0, advance=False)
    assert current.tolist() == [6, 3]


@pytest.mark.parametrize("offset", [0, 1])
def test_logits_inside_wider_rows(backend, offset):  # noqa: F811
    """A slice of a padded vocabulary, and two rows under the rules of one slot."""
    r, _ = rules(2, 77, 9, 3)
    wide, _ = rnd(backend, 3, 90, seed=8)
    d = [x.to(backend[0]) for x in r]
    got = op("shape_logits", backend, wide[:, offset:offset + 77], i32(backend, 1, 1, 0), i32(backend, 9, 4, 9), *d)
    alone = [op("shape_logits", backend, wide[i:i + 1, offset:offset + 77].contiguous(), i32(backend, s), i32(backend, n), *d)
             for i, (s, n) in enumerate(((1, 9), (1, 4), (0, 9)))]
    assert torch.equal(got, torch.cat(alone))


def test_append_tokens(backend):  # noqa: F811
    dev, T = backend[0], 5
    history = torch.full((4, 8), -1, dtype=torch.int32, device=dev)
    tokens = torch.arange(20, dtype=torch.int32, device=dev)
    op("append_tokens_", backend, history, tokens, i32(backend, 0, 6, 2, 3), i32(backend, 5, 5, 0, 2), T=T)
    assert history.tolist() == [[0, 1, 2, 3, 4, -1, -1, -1], [-1] * 6 + [5, 6], [-1] * 8, [-1] * 3 + [15, 16] + [-1] * 3]


def test_refusals():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def rules_of(slots=2, words=2, biases=(2, 3)):
            return ops.LogitRules(var((slots, 9)), var((slots,)), var((slots, 3), xl.float32), var(biases), var((slots, 3), xl.float32),
                                  var((slots, words)))

        logits = var((2, 50), xl.float32)
        ops.shape_logits(logits, var((2,)), var((2,)), rules_of())
        for bad in (rules_of(words=1), rules_of(biases=(2, 4))):
            with pytest.raises(ValueError, match="rules"):
                ops.shape_logits(logits, var((2,)), var((2,)), bad)
        with pytest.raises(ValueError, match="slots and lengths"):
            ops.shape_logits(logits, var((3,)), var((2,)), rules_of())
        with pytest.raises(ValueError, match="slots, lengths and counts"):
            ops.take_shaped_(var((2,)), logits, var((4, 2)), var((1,)), var((2,)), var((2,)), rules_of(slots=3, biases=(3, 3)))
        with pytest.raises(ValueError, match="slots, lengths and counts"):
            ops.take_shaped_(var((2,)), logits, var((4, 2)), var((1,)), var((1,)), var((2,)), rules_of())
        with pytest.raises(ValueError, match="choices go to"):
            ops.take_shaped_(var((2,)), logits, var((4, 3)), var((1,)), var((2,)), var((2,)), rules_of())
        with pytest.raises(ValueError, match="among 51"):
            ops.take_shaped_(var((2,)), logits, var((4, 2)), var((1,)), var((2,)), var((2,)), rules_of(), valid=51)
        with pytest.raises(ValueError, match="rules.penalties"):
            ops.shape_logits(logits, var((2,)), var((2,)), rules_of()._replace(penalties=var((2, 3))))
        for bad in ((var((4, 6)), var((9,)), 2), (var((2, 6)), var((2, 2)), 2)):
            with pytest.raises(ValueError, match="portions|pos"):
                ops.append_tokens_(bad[0], var((4,)), bad[1], var((2,)), bad[2])
