"""Attention over shared prefixes where a tile, a sum or a mask is at its edge: the kernels against the CPU reference's arithmetic."""
import math

import pytest
import torch

from popxl_addons_b200.xl.opdef import OPS
import popxl_addons_b200.xl.ops  # noqa: F401  (registers the ops)

NAN = float("nan")


def case(dev, dt, B, T, H, G, d, dv, room, pos, count, lead, shared, seed=0, wq=1.5, **kw):
    """Arguments of the op: random projections and caches, one place for all sequences or one each."""
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(dt).to(dev)

    def places(x):
        return (torch.full((B,), x) if isinstance(x, int) else torch.as_tensor(x)).int().to(dev)

    proj = rnd(B * T, (H + G) * d + (G + H) * dv)
    caches = [rnd(B, G, room, w) for w in (d, dv)]
    norms = [torch.full((d,), x, device=dev) for x in (wq, 1.2)]
    joint = torch.full((B * T, H * dv), -7.0, dtype=dt, device=dev)
    args = [proj, *norms, *caches, *map(places, (pos, count, lead, shared)), joint]
    return args, dict(T=T, heads=H, window=0, keep_first=0, scale=d ** -0.5, sink=0.0, eps=1e-6) | kw


def outputs(args, kw):
    """What the kernels leave, and the reference on the same device."""
    from popxl_addons_b200.ops import native

    other = [a.clone() for a in args]
    want = OPS["window_attention_shared_"].impl(*other, **kw)
    got = OPS["window_attention_shared_"].native["cuda"](*args, **kw)
    torch.cuda.synchronize()
    native.check_gemm_errors()
    return got, want


def assert_close(got, want):
    """Both sides round the same sums once, eps / 2 each, and weights and queries of two bf16 numbers lose 2^-12 (32 bits: 2e-5 for each side)."""
    top = want.float()[want != -7].abs().max().item()
    assert torch.isfinite(got).all()
    assert torch.equal(got == -7, want == -7)
    bound = 4e-5 if got.dtype == torch.float32 else 1.0625 * torch.finfo(got.dtype).eps
    assert (got.float() - want.float()).abs().max().item() <= bound * top


@pytest.mark.gpu
@pytest.mark.parametrize("members", [3, 5])
@pytest.mark.parametrize("heads", [16, 31])
def test_large_and_small_tiles_in_turn(members, heads):
    """Groups of several sequences and of one, a block each: tiles that take all of the queries' room and such that take a place of it follow one
    another in one CTA, and some warps have no rows in either."""
    per = members + 1
    B = 448 // per * per
    place = torch.arange(B)
    lead = torch.where(place % per < members, place // per * per, place)
    args, kw = case("cuda", torch.bfloat16, B, 1, heads, 1, 64, 64, 120, 100 + place % 7, 1, lead, 100)
    for _ in range(3):
        assert_close(*outputs([a.clone() for a in args], kw))


# tokens, position, shared, window, kept first ones, and positions (of the lead: 0, or its own: 1) that no row of sequence 1 sees
UNSEEN = {"lead's, portion": (64, 120, 100, 64, 0, [(0, 10), (0, 56)]), "lead's behind kept ones, portion": (40, 120, 100, 64, 7, [(0, 7), (0, 56)]),
          "own, portion": (40, 90, 0, 64, 0, [(1, 3), (1, 26)]), "own behind kept ones, portion": (40, 90, 10, 64, 12, [(1, 12), (1, 26)]),
          "lead's and own, portion": (40, 110, 20, 64, 2, [(0, 3), (1, 21), (1, 46)]), "several blocks, portion": (40, 300, 10, 160, 100, [(1, 100), (1, 140)]),
          "lead's, one token": (1, 120, 100, 64, 3, [(0, 3), (0, 56)]), "own, one token": (1, 100, 0, 64, 0, [(1, 3), (1, 36)]),
          "own behind kept ones, one token": (1, 100, 10, 64, 12, [(1, 12), (1, 36)]), "several blocks, one token": (1, 300, 0, 100, 130, [(1, 130), (1, 200)]),
          "lead's and own, some tokens": (5, 100, 10, 64, 3, [(0, 3), (1, 12), (1, 36)])}


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("junk", [NAN, math.inf])
@pytest.mark.parametrize("name", list(UNSEEN))
def test_values_that_no_row_sees_reach_nobody(dt, junk, name):
    """Not even where leaving their positions out would save no block of keys."""
    T, pos, shared, window, keep, unseen = UNSEEN[name]
    assert all(keep <= p <= pos - window and (p < shared) == (b == 0) for b, p in unseen)
    args, kw = case("cuda", dt, 2, T, 8, 2, 128, 128, 400, pos, T, [7, 0], [0, shared], window=window, keep_first=keep)
    args[6][0] = 0  # the lead only holds its positions
    for b, p in unseen:
        args[4][b, :, p] = junk
        args[3][b, :, p] = NAN
    assert_close(*outputs(args, kw))


BACKENDS = [("cuda", torch.bfloat16, 1), ("cuda", torch.bfloat16, 40), ("cuda", torch.float32, 1), ("cuda", torch.float32, 40), ("cuda", torch.float16, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dev,dt,T", BACKENDS)
@pytest.mark.parametrize("sink", [torch.finfo(torch.float32).min, -1e38, -1e30, 1e38, torch.finfo(torch.float32).max])
def test_sinks_of_any_size(dev, dt, T, sink):
    """A sink far below all scores is none, one far above them leaves nothing of the values; neither overflows where scores are counted in other units."""
    args, kw = case(dev, dt, 3, T, 8, 2, 128, 128, 400, 200, T, 0, 150, sink=sink)
    got, want = outputs(args, kw)
    if sink > 0:
        assert (got == 0).all()
    else:
        assert_close(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dev,dt,T", BACKENDS)
@pytest.mark.parametrize("junk", [NAN, -math.inf])
def test_values_that_are_not_finite_reach_those_who_see_them_with_any_weight(dev, dt, T, junk):
    """Scores of -113 and 113: the first block's weights are zero in 32 bits, and in another part than the others."""
    d, G = 128, 2
    args, kw = case(dev, dt, 2, T, 4, G, d, d, 1200, 1000, T, [7, 0], [0, 960], wq=10.0, scale=d ** -0.5)
    args[0][:, :4 * d] = 1.0
    args[3][:] = 1.0
    args[3][:, :, :128] = -1.0
    args[4][0, 1, 10, 3] = junk
    args[6][0] = 0
    got, want = outputs(args, kw)
    got = got.reshape(2, T, 4, d)[1]
    assert not torch.isfinite(got[:, 2:, 3]).any()
    assert torch.isfinite(got[:, :2]).all()
