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
