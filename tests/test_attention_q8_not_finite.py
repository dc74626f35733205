"""Attention over an 8-bit cache when a key or a value is not finite: the block's scale is NaN and its codes are zero, whatever kernel
completes it; positions that read the block are not finite, and all others are as if nothing had happened. CPU backend, and marked
`gpu` the kernels (32-bit and bf16): single tokens, few rows, portions on the tensor cores, and the general kernel."""
import math

import pytest
import torch

from popxl_addons_b200.xl.opdef import OPS
from test_attention_q8_ops import BLOCK, bound, empty_cache, norms
from test_dunelix_ops import backend, i32, op  # noqa: F401  (fixture and helpers)

# heads, key / value heads, dim, vdim: mma.sync and tensor cores, tensor cores alone (and CUDA cores in 32 bits), CUDA cores
SHAPES = {"full": (8, 2, 128, 128), "eights": (4, 2, 40, 24), "one": (2, 2, 64, 128), "odd": (4, 2, 10, 7)}
CUTS = {"ones": [1] * 6, "few": [3, 2, 4], "blocks": [30, 150, 30], "long": [300]}


def run(backend, rows, cuts, start, shape, window, keep, cache):  # noqa: F811
    """Portions of one sequence, one after another, beside an idle one."""
    H, G, d, dv = shape
    (qn, _), (kn, _) = norms(backend, d)
    outs, p = [], start
    for n in cuts:
        proj = torch.zeros(2, n, rows.shape[1], dtype=backend[1])
        proj[0] = rows[p:p + n]
        joint = torch.zeros(2 * n, H * dv, dtype=backend[1], device=backend[0])
        op("window_attention_q8_", backend, proj.reshape(2 * n, -1).to(backend[0]), qn, kn, *cache, i32(backend, p, 0), i32(backend, n, 0), joint, T=n,
           heads=H, window=window, keep_first=keep, scale=d ** -0.5, sink=0.0, eps=1e-5)
        outs.append(joint[:n].cpu())
        p += n
    return torch.cat(outs).reshape(p - start, H, dv).double()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["key", "value"])
@pytest.mark.parametrize("shape,cut,window", [("full", "ones", 0), ("full", "ones", 40), ("full", "few", 40), ("full", "blocks", 0), ("full", "long", 50),
                                              ("eights", "few", 40), ("eights", "long", 50), ("one", "few", 2), ("one", "long", 2), ("one", "blocks", 40), ("odd", "ones", 40),
                                              ("odd", "blocks", 50)])
def test_one_number_that_is_not_finite(backend, kind, value, shape, cut, window):  # noqa: F811
    """Of the second key head, in the first block or in one between others of the same portion. The history in front of the portions is one portion."""
    H, G, d, dv = SHAPES[shape]
    cuts, R, blocks = CUTS[cut], H // G, 8
    start = 61 if cut in ("ones", "few") else 0
    n, at = start + sum(cuts), 62 if start else 170
    clean = torch.randn(n + 70, (H + G) * d + (G + H) * dv, generator=torch.Generator().manual_seed(3)).to(backend[1])
    rows = clean.clone()
    feature = 5
    rows[at, (H + 1) * d + 2 if kind == "key" else (H + G) * d + dv + feature] = value
    keep = 3 if window == 40 else 0
    edges = [0] + [start] * bool(start) + [start + sum(cuts[:k + 1]) for k in range(len(cuts))]
    brings = max(e for e in edges if e <= at)  # first position of the portion that brings the token
    got, caches = {}, {}
    for name, x in (("clean", clean), ("spoiled", rows)):
        cache = caches[name] = [t.nan_to_num(1.0) for t in empty_cache(backend, 2, G, blocks, d, dv)]
        parts = ([run(backend, x, [start], 0, SHAPES[shape], window, keep, cache)] if start else []) + [run(backend, x, cuts, start, SHAPES[shape], window, keep, cache)]
        parts += [run(backend, x, [1, 3, 66], n, SHAPES[shape], window, keep, cache)]  # later positions, by every kind of kernel
        got[name] = torch.cat(parts)
    block = at // BLOCK
    for i in range(n + 70):
        seen = [j for j in range(i + 1) if not window or i - j < window or j < keep]
        reads = any(j // BLOCK == block for j in seen)  # as codes, or raw
        own = i // BLOCK == block
        x, want = got["spoiled"][i], got["clean"][i]
        assert torch.isfinite(want).all()
        assert torch.equal(x[:R], want[:R]), i  # heads of the other key head
        x, want = x[R:], want[R:]
        if not reads or i < min(brings, at):
            # its scale may have been the unit of other weights of the same launch: rounded anew, on either side within `bound`
            assert (x - want).abs().max() <= 2 * bound(backend, d) * want.abs().max(), i
        elif not own:
            assert torch.isnan(x).all(), i
        elif at in seen:
            assert not torch.isfinite(x[:, feature] if kind == "value" else x).any(), i
        # else: a position of the block that does not see the token, in the portion that brings it or later, may be either
    # the cache: the codes of the CPU reference, bit for bit
    ref = [t.cpu() for t in [t.nan_to_num(1.0) for t in empty_cache(("cpu", backend[1]), 2, G, blocks, d, dv)]]
    if backend[0] == "cuda":
        (qn, _), (kn, _) = norms(("cpu", backend[1]), d)
        m = n + 70
        OPS["window_attention_q8_"].impl(torch.cat((rows[:m], torch.zeros_like(rows[:m]))), qn, kn, *ref, i32(("cpu",), 0, 0), i32(("cpu",), m, 0),
                                         torch.zeros(2 * m, H * dv, dtype=backend[1]), T=m, heads=H, window=window, keep_first=keep, scale=d ** -0.5,
                                         sink=0.0, eps=1e-5)
        for a, b in zip(caches["spoiled"][:4], ref[:4]):
            assert torch.equal(a.cpu().nan_to_num(77.0) if a.is_floating_point() else a.cpu(), b.nan_to_num(77.0) if b.is_floating_point() else b)
    which = 2 if kind == "key" else 3
    scales, codes = caches["spoiled"][which][0, :, block].cpu(), caches["spoiled"][which - 2][0, :, block].cpu()
    assert torch.isnan(scales[1]) and torch.isfinite(scales[0]) and not codes[1].any()
    other = caches["spoiled"][5 - which][0, :, block].cpu()
    assert torch.isfinite(other).all() and torch.equal(other, caches["clean"][5 - which][0, :, block].cpu())


@pytest.mark.parametrize("T", [1, 4, 130])
def test_a_query_that_is_not_finite(backend, T):  # noqa: F811
    """Its own head's result is NaN, at every kind of position: right behind a block, in a block, with and without earlier keys."""
    H, G, d, dv = SHAPES["full"]
    for start in (0, 64, 100):
        n = start + T
        rows = torch.randn(n, (H + G) * d + (G + H) * dv, generator=torch.Generator().manual_seed(8)).to(backend[1])
        rows[start, 3 * d + 1] = math.nan
        cache = [t.nan_to_num(1.0) for t in empty_cache(backend, 2, G, 8, d, dv)]
        if start:
            run(backend, rows, [start], 0, SHAPES["full"], 0, 0, cache)
        got = run(backend, rows, [T], start, SHAPES["full"], 0, 0, cache)
        assert torch.isnan(got[0, 3]).all() and torch.isfinite(got[0, [0, 1, 2, 4, 5, 6, 7]]).all() and torch.isfinite(got[1:]).all()
