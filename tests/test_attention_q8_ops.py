"""Attention against a cache of 8 bits: whole sequences of the plain oracle against the op run in portions that are cut anywhere,
inside blocks, at their ends and across several of them. Codes, scales and tails are compared bit for bit: they depend on nothing but
the tokens. CPU backend, and marked `gpu` the kernels (32-bit and bf16)."""
import pytest
import torch

import plain_serving as plain
from test_dunelix_ops import backend, close, i32, op, rnd  # noqa: F401  (fixture and helpers)
from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from popxl_addons_b200.xl.opdef import OPS

BLOCK = plain.BLOCK
# heads, key / value heads, dim, vdim
SHAPES = {"grouped": (4, 2, 16, 24), "wide": (20, 1, 64, 32), "plain": (3, 3, 32, 16), "odd": (2, 1, 10, 7), "full": (8, 2, 128, 128),
          "long": (1, 1, 200, 264), "group_of_three": (6, 2, 96, 80)}


def empty_cache(backend, B, G, blocks, dim, vdim, junk=True):  # noqa: F811
    """What an earlier request may have left: anything finite in the codes, anything at all in the tails."""
    g = torch.Generator().manual_seed(99)
    t = [torch.randint(-127, 128, (B, G, blocks, BLOCK, w), generator=g).to(torch.int8) for w in (dim, vdim)]
    t += [torch.rand(B, G, blocks, generator=g) * 100 for _ in range(2)]
    t += [torch.full((B, G, BLOCK, w), float("nan")).to(backend[1]) for w in (dim, vdim)]
    return [x.to(backend[0]) for x in t]


def bound(backend, dim):  # noqa: F811
    """Largest difference over the largest output. 32 bits: scores of up to 8 from sums of `dim` roundings of 2^-24 relative to
    |q||k|, about 2^-18 of a weight, and as much again for sums over keys. bf16: the output's own rounding is 2^-8 of the value at
    most (half a step of 2^-7), a gate's input has none; queries, held to 2^-11 where products take 16 bits, move a score of up to 8 by
    the sum of `dim` independent roundings, about 2^-11 * 8 / sqrt(dim) and 2^-10 at most for widths of 16 and more; weights
    times scales in 16 bits add 2^-11: below 2 * 2^-8 in all."""
    return 2e-5 if backend[1] == torch.float32 else 2 * 2.0 ** -8


def run_portions(backend, rows, cuts, start, T, shape, window, keep, sink, gated, cache, eps=1e-5):  # noqa: F811
    """Portions of `rows (n, columns)` of the middle one of three slots, `cuts` their lengths; the last slot is idle, the first would
    not fit. Returns the outputs and what is left of the other rows."""
    H, G, d, dv = shape
    dev, outs = backend[0], []
    (qn, _), (kn, _) = norms(backend, d)
    p = start
    blocks = cache[0].shape[2]
    for n in cuts:
        T_now = max(T, n) if T else n
        proj = torch.full((3, T_now, rows.shape[1]), 3.0, dtype=backend[1])
        proj[1, :n] = rows[p:p + n]
        joint = torch.full((3 * T_now, H * dv + 5), -7.0, dtype=backend[1], device=dev)
        got = op("window_attention_q8_", backend, proj.reshape(3 * T_now, -1).to(dev), qn, kn, *cache, i32(backend, blocks * BLOCK - n + 1, p, 3),
                 i32(backend, n, n, 0), joint, T=T_now, heads=H, window=window, keep_first=keep, scale=d ** -0.5, sink=sink, eps=eps)
        got = got.reshape(3, T_now, -1)
        assert (got[0] == -7).all() and (got[2] == -7).all() and (got[1, n:] == -7).all() and (got[1, :, H * dv:] == -7).all()
        outs.append(got[1, :n, :H * dv])
        p += n
    return torch.cat(outs)


def norms(backend, d):  # noqa: F811
    f32 = (backend[0], torch.float32)
    (q, q64), (k, k64) = rnd(f32, d, std=0.3, seed=21), rnd(f32, d, std=0.3, seed=22)
    return (q + 1.5, (q.cpu() + 1.5).double()), (k + 1.2, (k.cpu() + 1.2).double())


# portions that are cut inside blocks, at their ends and across several of them
CUTS = {"ones": [1] * 3, "even": [64, 64, 2], "ragged": [5, 59, 1, 63, 64, 65, 1], "two": [200, 1, 1], "edges": [63, 1, 1, 127, 1],
        "whole": [130], "growing": [2, 3, 4, 8, 16, 33, 100, 40]}
# window, kept first tokens, sink, gate
MASKS = {"all": (0, 0, None, True), "window": (70, 4, 0.0, True), "narrow": (3, 1, 0.5, False), "kept": (40, 90, 0.0, True)}
MIXED = [("grouped", c, m) for c in CUTS for m in ("window", "narrow")] + [
    ("full", c, m) for c, m in zip(CUTS, ("all", "window", "kept", "narrow", "all", "window", "kept"))] + [
    ("wide", "growing", "window"), ("wide", "edges", "all"), ("plain", "ragged", "kept"), ("plain", "two", "all"), ("odd", "ragged", "kept"),
    ("odd", "edges", "all"), ("long", "two", "window"), ("long", "edges", "kept"), ("group_of_three", "growing", "all"),
    ("group_of_three", "edges", "narrow")]


@pytest.mark.parametrize("shape,cut,mask", MIXED)
def test_portions_against_whole_sequences(backend, shape, cut, mask):  # noqa: F811
    cuts, (window, keep, sink, gated) = CUTS[cut], MASKS[mask]
    H, G, d, dv = SHAPES[shape]
    eps, n = 1e-5, sum(cuts)
    blocks = n // BLOCK + 1
    cols = (H + G) * d + G * dv + (H * dv if gated else 0)
    rows = torch.randn(n, cols, generator=torch.Generator().manual_seed(1))
    rows[n // 3] *= 30.0  # a token whose block has a scale of its own
    rows = rows.to(backend[1])
    cache = empty_cache(backend, 3, G, blocks, d, dv)
    before = [x.clone() for x in cache]
    got = run_portions(backend, rows, cuts, 0, 0, SHAPES[shape], window, keep, sink, gated, cache, eps)
    (_, qn), (_, kn) = norms(backend, d)
    want, k, v = plain.q8_attention(rows.double(), qn, kn, H, G, d, dv, window, keep, d ** -0.5, sink, eps, backend[1])
    for i in range(n):  # row by row: a single wrong position would drown among larger ones
        close(got[i], want[i], backend, bound(backend, d), bound(backend, d))
    full = n // BLOCK
    for held, scale, tail, x in ((cache[0], cache[2], cache[4], k), (cache[1], cache[3], cache[5], v)):
        for j in range(full):
            for g in range(G):
                codes, step = plain.block_codes(x[j * BLOCK:(j + 1) * BLOCK, g])
                assert torch.equal(held[1, g, j].cpu().double(), codes) and scale[1, g, j].item() == step.item()
        assert torch.equal(tail[1, :, :n % BLOCK].cpu().double(), x[full * BLOCK:].transpose(0, 1))
    for now, was in zip(cache, before):  # the other slots, blocks that are not complete, places of the tail that are not in use
        assert torch.equal(now[[0, 2]].nan_to_num(5.0), was[[0, 2]].nan_to_num(5.0))
    for now, was in zip(cache[:4], before[:4]):
        assert torch.equal(now[:, :, full:], was[:, :, full:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_do_not_depend_on_the_kernel(dtype):
    """Every division of a prompt into portions, and the CPU, come to the same bits of codes, scales and tails."""
    H, G, d, dv = SHAPES["full"]
    rows = (torch.randn(321, (H + G) * d + (G + H) * dv, generator=torch.Generator().manual_seed(4)) * 3).to(dtype)
    held = []
    for dev, cuts in (("cpu", [321]), ("cuda", [321]), ("cuda", [1] * 321), ("cuda", [7, 200, 1, 50, 63])):
        cache = empty_cache((dev, dtype), 3, G, 6, d, dv)
        run_portions((dev, dtype), rows, cuts, 0, 0, SHAPES["full"], 100, 4, 0.0, True, cache)
        held.append([x.cpu()[1] for x in cache])
        held[-1][4], held[-1][5] = (x[:, :321 % BLOCK] for x in held[-1][4:])
    for other in held[1:]:
        assert all(torch.equal(x, y) for x, y in zip(held[0], other))


def test_blocks_of_zeros_and_of_one_large_value(backend):  # noqa: F811
    """A scale of zero, and a value next to which the others vanish: their code is zero."""
    H, G, d, dv = 2, 1, 16, 16
    rows = torch.zeros(70, (H + G) * d + G * dv, dtype=backend[1])
    rows[5, -1], rows[6, -2] = 1e6, 1.0
    rows[:, :H * d] = 1.0
    cache = empty_cache(backend, 3, G, 2, d, dv)
    got = run_portions(backend, rows, [64, 6], 0, 0, (H, G, d, dv), 0, 0, None, False, cache)
    assert cache[2][1, 0, 0] == 0 and (cache[0][1, 0, 0] == 0).all()
    assert cache[1][1, 0, 0].abs().sum() == 127 and cache[1][1, 0, 0, 5, -1] == 127
    close(got[5, dv - 1:dv], torch.tensor([float(rows[5, -1]) / 6]), backend, 1e-5, 2.0 ** -8)      # its own block: as computed
    close(got[69, dv - 2:dv], torch.tensor([0.0, float(rows[5, -1]) / 70]), backend, 1e-5, 2.0 ** -8)


@pytest.mark.parametrize("T", [1, 5, 130])
def test_values_of_very_different_size(backend, T):  # noqa: F811
    """A block with one value of a million, next to blocks of values around 1: what the others add up to keeps its precision."""
    H, G, d, dv = SHAPES["full"]
    n, (qn, qn64), (kn, kn64) = 200 + T, *norms(backend, d)
    g = torch.Generator().manual_seed(6)
    rows = torch.randn(n, (H + G) * d + G * dv, generator=g)
    rows[:, (H + G) * d:] = 0.5 + torch.rand(n, G * dv, generator=g)  # positive: nothing cancels
    rows[10, (H + G) * d], rows[10, (H + G) * d + dv] = 1e6, 1e6
    rows = rows.to(backend[1])
    cache = empty_cache(backend, 3, G, 6, d, dv)
    got = run_portions(backend, rows, [200, T], 0, 0, SHAPES["full"], 0, 0, None, False, cache)
    want, _, _ = plain.q8_attention(rows.double(), qn64, kn64, H, G, d, dv, 0, 0, d ** -0.5, None, 1e-5, backend[1])
    for i in range(200, n):  # value by value; bf16: half a step of the result, and as much again for what `bound` counts
        x, y = (t.reshape(H, dv)[:, 1:].double().cpu() for t in (got[i], want[i]))
        assert ((x - y).abs() / y).max().item() < (5e-5 if backend[1] == torch.float32 else 2 * 2.0 ** -8)


@pytest.mark.parametrize("T", [1, 40])
def test_repeated_passes_and_padding(backend, T):  # noqa: F811
    """The same pass twice gives the same state; padded rows and idle sequences touch nothing."""
    H, G, d, dv = SHAPES["grouped"]
    rows = torch.randn(150, (H + G) * d + (G + H) * dv, generator=torch.Generator().manual_seed(2)).to(backend[1])
    cache = empty_cache(backend, 3, G, 3, d, dv)
    run_portions(backend, rows, [127], 0, 0, SHAPES["grouped"], 30, 2, 0.0, True, cache)
    first = run_portions(backend, rows, [1], 127, T, SHAPES["grouped"], 30, 2, 0.0, True, cache)
    state = [x.clone() for x in cache]
    again = run_portions(backend, rows, [1], 127, T, SHAPES["grouped"], 30, 2, 0.0, True, cache)
    # the block that the first pass completed is whole: the second computes it from the tail, which it left alone
    assert torch.equal(first, again)
    assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(state, cache))


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("T", [1, 20, 130])
def test_projections_inside_wider_rows(backend, T, offset):  # noqa: F811
    """Columns of a wider buffer, whose rows start where 16-byte accesses can and where they cannot."""
    H, G, d, dv = SHAPES["full"]
    cols, n, (qn, qn64), (kn, kn64) = (H + G) * d + (G + H) * dv, 70 + T, *norms(backend, d)
    rows = torch.randn(n, cols, generator=torch.Generator().manual_seed(5)).to(backend[1])
    cache = empty_cache(backend, 1, G, 4, d, dv)
    want, _, _ = plain.q8_attention(rows.double(), qn64, kn64, H, G, d, dv, 100, 4, d ** -0.5, 0.0, 1e-5, backend[1])
    for p, T_now in ((0, 70), (70, T)):
        wide = torch.full((T_now, cols + 8), float("nan"), dtype=backend[1], device=backend[0])
        wide[:, offset:offset + cols] = rows[p:p + T_now].to(backend[0])
        joint = torch.zeros(T_now, H * dv, dtype=backend[1], device=backend[0])
        op("window_attention_q8_", backend, wide[:, offset:offset + cols], qn, kn, *cache, i32(backend, p), i32(backend, T_now), joint, T=T_now,
           heads=H, window=100, keep_first=4, scale=d ** -0.5, sink=0.0, eps=1e-5)
        for i in range(T_now):
            close(joint[i], want[p + i], backend, bound(backend, d), bound(backend, d))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(40))
def test_drawn_calls(seed):
    """Sizes, positions, counts and masks drawn at random, idle and misplaced sequences among them: the kernels against the CPU reference, bit
    for bit in the cache."""
    import random

    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dtype = r.choice([torch.bfloat16] * 4 + [torch.float32, torch.float16])
    d, dv = r.choice([(128, 128), (128, 64), (64, 128), (96, 80), (16, 16), (40, 24), (7, 10), (200, 264)])
    G, R, B, blocks = r.choice([1, 2, 3]), r.choice([1, 3, 4, 8, 20]), r.choice([1, 2, 5]), r.choice([1, 8, 70])
    T = min(r.choice([1, 1, 3, 17, 64, 129, 300]), blocks * BLOCK)
    H, end = G * R, blocks * BLOCK
    count = [r.choice([0, 1, T, T, -1]) for _ in range(B)]
    pos = [r.choice([0, 63, r.randint(0, end), end - max(n, 0), end, -1]) for n in count]
    proj = torch.randn(B * T, (H + G) * d + G * dv + r.choice([0, H * dv]), generator=g).to(dtype)
    cache = [t.nan_to_num(0.5) for t in empty_cache(("cpu", dtype), B, G, blocks, d, dv)]
    cache[2:4] = [t * 3e-4 for t in cache[2:4]]  # keys and values of ordinary size
    qn, kn = norms(("cpu", dtype), d)[0][0], norms(("cpu", dtype), d)[1][0]
    how = dict(T=T, heads=H, window=r.choice([0, 1, 65, 1000]), keep_first=r.choice([0, 4, 64, 300]), scale=d ** -0.5,
               sink=r.choice([None, 0.0]), eps=1e-5)
    held = []
    for backend in (("cpu", dtype), ("cuda", dtype)):  # noqa: F811
        state = [t.clone().to(backend[0]) for t in cache]
        joint = torch.full((B * T, H * dv + 8), -7.0, dtype=dtype, device=backend[0])
        op("window_attention_q8_", backend, proj.to(backend[0]), qn.to(backend[0]), kn.to(backend[0]), *state, i32(backend, *pos), i32(backend, *count),
           joint, **how)
        held.append([joint.cpu()] + [t.cpu() for t in state])
    assert all(torch.equal(x, y) for x, y in zip(held[0][1:], held[1][1:]))
    # both sides are rounded: twice what `bound` allows one of them (fp16: its half step is an eighth of that of bf16)
    tol = 2 * bound(("", dtype), d) / (8 if dtype == torch.float16 else 1)
    for x, y in zip(held[0][0].double(), held[1][0].double()):
        assert (x - y).abs().max() <= tol * x.abs().max()


@pytest.mark.gpu
def test_two_streams():
    """Single tokens whose keys are cut among CTAs, few rows, and portions, side by side on two streams: what each leaves alone."""
    from popxl_addons_b200.ops.native import check_gemm_errors

    backend, (H, G, d, dv) = ("cuda", torch.bfloat16), SHAPES["full"]
    (qn, _), (kn, _) = norms(backend, d)
    runs = []
    for seed, T in ((1, 1), (2, 1), (3, 12), (4, 300)):
        g = torch.Generator(device="cuda").manual_seed(seed)
        cache = [t.nan_to_num(1.0) for t in empty_cache(backend, 2, G, 80, d, dv)]
        proj = torch.randn(2 * T, (H + G) * d + (G + H) * dv, generator=g, device="cuda").bfloat16()
        where = (torch.tensor([4000 + 64 * seed, 700], dtype=torch.int32, device="cuda"), torch.tensor([T, T], dtype=torch.int32, device="cuda"))

        def run(T=T, cache=cache, proj=proj, where=where):
            joint = torch.zeros(2 * T, H * dv, dtype=torch.bfloat16, device="cuda")
            assert OPS["window_attention_q8_"].native["cuda"](proj, qn, kn, *cache, *where, joint, T=T, heads=H, window=0, keep_first=0, scale=d ** -0.5,
                                                              sink=None, eps=1e-5) is joint
            return joint

        runs.append(run)
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(40):  # a cache stays with its stream
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 2, [runs[k]() for k in (i % 2, 2 + i % 2)]))
    torch.cuda.synchronize()
    check_gemm_errors()
    for at, pair in got:
        assert torch.equal(pair[0], want[at]) and torch.equal(pair[1], want[2 + at])


def test_refusals():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def cache(dt=xl.bfloat16, **kw):
            spec = ops.cache8_spec(2, 2, 100, 16, 24, dt)
            t = {k: var(*kw.get(k, s)) for k, s in spec.items()}
            return ops.Cache8(**t)

        f32, i32_ = xl.float32, xl.int32
        proj = var((6, (4 + 2) * 16 + (2 + 4) * 24), xl.bfloat16)
        rest = (var((2,), i32_), var((2,), i32_))
        joint = var((6, 4 * 24), xl.bfloat16)
        norm = var((16,), f32)
        out = ops.window_attention_q8_(proj, norm, norm, cache(), *rest, joint, 3, 4, 0.25)
        assert out.shape == joint.shape
        with pytest.raises(ValueError, match="cache.k_scale"):
            ops.window_attention_q8_(proj, norm, norm, cache(k_scale=((2, 2, 1), f32)), *rest, joint, 3, 4, 0.25)
        with pytest.raises(ValueError, match="cache.v_tail"):
            ops.window_attention_q8_(proj, norm, norm, cache(v_tail=((2, 2, 64, 24), f32)), *rest, joint, 3, 4, 0.25)
        with pytest.raises(ValueError, match="multiple of the cache's"):
            ops.window_attention_q8_(proj, norm, norm, cache(), *rest, joint, 3, 3, 0.25)
        with pytest.raises(ValueError, match="projections"):
            ops.window_attention_q8_(proj, norm, norm, cache(), *rest, joint, 4, 4, 0.25)
        with pytest.raises(ValueError, match="joint buffer"):
            ops.window_attention_q8_(proj, norm, norm, cache(), *rest, var((6, 95), xl.bfloat16), 3, 4, 0.25)
        for bad in ((var((1,), i32_), rest[1]), (rest[0], var((2,), f32))):
            with pytest.raises(ValueError, match="pos|count"):
                ops.window_attention_q8_(proj, norm, norm, cache(), *bad, joint, 3, 4, 0.25)
        with pytest.raises(ValueError, match="q_norm"):
            ops.window_attention_q8_(proj, var((17,), f32), norm, cache(), *rest, joint, 3, 4, 0.25)
        with pytest.raises(ValueError, match="positive"):
            ops.window_attention_q8_(proj, norm, norm, cache(), *rest, joint, 3, 4, 0.0)
