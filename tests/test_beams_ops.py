"""The ops of sequences with a common beginning one by one against plain float64 oracles: attention over shared prefixes, selection of
beams, reordering of their states. CPU backend, and marked `gpu` the kernels in every type."""
import math

import pytest
import torch

import plain_beams as plain
from test_dunelix_ops import i32, op, rnd
from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops

BACKENDS = [("cpu", torch.float32)] + [pytest.param(("cuda", t), marks=pytest.mark.gpu) for t in (torch.float32, torch.bfloat16, torch.float16)]
NAN = float("nan")


@pytest.fixture(params=BACKENDS, ids=lambda b: f"{b[0]}-{str(b[1])[6:]}")
def backend(request):
    return request.param


# ---- attention ------------------------------------------------------------------------------------------------------

# heads, key / value heads, dim, vdim
SHAPES = {"grouped": (4, 2, 16, 24), "wide": (20, 1, 64, 32), "plain": (3, 3, 32, 16), "odd": (2, 1, 10, 7), "full": (8, 2, 128, 128),
          "long": (1, 1, 200, 264), "three": (6, 2, 96, 80), "twelve": (12, 1, 128, 64), "forty": (4, 2, 40, 24)}
# window, kept first tokens, sink, gate
MASKS = {"all": (0, 0, None, True), "window": (70, 4, 0.0, True), "narrow": (3, 1, 0.5, False), "kept": (40, 90, 0.0, True), "bare": (0, 0, None, False)}
# by sequence: lead, shared, position, tokens of the portion (up to T)
GROUPS = {
    # four beams of one prompt, the first holds it
    "beams": ([0, 0, 0, 0], [150] * 4, [163] * 4, [9] * 4),
    # two groups, a prefix that ends inside a tile, members that left it earlier, the last slot of the cache as a lead
    "ragged": ([5, 0, 5, 0, 0, 5], [130, 61, 17, 129, 61, 130], [133, 61, 190, 140, 75, 131], [1, 5, 9, 2, 9, 4]),
    # whatever the numbers say: leads that are not there, more shared than either holds, negative, a lead without positions
    "odd": ([7, -1, 1, 1, 3, 2], [50, 50, 1 << 30, -5, 64, 1000], [60, 64, 129, 70, 200, 0], [3, 1, 2, 9, 9, 6]),
    # idle sequences among them, a lead that only holds, one that would not fit
    "idle": ([1, 1, 1, 1, 4, 0], [128] * 6, [140, 128, 250, 131, 3, 260], [9, 0, 9, 1, 9, 9]),
    # nothing before the portion, one position shared, one key in all
    "first": ([0, 0, 0], [1, 1, 1], [0, 1, 2], [1, 1, 9]),
    # each its own lead
    "alone": ([0, 1], [100, 64], [129, 64], [9, 3])}
ROOM = 262


def bound(backend):
    """Largest difference over the largest output. 32 bits: scores of up to 10 from sums of `dim` roundings of 2^-24 relative to |q||k|,
    about 2^-18 of a weight, and as much again for sums over keys: 2e-5. 16 bits: the rounding of the output, half a step or eps / 2 of the
    value; queries and weights enter as two numbers of 16 bits each or in 32, which loses 2^-16 of a score and of a weight, 2^-12 of the
    result at most: eps / 16 of bf16, and of fp16, whose products are in 32 bits, less."""
    eps = torch.finfo(backend[1]).eps
    return 2e-5 if backend[1] == torch.float32 else 0.5625 * eps


def attention_case(backend, shape, mask, group, T, seed=0, wide=0):
    """Arguments for the op and what it should leave: junk wherever nobody may look."""
    H, G, d, dv = SHAPES[shape]
    window, keep, sink, gated = MASKS[mask]
    lead, shared, pos, count = GROUPS[group]
    B, dev, dt = len(lead), backend[0], backend[1]
    count = [min(n, T) for n in count]
    cols = (H + G) * d + G * dv + gated * H * dv
    proj, proj64 = rnd(backend, B * T, cols + wide, seed=seed)
    f32 = (dev, torch.float32)
    (wq, _), (wk, _) = rnd(f32, d, std=0.3, seed=21), rnd(f32, d, std=0.3, seed=22)
    wq, wk = wq + 1.5, wk + 1.2
    cache, cache64 = zip(*(rnd(backend, B, G, ROOM, w, seed=seed + 3 + i) for i, w in enumerate((d, dv))))
    held = [max(p, 0) for p in pos]
    for c, c64 in zip(cache, cache64):
        for b in range(B):  # beyond what a slot holds anything may lie
            c[b, :, held[b]:] = NAN
            c64[b, :, held[b]:] = NAN
    joint = torch.full((B * T, H * dv + 5), -7.0, dtype=dt, device=dev)
    args = [proj[:, :cols], wq, wk, *cache, i32(backend, *pos), i32(backend, *count), i32(backend, *lead), i32(backend, *shared), joint]
    kw = dict(T=T, heads=H, window=window, keep_first=keep, scale=d ** -0.5, sink=sink, eps=1e-5)
    after = [c.clone() for c in cache64]
    want = plain.shared_attention(proj64[:, :cols].reshape(B, T, -1), wq.cpu().double(), wk.cpu().double(), *after, pos, count, lead, shared, T, H,
                                  window, keep, d ** -0.5, sink, 1e-5, dt)
    return args, kw, want, after


def check_attention(backend, args, kw, want, after):
    got = op("window_attention_shared_", backend, *args, **kw)
    B, width, T = args[3].shape[0], kw["heads"] * args[4].shape[-1], kw["T"]
    got = got.reshape(B, T, -1).double().cpu()
    top = max([1e-30] + [w.abs().max().item() for w in want.values()])
    for b in range(B):
        for t in range(T):
            if (b, t) in want:
                assert (got[b, t, :width] - want[b, t]).abs().max().item() <= bound(backend) * top, (b, t)
                assert (got[b, t, width:] == -7).all()
            else:
                assert (got[b, t] == -7).all(), (b, t)
    # norms of keys are taken in 64 bits and rounded once: a border between two numbers within 2^-50 of one does not happen
    for now, ref in zip(args[3:5], after):
        now = now.double().cpu()
        assert (now.isnan() == ref.isnan()).all() and (now.nan_to_num() == ref.nan_to_num()).all()


@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("shape,mask,group", [(s, m, g) for i, s in enumerate(SHAPES) for j, m in enumerate(MASKS) for k, g in enumerate(GROUPS)
                                              if (i + 2 * j + 3 * k) % 5 < (3 if s in ("full", "three") else 1)])
def test_attention_over_shared_prefixes(backend, shape, mask, group, T):
    check_attention(backend, *attention_case(backend, shape, mask, group, T))


@pytest.mark.parametrize("T", [1, 9])
def test_attention_of_strided_projections(backend, T):
    """Rows of a wider product, off every boundary that wide loads ask for."""
    for wide in (1, 8):
        check_attention(backend, *attention_case(backend, "full", "window", "ragged", T, wide=wide))


@pytest.mark.parametrize("T", [1, 9])
def test_attention_where_nothing_is_shared_is_the_plain_one(backend, T):
    """The results of `window_attention_`, which rounds its queries and may round a key to the other side: eps / 2 of each of `dim` terms of a
    score, independent ones, 0.02 of a weight at most in bf16."""
    args, kw, _, _ = attention_case(backend, "full", "window", "alone", T)
    other = [a.clone() for a in args]
    got = op("window_attention_shared_", backend, *args, **kw).double()
    ref = op("window_attention_", backend, *other[:7], other[9], **kw).double()
    live = ref != -7
    assert torch.equal(live, got != -7)
    assert (got - ref)[live].abs().max() <= (2e-5 if backend[1] == torch.float32 else 3 * torch.finfo(backend[1]).eps) * ref[live].abs().max()


@pytest.mark.parametrize("T", [1, 9])
def test_what_is_not_finite_reaches_those_who_see_it(backend, T):
    """A value and a key of a prefix that are not finite: sequences that share them, and nobody else; a sequence that left the prefix before
    them neither. What a lead holds behind the prefix reaches none of those that share it."""
    for what in (NAN, math.inf):
        args, kw, want, _ = attention_case(backend, "full", "all", "ragged", T)
        k, v, count, heads = args[3], args[4], args[6].tolist(), kw["heads"]
        v[0, 0, 100, 3] = what  # of those behind lead 0 only sequence 3 shares 100 positions or more; sequence 0 itself shares 130 of lead 5
        k[5, 1, 40, 2] = what   # behind lead 5: sequences 0 and 5; sequence 2 shares 17 positions
        touched = {3: (0, heads // 2), 0: (heads // 2, heads), 5: (heads // 2, heads)}
        got = op("window_attention_shared_", backend, *args, **kw).reshape(6, T, -1)[..., :heads * v.shape[-1]].reshape(6, T, heads, -1).double().cpu()
        top = max(w.abs().max().item() for w in want.values())
        for (b, t), w in want.items():
            lo, hi = touched.get(b, (0, 0))
            w = w.reshape(heads, -1)
            for h in range(heads):
                if not lo <= h < hi:
                    assert (got[b, t, h] - w[h]).abs().max().item() <= bound(backend) * top, (b, t, h)
                elif b == 3:
                    assert not torch.isfinite(got[b, t, h, 3])
                elif what != what:  # (an infinite key may come to a score of minus infinity)
                    assert not torch.isfinite(got[b, t, h]).any()


def test_refusals_of_attention():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.float32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def call(B=3, T=1, H=4, G=2, d=16, v=24, smax=30, cols=None, dt=xl.float32, places=None, joint=None, norm=None, vcache=None, **kw):
            cols = cols or (H + G) * d + (G + H) * v
            i = places or [var((B,), xl.int32) for _ in range(4)]
            return ops.window_attention_shared_(var((B * T, cols), dt), norm or var((d,)), var((d,)), var((B, G, smax, d), dt),
                                                vcache or var((B, G, smax, v), dt), *i, joint or var((B * T, H * v), dt), **{"T": T, "heads": H, "scale": 0.5, **kw})

        call()
        call(T=3, window=4, keep_first=2, sink=0.0, dt=xl.bfloat16)
        call(joint=var((3, 4 * 24 + 7)))
        for bad in (dict(cols=100), dict(heads=3), dict(scale=0.0), dict(window=-1), dict(keep_first=-1), dict(joint=var((3, 90))), dict(joint=var((2, 96))),
                    dict(norm=var((15,))), dict(norm=var((16,), xl.bfloat16)), dict(vcache=var((3, 2, 29, 24))), dict(vcache=var((3, 2, 30, 24), xl.bfloat16)),
                    dict(places=[var((3,), xl.int32)] * 3 + [var((2,), xl.int32)]), dict(places=[var((3,))] * 4), dict(d=520), dict(v=520), dict(T=0),
                    dict(joint=var((3, 96), xl.bfloat16))):
            with pytest.raises(ValueError):
                call(**bad)
        with pytest.raises(ValueError, match="one tensor"):
            cache = var((3, 2, 30, 16))
            ops.window_attention_shared_(var((3, 160)), var((16,)), var((16,)), cache, cache, *(var((3,), xl.int32) for _ in range(4)), var((3, 64)), 1, 4, 0.5)



def test_one_device_per_call():
    from popxl_addons_b200.ops.native_beams import _on_their_device
    call = _on_their_device(lambda *a: len(a))
    assert call(torch.zeros(1), 2, torch.zeros(1)) == 3
    with pytest.raises(ValueError, match="lie on"):
        call(torch.zeros(1), torch.zeros(1, device="meta"))


# ---- selection ------------------------------------------------------------------------------------------------------


def beams_case(backend, groups, K, V, valid, seed=0, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    n = groups * K
    logits = torch.randn(n, V, generator=g) * 3
    if kind == "ties":  # few distinct values
        logits = torch.randint(-3, 4, (n, V), generator=g).float()
    logits[:, valid:] = 1000.0
    scores = -torch.rand(n, generator=g) * 20
    ended = (torch.rand(n, generator=g) < 0.2).int()
    length = torch.randint(0, 30, (n,), generator=g).int()
    if n > 2:
        scores[n // 2] = -math.inf
    return logits.to(backend[1]), scores, ended, length


def check_beams(backend, logits, scores, ended, length, K, end, valid, penalty, in_place=False, strided=False):
    dev, n = backend[0], logits.shape[0]
    given = [scores, ended, length]
    state = [x.clone().to(dev) for x in given]
    into = [] if in_place else [torch.full_like(x, -9) for x in state]
    current, parent = i32(backend, *[-7] * n), i32(backend, *[-7] * n)
    buf, parents = torch.full((3, n), -7, dtype=torch.int32, device=dev), torch.full((3, n), -7, dtype=torch.int32, device=dev)
    step = i32(backend, 5)
    rows = logits.to(dev)
    if strided:  # a slice of wider rows, off a 16-byte boundary
        rows = torch.cat((torch.full((n, 3), 99.0), logits.float().cpu(), torch.full((n, 2), 99.0)), 1).to(logits.dtype).to(dev)[:, 3:-2]
    op("take_beams_", backend, current, parent, rows, buf, parents, step, *state, *into, beams=K, end=-1 if end is None else end, valid=valid,
       length_penalty=penalty, base=5, ahead=1, advance=True)
    assert step.tolist() == [6] and (buf[[0, 2]] == -7).all() and (parents[[0, 2]] == -7).all()
    out = into or state
    if into:
        assert all(torch.equal(a.cpu().nan_to_num(), b.nan_to_num()) for a, b in zip(state, given))
    for g in range(n // K):
        mine = slice(g * K, (g + 1) * K)
        want = plain.next_beams(logits[mine], scores[mine].tolist(), ended[mine].tolist(), length[mine].tolist(), K, end, valid, penalty)
        got = [t[mine].tolist() for t in (parent, current, *out)]
        if want is None:
            assert got[0] == got[1] == [-7] * K
            if into:
                assert all(x == [-9] * K for x in got[2:])
            continue
        assert got[0] == [g * K + w[1] for w in want] and got[1] == [w[2] for w in want]
        assert buf[1, mine].tolist() == got[1] and parents[1, mine].tolist() == got[0]
        assert got[3] == [w[4] for w in want] and got[4] == [w[5] for w in want]
        for x, w in zip(got[2], want):  # half a step of the sum in 32 bits, and 2^-21 for the sum over the row
            assert x == w[3] or abs(x - w[3]) <= 2.0 ** -24 * abs(w[3]) + 2.0 ** -21, (x, w[3])


@pytest.mark.parametrize("groups,K,V,valid", [(1, 1, 7, 7), (1, 4, 3, 3), (3, 2, 130, 129), (2, 5, 1021, 1000), (1, 32, 5003, 5003), (2, 24, 40, 33), (7, 8, 4097, 4097),
                                              (2, 3, 50257, 50257), (1, 4, 130001, 130000), (40, 4, 9000, 9000)])
@pytest.mark.parametrize("kind", ["normal", "ties"])
def test_choice_of_beams(backend, groups, K, V, valid, kind):
    if backend[0] == "cpu" and groups > 7:
        pytest.skip("covered by the smaller ones")
    for seed, (end, penalty, in_place) in enumerate(((2, 0.0, False), (None, 0.0, True), (0, 0.7, True), (1, -1.0, False))):
        check_beams(backend, *beams_case(backend, groups, K, V, valid, seed, kind), K, end, valid, penalty, in_place)


def test_choice_from_rows_of_wider_ones(backend):
    check_beams(backend, *beams_case(backend, 2, 4, 999, 990, 5), 4, 2, 990, 0.5, strided=True)


def test_choice_where_rows_are_equal_or_sorted(backend):
    """Every entry of a row is worth the same, or each is worth more than those before: the parts' lists are longer than what they keep."""
    V, K = 20011, 6
    logits, scores, ended, length = beams_case(backend, 2, K, V, V)
    scores[:], ended[:], length[:] = -1.5, 0, 3
    logits[:] = 0.25  # all beams and all tokens alike: the first beam's first tokens
    check_beams(backend, logits, scores, ended, length, K, None, V, 0.0)
    logits[:] = torch.arange(V, dtype=torch.float32) * 2.0 ** -10
    scores -= torch.arange(2 * K) * 0.125
    check_beams(backend, logits, scores, ended, length, K, None, V, 1.0)
    check_beams(backend, logits.flip(1), scores, ended, length, K, None, V, 0.0)


def test_choice_with_masks_and_undefined_logits(backend):
    """Masked by minus infinity and by the type's lowest value, NaN, a row with plus infinity, rows where nothing or too little is left."""
    V, K = 5000, 4
    logits, scores, ended, length = beams_case(backend, 6, K, V, V)
    scores[:] = -torch.rand(len(scores), generator=torch.Generator().manual_seed(9))
    ended[:] = 0
    lowest = torch.finfo(backend[1]).min
    logits[:4, 5:] = -math.inf                       # group 0: five tokens each
    logits[4:8] = -math.inf                          # group 1: one token of one beam, others follow at minus infinity
    logits[6, 4321] = 1.0
    logits[8:12, 100:] = lowest                      # group 2: the lowest value counts like any other
    logits[8:10] = lowest
    logits[12:16, ::2] = NAN                         # group 3
    logits[16, 77] = math.inf                        # group 4: a row whose probabilities are not defined
    logits[20:24] = NAN                              # group 5: nothing at all
    scores[16 + 3], scores[17] = NAN, math.inf       # no beams there
    check_beams(backend, logits, scores, ended, length, K, 3, V, 0.0)
    ended[4:8] = 1
    check_beams(backend, logits, scores, ended, length, K, 3, V, 0.6, in_place=True)
    scores[8:12] = -math.inf                         # a group without beams is left as it is
    check_beams(backend, logits, scores, ended, length, K, 3, V, 0.0)


def test_rows_that_do_not_count_are_not_read(backend):
    """NaN in the rows of ended beams and of slots without one, which would spread through sums."""
    logits, scores, ended, length = beams_case(backend, 2, 4, 300, 300)
    scores[1:4], ended[:] = -math.inf, 0
    ended[4:6] = 1
    logits[1:6] = NAN
    check_beams(backend, logits, scores, ended, length, 4, 7, 300, 0.0)


def test_sums_of_close_beams_are_compared_in_64_bits(backend):
    """Two beams whose best sums differ by less than a step of the sums in 32 bits: the better one is first."""
    V = 64
    logits = torch.full((2, V), -30.0)
    logits[:, 5] = 0.0
    logits[1, 9] = -17.0  # 4e-8 less for its best token: a step of 100 in 32 bits is 8e-6
    for order in ((0, 1), (1, 0)):
        x = logits[list(order)].to(backend[1])
        check_beams(backend, x, torch.tensor([-100.0, -100.0]), torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), 2, None, V, 0.0)


def test_choice_out_of_the_buffers_range(backend):
    logits, scores, ended, length = (x.to(backend[0]) for x in beams_case(backend, 1, 2, 50, 50))
    buf, step = torch.full((3, 2), -7, dtype=torch.int32, device=backend[0]), i32(backend, 4)
    current, parent = i32(backend, 0, 0), i32(backend, 0, 0)
    for base, ahead in ((0, 0), (5, 0), (0, -5)):
        op("take_beams_", backend, current, parent, logits, buf, buf.clone(), step, scores.clone(), ended, length, beams=2, end=-1, valid=50, length_penalty=0.0,
           base=base, ahead=ahead, advance=False)
        assert (buf == -7).all() and step.tolist() == [4]


def test_refusals_of_choices():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def state(n=8, dts=(xl.float32, xl.int32, xl.int32)):
            return ops.BeamState(*(var((n,), dt) for dt in dts))

        def call(logits=None, current=None, parent=None, buf=None, parents=None, step=None, s=None, beams=4, **kw):
            return ops.take_beams_(current or var((8,)), parent or var((8,)), logits or var((8, 50), xl.float32), buf or var((5, 8)), parents or var((5, 8)),
                                   step or var((1,)), s or state(), beams, **kw)

        call()
        call(end=49, valid=50, length_penalty=0.5, into=state())
        for bad in (dict(beams=3), dict(beams=0), dict(beams=33), dict(logits=var((8, 50))), dict(logits=var((8,), xl.float32)), dict(valid=51), dict(end=50),
                    dict(end=-1), dict(end=30, valid=30), dict(current=var((7,))), dict(parent=var((8,), xl.float32)), dict(buf=var((5, 7))), dict(parents=var((4, 8))),
                    dict(step=var((2,))), dict(step=var((1,), xl.float32)), dict(s=state(7)), dict(s=state(dts=(xl.int32,) * 3)), dict(into=state(4)),
                    dict(length_penalty=NAN), dict(length_penalty=1e9)):
            with pytest.raises(ValueError):
                call(**bad)
        one, two = var((8,)), var((5, 8))
        for bad in (dict(current=one, parent=one), dict(buf=two, parents=two), dict(s=ops.BeamState(var((8,), xl.float32), one, one))):
            with pytest.raises(ValueError, match="of their own"):
                call(**bad)


# ---- reordering -----------------------------------------------------------------------------------------------------

PARENTS = {"stay": [0, 1, 2, 3, 4, 5], "one": [1, 1, 1, 4, 4, 4], "turn": [1, 2, 0, 4, 3, 5], "mixed": [2, 2, 0, 3, 3, 3],
           "elsewhere": [0, -1, 4, 6, 1 << 30, 3]}
# type, shape behind the rows, axis of positions, positions of an entry
STATES = [(torch.float32, (3, 40, 8), 2, 1), (torch.bfloat16, (2, 2, 40, 24), 3, 1), (torch.float32, (33,), None, 1), (torch.int32, (40,), 1, 1),
          (torch.int8, (2, 5, 8, 3), 2, 8), (torch.float32, (2, 5), 2, 8), (torch.bfloat16, (7, 5), None, 1), (torch.int8, (2, 40, 3), 2, 1),
          (torch.float16, (40, 5), 1, 1), (torch.bfloat16, (40, 2000), 1, 1)]


@pytest.mark.parametrize("name", list(PARENTS))
@pytest.mark.parametrize("K", [3, 6, 2, 1])
def test_states_follow_their_beams(backend, name, K):
    if backend[1] in (torch.bfloat16, torch.float16):
        pytest.skip("states bring their own types")
    dev, parent = backend[0], PARENTS[name]
    begin, end = [0, 3, 17, 8, 40, -4], [40, 30, 17, 9, 50, 21]
    g = torch.Generator().manual_seed(3)
    states = [torch.randint(-100, 100, (6, *s), generator=g).to(dt) for dt, s, _, _ in STATES]
    axes, per = tuple(s[2] for s in STATES), tuple(s[3] for s in STATES)
    moved = [x.clone().to(dev) for x in states]
    op("reorder_", backend, i32(backend, *parent), i32(backend, *begin), i32(backend, *end), *moved, beams=K, axes=axes, per=per)
    for x, y, axis, n in zip(states, moved, axes, per):
        assert torch.equal(y.cpu(), plain.reordered(x, parent, begin, end, K, axis, n)), (x.shape, x.dtype)


@pytest.mark.parametrize("K", [4, 8, 16, 32])
def test_many_large_states_follow_their_beams(backend, K):
    """More states than one launch takes, spans of several CTAs, groups of every size."""
    if backend != ("cuda", torch.bfloat16):
        pytest.skip("one type of state is enough")
    g = torch.Generator().manual_seed(K)
    n = 3 * K
    parent = torch.cat([torch.randint(0, K, (K,), generator=g) + i * K for i in range(3)])
    states = [torch.randn(n, 2, 700, 64, generator=g).bfloat16() for _ in range(3)] + [torch.randn(n, 5 + i, generator=g) for i in range(66)]
    axes = (2,) * 3 + (None,) * 66
    moved = [x.cuda() for x in states]
    begin, end = torch.full((n,), 100), torch.full((n,), 650)
    op("reorder_", backend, parent.int().cuda(), begin.int().cuda(), end.int().cuda(), *moved, beams=K, axes=axes, per=(1,) * 69)
    for x, y, axis in zip(states, moved, axes):
        want = x[parent]
        if axis:
            want = torch.cat((x[:, :, :100], want[:, :, 100:650], x[:, :, 650:]), 2)
        assert torch.equal(y.cpu(), want)


def test_refusals_of_reordering():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        rows = [var((6,)) for _ in range(3)]
        x, y = var((6, 4, 5), xl.float32), var((6, 3), xl.bfloat16)
        ops.reorder_([ops.StateRows(x, 2), ops.StateRows(y)], *rows, 3)
        ops.reorder_([], *rows, 3)
        for states, places, K in (([ops.StateRows(x)], rows, 4), ([ops.StateRows(x)], rows, 0), ([ops.StateRows(x)], rows, 33), ([ops.StateRows(x, 0)], rows, 3),
                                  ([ops.StateRows(x, 3)], rows, 3), ([ops.StateRows(x, 1, 0)], rows, 3), ([ops.StateRows(var((5, 4)))], rows, 3),
                                  ([ops.StateRows(x), ops.StateRows(x)], rows, 3), ([ops.StateRows(rows[0])], rows, 3), ([ops.StateRows(x)], rows[:2] + [var((5,))], 3),
                                  ([ops.StateRows(x)], rows[:2] + [var((6,), xl.float32)], 3), ([ops.StateRows(var((6, 0)))], rows, 3)):
            with pytest.raises(ValueError):
                ops.reorder_(states, *places, K)
