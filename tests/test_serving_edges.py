"""Calls at the edges of the serving ops: shapes that have to be refused because a kernel would read or write past them, and operands that
are allowed but unusual. CPU backend, and marked `gpu` the kernels."""
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from test_dunelix_ops import backend, i32, op  # noqa: F401  (fixture and helpers)
from test_serving_order import OnDevice


def test_shapes_that_do_not_fit_are_refused():
    """No shape may reach a kernel that would read or write outside a tensor: every operand is compared with the others."""
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def rules(**kw):
            shapes = dict(history=((2, 9), xl.int32), start=((2,), xl.int32), penalties=((2, 3), xl.float32), bias_tokens=((2, 4), xl.int32),
                          bias_values=((2, 4), xl.float32), allowed=((2, 2), xl.int32))
            return ops.LogitRules(*(var(*kw.get(k, s)) for k, s in shapes.items()))

        f32, bf16 = xl.float32, xl.bfloat16
        x, y = var((6, 16), f32), var((4, 16), bf16)
        assert ops.residual_rms_(x, y, var((16,), f32)).shape == (4, 16) and ops.residual_rms_(x, y) is None
        for args in ((x, var((4, 8), bf16)), (x, var((4, 24), bf16)), (x, var((7, 16), bf16)), (x, y, var((8,), f32)), (x, y, var((16,), bf16)),
                     (var((6, 16), bf16), y), (x, var((16,), bf16))):
            with pytest.raises(ValueError, match="residual stream|norm"):
                ops.residual_rms_(*args)

        plain, joint = ops.split_glu(var((3, 20), bf16), 8, 5, 7.0)
        assert plain.shape == (3, 8) and joint.shape == (3, 11)
        assert ops.split_glu(var((3, 8), bf16), 8, 5, 7.0)[1].shape == (3, 5)
        for shape, cols, lead in (((3, 21), 8, 5), ((3, 6), 8, 5), ((3, 20), -2, 5), ((3, 20), 8, -1), ((20,), 8, 5)):
            with pytest.raises(ValueError, match="gate and up"):
                ops.split_glu(var(shape, bf16), cols, lead, 7.0)

        logits, slot = var((2, 50), f32), var((2,))
        ops.shape_logits(logits, slot, slot, rules())
        for bad in (dict(bias_tokens=((1, 4), xl.int32)), dict(bias_values=((1, 4), f32)), dict(start=((1,), xl.int32)),
                    dict(allowed=((1, 2), xl.int32)), dict(penalties=((1, 3), f32)), dict(history=((3, 9), xl.int32))):
            with pytest.raises(ValueError, match="rules"):
                ops.shape_logits(logits, slot, slot, rules(**bad))
        for bad in (var((2, 50)), var((50,), f32)):
            with pytest.raises(ValueError, match="logits"):
                ops.shape_logits(bad, slot, slot, rules())
            with pytest.raises(ValueError, match="logits"):
                ops.take_shaped_(var((2,)), bad, var((4, 2)), var((1,)), slot, slot, rules())
        with pytest.raises(ValueError, match="position"):
            ops.take_shaped_(var((2,)), logits, var((4, 2)), var((2,)), slot, slot, rules())

        ops.append_tokens_(var((2, 6)), var((4,)), slot, slot, 2)
        for history, tokens in ((var((2, 6), f32), var((4,))), (var((2, 6)), var((4,), f32))):
            with pytest.raises(ValueError, match="int32"):
                ops.append_tokens_(history, tokens, slot, slot, 2)


@pytest.fixture
def launches(monkeypatch):
    """What the binding of attention over 8-bit codes hands to its kernels, without a GPU: a list of (name, arguments)."""
    from popxl_addons_b200.ops import native_serving as ns

    seen = []
    for name, fake in (("_ok", lambda *t: True), ("_i32", lambda *t: True), ("_stream", lambda: 0), ("_sms", lambda device: 148),
                       ("_count", lambda name: None), ("counters", lambda n, *a: torch.zeros(n, dtype=torch.int32)),
                       ("gemm_error_flag", lambda device: torch.zeros(1, dtype=torch.int32))):
        monkeypatch.setattr(ns, name, fake)
    for name in ("_q8_few", "_q8_append", "_q8_general", "_q8_append_expand", "_q8_tcgen05"):
        monkeypatch.setattr(ns, name, lambda *a, name=name: seen.append((name, a)) or 0)
    return seen


def call_of_attention(B=1, T=1, H=2, G=1, dim=16, vdim=16, blocks=2, dtype=torch.bfloat16, **kw):
    """The binding on tensors of the CPU (see `launches`)."""
    from popxl_addons_b200.ops import native_serving as ns

    cache = [torch.zeros(B, G, blocks, 64, w, dtype=torch.int8) for w in (dim, vdim)] + [torch.zeros(B, G, blocks) for _ in range(2)]
    cache += [torch.zeros(B, G, 64, w, dtype=dtype) for w in (dim, vdim)]
    rows = [torch.zeros(B * T, n, dtype=dtype) for n in ((H + G) * dim + G * vdim, H * vdim)]
    where = [torch.zeros(B, dtype=torch.int32), torch.ones(B, dtype=torch.int32)]
    proj, *cache, pos, count, joint = (t.as_subclass(OnDevice) for t in (rows[0], *cache, *where, rows[1]))
    how = dict(T=T, heads=H, window=0, keep_first=0, scale=0.25, sink=None, eps=1e-6)
    return ns.window_attention_q8_cuda(proj, torch.ones(dim), torch.ones(dim), *cache, pos, count, joint, **{**how, **kw})


@pytest.mark.parametrize("T,dtype,kernel", [(1, torch.bfloat16, "_q8_few"), (3, torch.bfloat16, "_q8_few"), (100, torch.bfloat16, "_q8_append_expand"),
                                            (100, torch.bfloat16, "_q8_tcgen05"), (2, torch.float32, "_q8_general")])
def test_windows_wider_than_an_int(launches, T, dtype, kernel):
    """A window or a number of kept tokens past 2^31 arrives as one that hides nothing, not as its low 32 bits."""
    call_of_attention(T=T, dtype=dtype, window=(1 << 32) + 5, keep_first=(1 << 33) + 1)
    args = dict(launches)[kernel]
    sizes = [a for a in args if isinstance(a, int)]
    assert (1 << 32) + 5 not in sizes and (1 << 33) + 1 not in sizes
    at = max(i for i in range(len(args) - 2) if args[i] == 2 and i > 8)  # blocks, window, keep_first
    assert args[at + 1] >= 128 and args[at + 2] >= 128 and max(args[at + 1:at + 3]) < 1 << 31


def shifted(t, by=1):
    """The same numbers, `by` elements behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    assert flat.data_ptr() % 16 == 0
    flat[by:by + t.numel()] = t.reshape(-1)
    return flat[by:by + t.numel()].view(t.shape)


@pytest.mark.parametrize("T", [1, 5, 130])
@pytest.mark.parametrize("which", ["norms", "tails", "joint"])
def test_operands_off_a_16_byte_boundary(backend, which, T):  # noqa: F811
    """Factors of norms out of a table of odd rows, tails and results inside a larger buffer: taken by the kernels, and with them by a
    captured program, with the results of operands on such a boundary."""
    B, (H, G, d, dv), dev, dt = 2, (8, 2, 64, 64), *backend
    g = torch.Generator().manual_seed(4)
    cache = [torch.randint(-127, 128, (B, G, 4, 64, w), generator=g).to(torch.int8) for w in (d, dv)] + [torch.full((B, G, 4), 0.02) for _ in range(2)]
    cache += [torch.randn(B, G, 64, w, generator=g).to(dt) for w in (d, dv)]
    qn, kn = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    proj, joint = torch.randn(B * T, (H + G) * d + G * dv, generator=g).to(dt).to(dev), torch.zeros(B * T, H * dv + 3, dtype=dt)
    cache, qn, kn, joint = [t.to(dev) for t in cache], qn.to(dev), kn.to(dev), joint.to(dev)
    how = dict(T=T, heads=H, window=0, keep_first=0, scale=d ** -0.5, sink=None, eps=1e-5)
    where = (i32(backend, 100, 40), i32(backend, T, T))
    want_cache = [t.clone() for t in cache]
    want = op("window_attention_q8_", backend, proj, qn, kn, *want_cache, *where, joint.clone(), **how)
    if which == "norms":
        qn, kn = shifted(qn), shifted(kn, 3)
    elif which == "tails":
        cache[4:] = [shifted(t) for t in cache[4:]]
    else:
        joint = shifted(joint)
    got = op("window_attention_q8_", backend, proj, qn, kn, *cache, *where, joint, **how)
    assert all(torch.equal(a, b) for a, b in zip(cache, want_cache))
    # other kernels may take it: each side is off by two half steps of bf16 at most, 2 * 2^-8, and by 2e-5 in 32 bits
    assert (got.double() - want.double()).abs().max() <= (4e-5 if dt == torch.float32 else 4 * 2.0 ** -8) * want.double().abs().max()


def test_copied_factors_are_not_read_ahead(launches, monkeypatch):
    """Factors that had to be copied were written by the launch before."""
    from popxl_addons_b200.ops import native_serving as ns

    monkeypatch.setattr(ns.read_ahead, "allowed", lambda *t: True)
    call_of_attention()
    monkeypatch.setattr(ns, "_rows16", lambda t: t.clone())
    call_of_attention()
    assert [(name, args[-3]) for name, args in launches] == [("_q8_few", 1), ("_q8_few", 0)]


@pytest.mark.parametrize("T", [1, 4, 32])
@pytest.mark.parametrize("dim,vdim,kernels", [(48, 32, {"_q8_few"}), (40, 24, {"_q8_append_expand", "_q8_tcgen05"}),
                                              (48, 24, {"_q8_append_expand", "_q8_tcgen05"}), (40, 21, {"_q8_append", "_q8_general"})])
def test_which_kernel_takes_few_rows(launches, T, dim, vdim, kernels):
    """No size is kept for a kernel that does not take it: features in multiples of 8, but not of 16, go to the tensor cores."""
    call_of_attention(T=T, dim=dim, vdim=vdim)
    assert {name for name, _ in launches} - {"_q8_append"} == kernels - {"_q8_append"}


def terms_that_cancel(dt, rows, K, N, r, seed=0):
    """Whole numbers: `x`, a weight that is minus the adapter's product plus a small matrix, and the adapter; all exact in 16 bits."""
    g = torch.Generator().manual_seed(seed)

    def ints(*shape, most=8):
        return torch.randint(1, most + 1, shape, generator=g) * (torch.randint(0, 2, shape, generator=g) * 2 - 1)

    a, b = torch.zeros(1, r, K, dtype=torch.int64), torch.zeros(1, N, r, dtype=torch.int64)
    a[0, 0], b[0, :, 0] = ints(K), ints(N)
    w = torch.randint(-1, 2, (N, K), generator=g) - b[0] @ a[0]
    x = torch.randn(rows, K, generator=g).to(dt)
    return x, w.to(dt), a.to(dt), b.to(dt)


@pytest.mark.parametrize("N", [128, 264, 131])
@pytest.mark.parametrize("T,r", [(1, 1), (7, 16), (8, 1), (8, 16), (40, 24), (300, 16), (8, 100)])
def test_adapters_that_cancel_the_shared_product(backend, T, r, N):  # noqa: F811
    """The sum of both products is rounded once, whatever they are by themselves, and however a prompt is cut into portions."""
    dev, K, seqs = backend[0], 200, 1 if T == 300 else 140 // T
    for dt in (backend[1],) if backend[1] == torch.float32 else (torch.bfloat16, torch.float16):
        x, w, a, b = (t.to(dev) for t in terms_that_cancel(dt, seqs * T, K, N, r))
        y = op("linear_adapted", backend, x, w, a, b, torch.ones(1, device=dev), i32(backend, *[0] * seqs), T=T, out_dtype=dt)
        term = x.double() @ a[0].double().T @ b[0].double().T
        want = x.double() @ w.double().T + term
        assert term.abs().mean() > 15 * want.abs().mean()
        # half a step of the result; sums of K + r products in 32 bits, 2^-24 each of at most the sum of K absolute terms (some 20 times the
        # largest); the numbers between the products as two of 8 bits or more, 2^-16 of a term
        step = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
        assert ((y.double() - want).abs() <= step * want.abs() + (2.0 ** -15 if dt == torch.bfloat16 else 2.0 ** -18) * term.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 8, 64])
def test_fp16_adapters_whose_product_alone_is_past_its_range(T):
    """70000 and -60000 are 10000, although fp16 ends at 65504."""
    K, N, seqs, dt = 16, 256, 140 // T, torch.float16
    x = torch.ones(seqs * T, K, dtype=dt, device="cuda")
    a, b = torch.zeros(1, 8, K, dtype=dt, device="cuda"), torch.zeros(1, N, 8, dtype=dt, device="cuda")
    a[0, 0, :7], b[0, :, 0] = 1.0, 10000.0
    w = torch.full((N, K), -3750.0, dtype=dt, device="cuda")
    y = op("linear_adapted", ("cuda", dt), x, w, a, b, torch.ones(1, device="cuda"), i32(("cuda",), *[0] * seqs), T=T, out_dtype=dt)
    assert (y == 10000.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-9, 1e-38])
@pytest.mark.parametrize("r", [8, 40])
def test_small_fp16_numbers_between_the_products(r, size):
    """What stands between the products may be far below fp16's smallest normal number, 2^-14, in front of large rows of `b`."""
    T, seqs, K, N, dt = 40, 4, 64, 256, torch.float16
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(seqs * T, K, generator=g).to(dt), torch.zeros(N, K, dtype=dt)
    a, b = (torch.randn(2, r, K, generator=g) * 0.1).to(dt), (torch.randn(2, N, r, generator=g) * 4000).to(dt)
    scale = torch.full((2,), size)
    args = [t.cuda() for t in (x, w, a, b, scale)]
    y = op("linear_adapted", ("cuda", dt), *args, i32(("cuda",), 0, 1, 1, 0), T=T, out_dtype=dt).double().cpu()
    for i, s in enumerate((0, 1, 1, 0)):
        want = scale.double()[s] * (x[i * T:(i + 1) * T].double() @ a[s].double().T @ b[s].double().T)
        # half a step of the result (of its smallest step where it is below 2^-14), and 2^-18 for sums in 32 bits
        assert ((y[i * T:(i + 1) * T] - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + 2.0 ** -18 * want.abs().max()).all()


def test_signs_of_zeros(backend):  # noqa: F811
    """Results of zero have the sign that the formula gives them: 2 - 2 is zero, minus zero times a penalty minus zero."""
    dev, V = backend[0], 300
    logits = torch.zeros(1, V).to(backend[1])
    logits[0, :8] = torch.tensor([2.0, -0.0, -0.0, 0.0, -0.0, 3.0, -0.0, 2.0])
    history, tokens = i32(backend, 0, 1, 5, 7).reshape(1, 4), i32(backend, 2, 5, -1, 7).reshape(1, 4)
    values = torch.tensor([[0.0, -1.0, 0.0, -0.0]], device=dev)
    rules = (history, i32(backend, 0), torch.tensor([[1.0, 0.5, 1.5]], device=dev), tokens, values, torch.full((1, 10), -1, dtype=torch.int32, device=dev))
    x = op("shape_logits", backend, logits.to(dev), i32(backend, 0), i32(backend, 4), *rules).cpu()[0]
    # 2 - 0.5 - 1.5; (-0 - 0.5) - 1.5; -0 + 0; untouched ones; ((3 - 0.5) - 1.5) - 1; untouched; ((2 - 0.5) - 1.5) - 0
    assert x[:8].tolist() == [0.0, -2.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0]
    assert torch.signbit(x[:8]).tolist() == [False, True, False, False, True, False, True, False] and not torch.signbit(x[8:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S,V", [(2, 70001), (90, 50400), (3, 200000)])
def test_choice_from_parts_of_several_chunks(S, V, dtype):
    """A CTA of the choice takes its part of the row 8192 entries at a time: tokens, biases and masks of every chunk."""
    from popxl_addons_b200.xl.opdef import OPS
    from test_logits_ops import rules

    r, _ = rules(S, V, 3000, 12, seed=4)
    g = torch.Generator().manual_seed(6)
    r[0][:] = torch.randint(0, V, r[0].shape, generator=g)  # all over the vocabulary
    logits = torch.randint(-6, 7, (S, V), generator=g).to(dtype)
    for s in range(S):  # what wins without the rules lies in another chunk from row to row, and the tokens lose by the penalties
        logits[s, (s * 8191 + 17) % V] = 9.0
    length = torch.randint(0, 3000, (S,), generator=g).int()
    ref = OPS["shape_logits"].impl(logits, torch.arange(S, dtype=torch.int32), length, *r)
    want = [int((x == x.max()).int().argmax()) for x in ref]
    d = [x.cuda() for x in r]
    current, buf, pos = torch.full((S,), -7, dtype=torch.int32, device="cuda"), torch.zeros(1, S, dtype=torch.int32, device="cuda"), i32(("cuda",), 0)
    op("take_shaped_", ("cuda", dtype), current, logits.cuda(), buf, pos, length.cuda(), torch.ones(S, dtype=torch.int32, device="cuda"), *d, valid=V,
       base=0, ahead=0, advance=True)
    assert current.tolist() == want and len(set(want)) > min(S, 3) - 2 and pos.tolist() == [1]


@pytest.mark.gpu
def test_shaped_logits_of_parts_of_several_chunks():
    """Past 1024 parts of 8192 entries a CTA of the shaped row takes several chunks too."""
    from popxl_addons_b200.xl.opdef import OPS
    from test_logits_ops import rules

    V = 1024 * 8192 + 100001
    r, _ = rules(1, V, 5000, 2, seed=4)
    g = torch.Generator().manual_seed(6)
    r[0][:], r[2][:] = torch.randint(0, V, r[0].shape, generator=g), torch.tensor([1.3, 0.5, 0.25])
    logits = torch.randn(1, V, generator=g)
    args = (i32(("cpu",), 0), i32(("cpu",), 5000), *r)
    want = OPS["shape_logits"].impl(logits, *args)
    got = op("shape_logits", ("cuda", torch.float32), logits.cuda(), *[t.cuda() for t in args])
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("rows,K", [(1, 200), (9, 200), (40, 64), (100, 200)])
@pytest.mark.parametrize("which", ["x", "weight", "adapters"])
def test_adapted_operands_off_a_16_byte_boundary(backend, which, rows, K):  # noqa: F811
    """Rows and weights inside larger buffers: the sum is rounded once all the same."""
    dev, N, r = backend[0], 264, 8
    for dt in (backend[1],) if backend[1] == torch.float32 else (torch.bfloat16, torch.float16):
        x, w, a, b = (t.to(dev) for t in terms_that_cancel(dt, rows, K, N, r, seed=3))
        term = x.double() @ a[0].double().T @ b[0].double().T
        want = x.double() @ w.double().T + term
        if which == "x":
            x = shifted(x)
        elif which == "weight":
            w = shifted(w)
        else:
            a, b = shifted(a), shifted(b)
        y = op("linear_adapted", backend, x, w, a, b, torch.ones(1, device=dev), i32(backend, *[0] * rows), T=1, out_dtype=dt)
        step = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2  # as above
        assert ((y.double() - want).abs() <= step * want.abs() + (2.0 ** -15 if dt == torch.bfloat16 else 2.0 ** -18) * term.abs().max()).all()


def test_replays_do_not_record_gradients():
    """Inputs that require gradients leave the static inputs of a captured program without a history that grows with every replay."""
    from types import SimpleNamespace

    ir = xl.Ir()
    with ir.main_graph:
        stream = xl.h2d_stream((4,), xl.float32, "x")
    session, static = xl.Session(ir, "cpu"), torch.zeros(4)
    state = {"static_in": {stream: static}, "shared": None, "graph": SimpleNamespace(replay=lambda: None), "kernels": []}
    for i in range(3):
        session._stage_inputs({stream: torch.full((4,), float(i), requires_grad=True)}, keep_on_host=True)
        session._replay(state)
        assert static.tolist() == [i] * 4 and not static.requires_grad and static.grad_fn is None
