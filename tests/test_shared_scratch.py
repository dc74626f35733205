"""Large scratch memory that the programs of a session share: the bookkeeping on the CPU; on the GPU captured programs of many sizes
whose memory does not add up, and programs that are replayed on several streams."""
import numpy as np
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.ops import native as nat
from popxl_addons_b200.xl import ops, read_ahead


class Stream:
    """Stands in for a CUDA stream; remembers whom it waited for."""

    def __init__(self, handle):
        self.handle, self.waited = handle, []

    def wait_stream(self, other):
        self.waited.append(other.handle)


@pytest.fixture
def on_cpu(monkeypatch):
    streams = {h: Stream(h) for h in (1, 2, 9)}
    state = {"stream": 1, "capturing": False, "streams": streams}
    monkeypatch.setattr(nat, "_stream", lambda: state["stream"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: streams[state["stream"]])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(nat, "_STREAM_SCRATCH", type(nat._STREAM_SCRATCH)())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
    return state


def taken(nbytes, most=1 << 20):
    return nat.large_scratch(nbytes, torch.device("cpu"), "x", most)


def test_programs_share_one_buffer(on_cpu):
    scratch = nat.SharedScratch()
    assert taken(100).data_ptr() != 0 and not scratch._buffers  # nobody shares
    with nat.sharing(scratch):
        assert taken(100) is not taken(100) and not scratch._buffers  # not in a program's order
        with read_ahead.following(read_ahead.LaunchOrder(1)):
            a = taken(1000)
            assert taken(500) is a and taken(1000) is a
            b = taken(1001)
            assert b is not a and b.numel() == 2000 and taken(1000) is b  # grows to twice as much
            assert taken(2001, most=2500).numel() == 2500 and taken(9000, most=2500).numel() == 9000
            c = taken(1)
        with read_ahead.following(read_ahead.LaunchOrder(5)):  # a side stream of the program
            assert taken(1) is not c
        with nat.sharing(None), read_ahead.following(read_ahead.LaunchOrder(1)):
            assert taken(1) is not c
    assert getattr(nat._CAPTURES, "shared", None) is None


def test_a_captured_graph_keeps_its_buffer(on_cpu):
    scratch, dev = nat.SharedScratch(), torch.device("cpu")
    with nat.sharing(scratch):
        with read_ahead.following(read_ahead.LaunchOrder(1)):
            a = taken(1000)
        on_cpu.update(capturing=True, stream=9)
        assert taken(10) is not a  # a capture that nobody keeps scratch for
        with nat.capture_scratch(dev) as held, read_ahead.following(read_ahead.LaunchOrder(9)):
            assert taken(1000) is a and taken(10) is a
            own = taken(1001)  # more than there is: the graph's own memory, nothing is allocated for others during a capture
            assert own is not a and scratch._buffers["x"] is a
        assert nat.uses_shared(held) and any(t is a for t in held.values()) and not any(t is own for t in held.values())
        with nat.capture_scratch(dev) as none, read_ahead.following(read_ahead.LaunchOrder(9)):
            taken(5000)
        assert not nat.uses_shared(none)
        on_cpu.update(capturing=False, stream=1)
        with read_ahead.following(read_ahead.LaunchOrder(1)):
            assert taken(5000) is not a
    assert held[f"shared x {a.data_ptr()}"] is a


def test_streams_take_turns(on_cpu):
    scratch, streams = nat.SharedScratch(), on_cpu["streams"]
    for at, waits in ((1, []), (1, []), (2, [1]), (2, [1]), (1, [2])):
        on_cpu["stream"] = at
        scratch.follow()
        assert streams[at].waited == waits


# ---- on the GPU ---------------------------------------------------------------------------------------------------------


def program_of(ir, held, B, T, H, G, d, window=0):
    """A portion of `T` tokens of each of `B` sequences, all projections the same number of columns."""
    p = xl.Program(ir, f"portion_{T}_{window}")
    with p:
        src, where = xl.h2d_stream((B * T, (H + 2 * G) * d), xl.bfloat16, "proj"), xl.h2d_stream((B,), xl.int32, "pos")
        dst = xl.d2h_stream((B * T, H * d), xl.float32, "y")
        cache = ops.Cache8(*(p.use(held[k], by_ref=True) for k in ops.Cache8._fields))
        pos = ops.host_load(where)
        joint = ops.cast(ops.host_load(xl.h2d_stream((B * T, H * d), xl.float32, "joint")), xl.bfloat16)
        y = ops.window_attention_q8_(ops.host_load(src), p.use(held["ones"]), p.use(held["ones"]), cache, pos, p.use(held["count"]), joint, T, H,
                                     d ** -0.5, window, 4 if window else 0)
        ops.host_store(dst, ops.cast(y, xl.float32))
    return p, {o.attrs["stream"].name: o.attrs["stream"] for o in p.graph.ops if o.opdef.name in ("host_load", "host_store")}


def session_of(B, G, blocks, d, T):
    ir, gen = xl.Ir(), torch.Generator().manual_seed(1)
    spec = ops.cache8_spec(B, G, blocks * 64, d, d, xl.bfloat16)
    held = {}
    with ir.main_graph:
        for k, (shape, dt) in spec.items():
            value = torch.randint(-127, 128, shape, generator=gen).to(torch.int8) if dt == xl.int8 else torch.full(shape, 0.02) if dt == xl.float32 else \
                torch.randn(shape, generator=gen).bfloat16()
            held[k] = xl.variable(value, dt, k)
        held["ones"], held["count"] = xl.variable(np.ones(d, np.float32), xl.float32, "ones"), xl.variable(np.full(B, T, np.int32), xl.int32, "count")
    return ir, held


@pytest.mark.gpu
def test_memory_of_captured_programs_does_not_add_up():
    """Twelve sizes of portions against caches whose codes are 134 MB as 16-bit numbers: once for all of them."""
    B, H, G, d, blocks = 2, 8, 4, 128, 512
    expanded = B * G * blocks * 64 * 2 * d * 2
    ir, held = session_of(B, G, blocks, d, 1)
    sizes = [65 + 16 * i for i in range(12)]  # rows for the tensor cores: those of 64 tokens of two heads run without expanded codes
    programs = [program_of(ir, held, B, T, H, G, d) for T in sizes]
    session = xl.Session(ir, "cuda:0")
    g = torch.Generator().manual_seed(2)

    def run(i):
        p, s = programs[i]
        return session.run_program(p, {s["proj"]: torch.randn(B * sizes[i], (H + 2 * G) * d, generator=g).bfloat16(),
                                       s["pos"]: torch.full((B,), 20000, dtype=torch.int32), s["joint"]: torch.zeros(B * sizes[i], H * d)})

    for _ in range(3):
        run(0)
    before = torch.cuda.memory_reserved()
    for i in range(1, 12):
        for _ in range(3):
            run(i)
    assert all(session._programs[p] is not None and session._programs[p]["shared"] is not None for p, _ in programs)
    assert torch.cuda.memory_reserved() - before < 2 * expanded  # eleven more without sharing


@pytest.mark.gpu
def test_portions_behind_a_window_hold_what_they_see():
    """Codes of the window and of the kept first tokens alone become 16-bit numbers, of a cache of 65536 positions that would be 268 MB."""
    from popxl_addons_b200.xl.opdef import OPS

    B, H, G, d, blocks, T = 2, 8, 4, 64, 1024, 130
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    cache = [torch.randint(-127, 128, (B, G, blocks, 64, d), generator=gen, device="cuda").to(torch.int8) for _ in range(2)]
    cache += [torch.full((B, G, blocks), 0.02, device="cuda") for _ in range(2)] + [n(B, G, 64, d).bfloat16() for _ in range(2)]
    proj, joint, ones = n(B * T, (H + 2 * G) * d).bfloat16(), torch.zeros(B * T, H * d, device="cuda").bfloat16(), torch.ones(d, device="cuda")
    where = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([60000, 7], [T, T])]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert OPS["window_attention_q8_"].native["cuda"](proj, ones, ones, *cache, *where, joint, T=T, heads=H, window=70, keep_first=100, scale=d ** -0.5,
                                                      sink=None, eps=1e-6) is joint
    assert torch.cuda.max_memory_allocated() - before < 8 << 20


@pytest.mark.gpu
def test_replays_on_several_streams():
    """Two programs of one session, with caches of their own, replayed in turn on two streams without anything else that orders them."""
    B, H, G, d, blocks, T = 2, 8, 4, 128, 128, 200
    ir, held = session_of(B, G, blocks, d, T)
    other = {**held}
    with ir.main_graph:
        gen = torch.Generator().manual_seed(5)
        for k in ("k", "v"):
            other[k] = xl.variable(torch.randint(-127, 128, held[k].shape, generator=gen).to(torch.int8), xl.int8, k + "_other")
        for k in ("k_scale", "v_scale", "k_tail", "v_tail"):
            other[k] = xl.variable(torch.full(held[k].shape, 0.02).to(held[k].dtype.as_torch()), held[k].dtype, k + "_other")
    programs = [program_of(ir, held, B, T, H, G, d), program_of(ir, other, B, T, H, G, d, window=3000)]
    session = xl.Session(ir, "cuda:0")
    g = torch.Generator().manual_seed(2)
    # from the start of a block: a portion that begins inside one and completes it cannot be run again, its tail is another block's then
    inputs = [{s["proj"]: torch.randn(B * T, (H + 2 * G) * d, generator=g).bfloat16(), s["pos"]: torch.full((B,), 94 * 64, dtype=torch.int32),
               s["joint"]: torch.zeros(B * T, H * d)} for _, s in programs]
    want = [session.run_program(p, x)[s["y"]] for (p, s), x in zip(programs, inputs)]
    for (p, _), x in zip(programs, inputs):
        session.run_program(p, x)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(40):
        k = i % 2
        with torch.cuda.stream(streams[k]):
            got.append((k, session.run_program(programs[k][0], inputs[k], fetch=False)[programs[k][1]["y"]]))
    torch.cuda.synchronize()
    for k, y in got:
        assert torch.equal(y.reshape(B * T, H * d).cpu(), torch.from_numpy(np.asarray(want[k])).reshape(B * T, H * d))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 150])
def test_portions_in_slices_of_sequences(monkeypatch, window):
    """Sequences whose codes do not fit what is set aside for them together go one or two at a time, with the same results."""
    from popxl_addons_b200.ops import native_serving as ns
    from popxl_addons_b200.xl.opdef import OPS

    B, H, G, d, dv, blocks, T = 5, 8, 2, 64, 128, 12, 140
    outs = []
    for limit in (None, 2, 1):
        gen = torch.Generator(device="cuda").manual_seed(1)
        n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
        cache = [torch.randint(-127, 128, (B, G, blocks, 64, w), generator=gen, device="cuda").to(torch.int8) for w in (d, dv)]
        cache += [torch.full((B, G, blocks), 0.02, device="cuda") for _ in range(2)] + [n(B, G, 64, w).bfloat16() for w in (d, dv)]
        proj, norm = n(B * T, (H + G) * d + (G + H) * dv).bfloat16(), 1 + 0.1 * n(d)
        joint = torch.full((B * T, H * dv + 8), -7.0, device="cuda").bfloat16()
        where = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([600, 0, 63, 400, 5], [T, T, 0, 77, 139])]
        calls = []
        with monkeypatch.context() as m:
            m.setattr(ns, "_q8_portion", lambda at, *a, real=ns._q8_portion: (calls.append(at), real(at, *a)))
            if limit:
                m.setattr(ns, "_Q8_EXPANDED", limit * G * ns._q8_held(T, blocks, window, 4) * 64 * (d + dv) * 2)
            OPS["window_attention_q8_"].native["cuda"](proj, norm, norm, *cache, *where, joint, T=T, heads=H, window=window, keep_first=4,
                                                       scale=d ** -0.5, sink=0.0, eps=1e-6)
        assert len(calls) == {None: 1, 2: 3, 1: 5}[limit]
        outs.append([joint, *cache])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.gpu
def test_adapted_products_share_what_is_between_them():
    """Results in 32 bits before adapters are added: one buffer, 67 MB, for eight programs, each with the results of the plain formula."""
    K, N, r, n = 256, 8192, 16, 2
    ir, gen = xl.Ir(), torch.Generator().manual_seed(1)
    shapes = {"w": (N, K), "a": (n, r, K), "b": (n, N, r)}
    values = {k: (torch.randn(s, generator=gen) * s[-1] ** -0.5).bfloat16() for k, s in shapes.items()}
    with ir.main_graph:
        held = {k: xl.variable(v, xl.bfloat16, k) for k, v in values.items()}
        held["scale"], held["slot"] = xl.variable(np.ones(n, np.float32), xl.float32, "scale"), xl.variable(np.array([1, 0], np.int32), xl.int32, "slot")
    programs = []
    for T in (1024, 960, 896, 832, 768, 704, 640, 576):
        p = xl.Program(ir, f"adapted_{T}")
        with p:
            src, dst = xl.h2d_stream((2 * T, K), xl.bfloat16, "x"), xl.d2h_stream((2,), xl.float32, "y")
            x = ops.host_load(src)
            y = ops.linear_adapted(x, p.use(held["w"]), ops.Adapters(*(p.use(held[k]) for k in ("a", "b", "scale"))), p.use(held["slot"]), T)
            picked = ops.reshape(ops.cast(y, xl.float32), (2, T * N))
            ops.host_store(dst, picked[:, T * N - 1])
        programs.append((p, src, dst, T))
    session = xl.Session(ir, "cuda:0")
    for p, src, dst, T in programs:
        x = torch.randn(2 * T, K, generator=gen).bfloat16()
        rows = x[[T - 1, 2 * T - 1]].double()
        want = torch.stack([row @ values["w"][-1].double() + row @ values["a"][s].double().T @ values["b"][s][-1].double() for row, s in zip(rows, (1, 0))])
        for _ in range(3):
            got = torch.from_numpy(np.asarray(session.run_program(p, {src: x})[dst])).double().reshape(2)
            assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15).all()  # one rounding, and sums in 32 bits
    kept = [{t.data_ptr() for tag, t in session._programs[p]["scratch"].items() if tag.startswith("shared")} for p, *_ in programs]
    assert all(len(k) == 1 and k == kept[0] for k in kept)
