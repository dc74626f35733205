"""Scratch memory of attention over shared prefixes: one buffer for all programs of a session."""
import numpy as np
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from popxl_addons_b200.xl.opdef import OPS

SIZES = {"groups": (xl.bfloat16, (4, 3, 2, 1)), "general": (xl.float32, (40, 30, 20, 5))}  # tokens of the programs, the most first


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(SIZES))
def test_programs_share_parts_of_sums_and_queries(kind):
    """Programs of several numbers of tokens, each replayed after the others have run: the reference's results, and one buffer for all."""
    dt, sizes = SIZES[kind]
    B, H, G, d, room = 64, 16, 2, 128, 700
    ir, gen = xl.Ir(), torch.Generator().manual_seed(1)
    torch_dt = torch.bfloat16 if dt == xl.bfloat16 else torch.float32
    values = {k: torch.randn(B, G, room, d, generator=gen).to(torch_dt) for k in "kv"}
    where = {"pos": torch.arange(B) % 50 + 600, "lead": torch.arange(B) // 16 * 16, "shared": torch.full((B,), 580)}
    with ir.main_graph:
        held = {k: xl.variable(v, dt, k) for k, v in values.items()}
        held |= {k: xl.variable(v.int().numpy(), xl.int32, k) for k, v in where.items()}
        held["unit"] = xl.variable(torch.eye((H + 2 * G) * d).to(torch_dt), dt, "unit")
        held["ones"] = xl.variable(np.ones(d, np.float32), xl.float32, "ones")
    programs = []
    for T in sizes:
        p = xl.Program(ir, f"portion_{T}")
        with p:
            src, dst = xl.h2d_stream((B * T, (H + 2 * G) * d), dt, "proj"), xl.d2h_stream((B * T, H * d), xl.float32, "y")
            proj = ops.linear_rows(ops.host_load(src), p.use(held["unit"]))  # as in a model, and exactly what was loaded
            joint = ops.cast(ops.host_load(xl.h2d_stream((B * T, H * d), xl.float32, "joint")), dt)
            y = ops.window_attention_shared_(proj, p.use(held["ones"]), p.use(held["ones"]), p.use(held["k"], by_ref=True), p.use(held["v"], by_ref=True),
                                             p.use(held["pos"]), xl.constant(np.full(B, T), xl.int32, "count"), p.use(held["lead"]), p.use(held["shared"]),
                                             joint, T, H, d ** -0.5)
            ops.host_store(dst, ops.cast(y, xl.float32))
        streams = {o.attrs["stream"].name: o.attrs["stream"] for o in p.graph.ops if o.opdef.name in ("host_load", "host_store")}
        programs.append((p, streams, T))
    session = xl.Session(ir, "cuda:0")
    eps = torch.finfo(torch_dt).eps
    for _ in range(4):
        for p, s, T in programs:
            x = torch.randn(B * T, (H + 2 * G) * d, generator=gen).to(torch_dt)
            got = torch.from_numpy(np.asarray(session.run_program(p, {s["proj"]: x, s["joint"]: torch.zeros(B * T, H * d)})[s["y"]])).reshape(B * T, -1)
            args = [x, torch.ones(d), torch.ones(d), values["k"], values["v"], where["pos"], torch.full((B,), T), where["lead"], where["shared"],
                    torch.zeros(B * T, H * d, dtype=torch_dt)]
            args = [a.cuda() if a.dtype != torch.int64 else a.int().cuda() for a in args]
            want = OPS["window_attention_shared_"].impl(*args, T=T, heads=H, window=0, keep_first=0, scale=d ** -0.5, sink=None, eps=1e-6).float().cpu()
            bound = 1.0625 * eps if torch_dt == torch.bfloat16 else 4e-5  # as for the kernels by themselves
            assert (got - want).abs().max() <= bound * want.abs().max()
    kept = [{t.data_ptr() for tag, t in session._programs[p]["scratch"].items() if tag.startswith("shared")} for p, *_ in programs]
    assert all(len(k) == 1 and k == kept[0] for k in kept)


@pytest.mark.gpu
def test_nothing_comes_between_the_append_and_the_groups(monkeypatch):
    """Taking memory may make the stream wait for another one, and the groups read what came before the append without waiting for it."""
    from popxl_addons_b200.ops import native_beams
    from test_shared_attention_edges import case, outputs

    order = []
    for name in ("large_scratch", "_shared_append", "_shared_groups"):
        monkeypatch.setattr(native_beams, name, lambda *a, f=getattr(native_beams, name), n=name, **kw: order.append(n) or f(*a, **kw))
    outputs(*case("cuda", torch.bfloat16, 4, 1, 8, 2, 64, 64, 300, 200, 1, 0, 150))
    assert order == ["large_scratch", "_shared_append", "_shared_groups"]
