"""What attention over an 8-bit cache reads before its predecessor on the stream has ended: only what was complete before that
predecessor started. The question that the binding asks, on the CPU; and on the GPU replayed programs in which the launch before writes
factors of norms, positions, or the cache itself."""
import numpy as np
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops
from popxl_addons_b200.xl.opdef import OPS
from test_read_ahead import _replayed

B, H, G, D, DV, BLOCKS = 2, 8, 2, 64, 64, 3
COLS = (H + G) * D + G * DV


def cache_of(seed):
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(-127, 128, (B, G, BLOCKS, 64, w), generator=g).to(torch.int8) for w in (D, DV)]
    return codes + [torch.full((B, G, BLOCKS), 0.02) for _ in range(2)] + [torch.randn(B, G, 64, w, generator=g).bfloat16() for w in (D, DV)]


class OnDevice(torch.Tensor):
    """A tensor of the CPU that says it is the device's."""

    @property
    def is_cuda(self):
        return True


def test_every_operand_that_is_read_ahead_is_asked_about(monkeypatch):
    """The kernel reads all but the projections ahead: factors of both norms, positions, counts and the cache."""
    from popxl_addons_b200.ops import native_serving as ns

    asked, ahead = [], []
    for name, fake in (("_ok", lambda *t: True), ("_i32", lambda *t: True), ("_stream", lambda: 0), ("_sms", lambda device: 148),
                       ("_count", lambda name: None), ("counters", lambda n, *a: torch.zeros(n, dtype=torch.int32)),
                       ("gemm_error_flag", lambda device: torch.zeros(1, dtype=torch.int32)),
                       ("_q8_few", lambda *a: ahead.append(a[-3]) or 0)):
        monkeypatch.setattr(ns, name, fake)
    monkeypatch.setattr(ns.read_ahead, "allowed", lambda *t: asked.extend(t) or True)
    proj, joint = (torch.zeros(B, n).bfloat16().as_subclass(OnDevice) for n in (COLS, H * DV))
    operands = {"q_norm": torch.ones(D), "k_norm": torch.ones(D), **dict(zip(ops.Cache8._fields, cache_of(0))),
                "pos": torch.zeros(B, dtype=torch.int32), "count": torch.ones(B, dtype=torch.int32)}
    operands = {k: t.as_subclass(OnDevice) for k, t in operands.items()}
    ns.window_attention_q8_cuda(proj, *operands.values(), joint, T=1, heads=H, window=0, keep_first=0, scale=0.125, sink=None, eps=1e-6)
    assert ahead == [1]
    held = {t.data_ptr() for t in asked}
    assert [k for k, t in operands.items() if t.data_ptr() not in held] == []


@pytest.mark.gpu
@pytest.mark.parametrize("written", ["factors", "positions", "cache"])
def test_operands_written_by_the_launch_before(written):
    """Factors that a gather takes out of a table, positions that were just advanced, and a block that the token before completed,
    each directly in front of the attention of one token."""
    table = 0.5 + torch.rand(2000, D, generator=torch.Generator().manual_seed(3))
    start = cache_of(1)
    want_cache = [t.clone() for t in start]

    def build(use, streams):
        for name, shape, dt in (("pos", (B,), xl.int32), ("by", (B,), xl.int32), ("row", (2,), xl.int32), ("first", (B, COLS), xl.bfloat16),
                                ("proj", (B, COLS), xl.bfloat16)):
            streams[name] = xl.h2d_stream(shape, dt, name)
        streams["y"] = xl.d2h_stream((B, H * DV), xl.float32, "y")
        pos, by, row, first, proj = (ops.host_load(streams[k]) for k in ("pos", "by", "row", "first", "proj"))
        joint = ops.cast(use("zeros"), xl.bfloat16)
        cache, factors = ops.Cache8(*(use(k) for k in ops.Cache8._fields)), ops.reshape(ops.gather(use("table"), row), (2, D))
        ops.linear_rows(first, use("w"))  # a launch of this library, so that only what follows is in doubt
        if written == "factors":
            factors = ops.reshape(ops.gather(use("table"), row), (2, D))
        elif written == "positions":
            ops.advance_by_(pos, by)
        else:
            ops.window_attention_q8_(first, factors[0], factors[1], cache, pos, use("count"), joint, 1, H, 0.125)
            pos = pos + by
            ops.linear_rows(first, use("w"))
            ops.window_attention_q8_(first, factors[0], factors[1], cache, pos, use("count"), joint, 1, H, 0.125)
            pos = use("after")
        y = ops.window_attention_q8_(proj, factors[0], factors[1], cache, pos, use("count"), joint, 1, H, 0.125)
        ops.host_store(streams["y"], ops.cast(y, xl.float32))

    def make(g):
        pos = torch.randint(0, 120, (B,), generator=g, dtype=torch.int32)
        if written == "cache":
            pos = torch.full((B,), 62, dtype=torch.int32)
        return {"pos": pos, "by": torch.ones(B, dtype=torch.int32) if written == "cache" else torch.randint(0, 60, (B,), generator=g, dtype=torch.int32),
                "row": torch.randint(0, 2000, (2,), generator=g, dtype=torch.int32),
                "first": torch.randn(B, COLS, generator=g).bfloat16(), "proj": torch.randn(B, COLS, generator=g).bfloat16()}

    def check(inputs, y, held):
        factors, pos, one = table[inputs["row"].long()], inputs["pos"].clone(), torch.ones(B, dtype=torch.int32)
        how = dict(T=1, heads=H, window=0, keep_first=0, scale=0.125, sink=None, eps=1e-6)

        def run(rows, at):
            return OPS["window_attention_q8_"].impl(rows, factors[0], factors[1], *want_cache, at, one, torch.zeros(B, H * DV), **how)

        if written == "positions":
            pos = pos + inputs["by"]
        elif written == "cache":
            run(inputs["first"], pos)
            run(inputs["first"], pos + 1)
            pos = pos + 2
        want = run(inputs["proj"], pos)
        for name, t in zip(ops.Cache8._fields, want_cache):
            assert torch.equal(held[name].cpu(), t), name
        # queries and weights over codes in fp16 (2^-11 each, a score below 8 off by 2^-8 at most), values of one size, bf16 results (2^-8)
        assert float((y - want).abs().max() / want.abs().max()) <= 2 * 2.0 ** -8

    variables = {**{k: (t, dt) for (k, (_, dt)), t in zip(ops.cache8_spec(B, G, BLOCKS * 64, D, DV, xl.bfloat16).items(), start)},
                 "table": (table, xl.float32), "count": (np.ones(B, np.int32), xl.int32), "after": (np.full(B, 64, np.int32), xl.int32),
                 "zeros": (torch.zeros(B, H * DV), xl.float32), "w": (torch.randn(64, COLS).bfloat16(), xl.bfloat16)}
    _replayed(build, variables, make, check, runs=60)
