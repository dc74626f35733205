"""Projections with an adapter of each request's own against the plain oracle: sequences without one, adapters that several share,
ranks that fill no tile, rows and columns that vector accesses do not divide. CPU backend, and marked `gpu` the kernels."""
import pytest
import torch

import plain_serving as plain
from test_dunelix_ops import backend, close, i32, op, rnd  # noqa: F401  (fixture and helpers)
from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops

# sequences, tokens of each, K, N, adapters, rank
SIZES = [(1, 1, 8, 8, 1, 1), (5, 1, 72, 130, 3, 8), (40, 1, 264, 514, 7, 16), (3, 7, 40, 33, 2, 5), (2, 16, 64, 128, 2, 16), (3, 70, 200, 250, 2, 24),
         (2, 129, 1032, 384, 4, 64), (4, 40, 136, 1001, 2, 3), (2, 100, 96, 256, 1, 128), (1, 300, 4096, 260, 2, 4), (70, 2, 128, 256, 5, 12)]


@pytest.mark.parametrize("B,T,K,N,n,r", SIZES)
def test_adapted_products(backend, B, T, K, N, n, r):  # noqa: F811
    x, x64 = rnd(backend, B * T, K, seed=1)
    w, w64 = rnd(backend, N, K, std=K ** -0.5, seed=2)
    a, a64 = rnd(backend, n, r, K, std=K ** -0.5, seed=3)
    b, b64 = rnd(backend, n, N, r, std=r ** -0.5, seed=4)
    scale = torch.linspace(0.5, 2.0, n)
    slot = [(3 * i) % (n + 2) - 1 for i in range(B)]  # -1 and n: no adapter
    want = plain.adapted(x64, w64, a64, b64, scale.double(), slot, T)
    outs = [backend[1]] + ([torch.float32] if backend[1] != torch.float32 else [])
    for out in outs:
        y = op("linear_adapted", backend, x, w, a, b, scale.to(backend[0]), i32(backend, *slot), T=T, out_dtype=out)
        assert y.dtype == out
        # fp32: sums of K + r products, each off by 2^-24 of terms below the largest result: 2e-5 covers 4096 of them many times.
        # bf16 results: one rounding of the sum, half a step, 2^-8 of the value at most
        # where rows are many (T >= 8) the adapters' term is rounded ahead of it: no more than 2^-8 of a term that here is smaller than
        # the largest result
        close(y, want, (backend[0], out), 2e-5, (1 if T < 8 else 2) * 2.0 ** -8 + 1e-4)


@pytest.mark.parametrize("T", [1, 64])
def test_rows_without_an_adapter_are_the_shared_product(backend, T):  # noqa: F811
    """What other sequences' adapters hold must not reach them: those here are infinite."""
    x, _ = rnd(backend, 3 * T, 64, seed=1)
    w, _ = rnd(backend, 256, 64, std=0.1, seed=2)
    a, b = torch.full((2, 16, 64), float("inf")).to(x), torch.full((2, 256, 16), float("inf")).to(x)
    y = op("linear_adapted", backend, x, w, a, b, torch.ones(2, device=backend[0]), i32(backend, -1, 1, 2), T=T, out_dtype=backend[1])
    want = x.double().cpu() @ w.double().cpu().T
    close(y[:T], want[:T], backend, 2e-5, 2.0 ** -8)
    close(y[2 * T:], want[2 * T:], backend, 2e-5, 2.0 ** -8)
    assert not torch.isfinite(y[T:2 * T]).any()


@pytest.mark.parametrize("T", [1, 40])
def test_strided_rows(backend, T):  # noqa: F811
    x, x64 = rnd(backend, 2 * T, 72, seed=1)
    w, w64 = rnd(backend, 136, 40, std=0.15, seed=2)
    a, a64 = rnd(backend, 3, 8, 40, std=0.15, seed=3)
    b, b64 = rnd(backend, 3, 136, 8, std=0.3, seed=4)
    scale = torch.ones(3)
    y = op("linear_adapted", backend, x[:, 3:43], w, a, b, scale.to(backend[0]), i32(backend, 2, 2), T=T, out_dtype=backend[1])
    close(y, plain.adapted(x64[:, 3:43], w64, a64, b64, scale.double(), [2, 2], T), backend, 2e-5, 2 * 2.0 ** -8 + 1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("r", [8, 40])
def test_fp16_numbers_past_its_range(r):
    """What stands between the products may be larger than fp16 holds (65504), next to rows of ordinary size."""
    backend, T = ("cuda", torch.float16), 50  # noqa: F811
    x, x64 = rnd(backend, T, 256, seed=1)
    x[::3] *= 40.0  # exact powers are not needed: both sides read the rounded values
    x64 = x.double().cpu()
    w, w64 = rnd(backend, 256, 256, std=1e-3, seed=2)
    a, a64 = rnd(backend, 1, r, 256, std=200.0, seed=3)
    b, b64 = rnd(backend, 1, 256, r, std=2e-4, seed=4)
    assert (x64 @ a64[0].T).abs().max() > 65504
    y = op("linear_adapted", backend, x, w, a, b, torch.ones(1, device="cuda"), i32(backend, 0), T=T, out_dtype=torch.float16)
    want = plain.adapted(x64, w64, a64, b64, torch.ones(1).double(), [0], T)
    for i in range(T):  # two roundings of half a step of fp16, 2^-11 each, and sums in 32 bits
        close(y[i], want[i], backend, 0, 2 * 2.0 ** -11 + 1e-4)


def test_refusals():
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.bfloat16):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def adapters(n=2, r=4, K=16, N=24, dt=xl.bfloat16):
            return ops.Adapters(var((n, r, K), dt), var((n, N, r), dt), var((n,), xl.float32))

        x, w, slot = var((6, 16)), var((24, 16)), var((3,), xl.int32)
        assert ops.linear_adapted(x, w, adapters(), slot, 2).shape == (6, 24)
        with pytest.raises(ValueError, match="sequences of"):
            ops.linear_adapted(x, w, adapters(), slot, 3)
        with pytest.raises(ValueError, match="sequences of"):
            ops.linear_adapted(x, w, adapters(), var((3,), xl.float32), 2)
        with pytest.raises(ValueError, match="adapters.a"):
            ops.linear_adapted(x, w, adapters(K=8), slot, 2)
        with pytest.raises(ValueError, match="adapters.b"):
            ops.linear_adapted(x, w, adapters(N=8), slot, 2)
        with pytest.raises(ValueError, match="adapters.a"):
            ops.linear_adapted(x, w, adapters(dt=xl.float32), slot, 2)
        with pytest.raises(ValueError, match="cannot multiply"):
            ops.linear_adapted(x, var((24, 17)), adapters(), slot, 2)
