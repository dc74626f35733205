"""Attention over shared prefixes at sizes where tiles have several row blocks, CTAs several tiles and tiles several CTAs: the kernels against the
CPU reference's arithmetic on the GPU."""
import pytest
import torch

from popxl_addons_b200.xl.opdef import OPS
import popxl_addons_b200.xl.ops  # noqa: F401  (registers the ops)

pytestmark = pytest.mark.gpu

# sequences, leads (every so many), T, query heads, key / value heads, dim, vdim, prefix, own tokens up to, window, kept
SIZES = {"rows": (70, 70, 1, 32, 4, 128, 128, 1500, 300, 0, 0),        # five tiles of one group's rows
         "groups": (120, 5, 1, 6, 2, 64, 64, 700, 600, 0, 0),           # small tiles, own keys of several blocks
         "windows": (48, 12, 1, 16, 2, 96, 80, 900, 500, 260, 70),
         "heads": (5, 5, 1, 300, 2, 40, 24, 333, 20, 0, 0),             # a sequence's heads do not fit a tile
         "many": (440, 440, 1, 16, 16, 8, 8, 6000, 60, 0, 0),           # more tiles of a CTA than its table has places
         "more": (500, 100, 1, 4, 2, 16, 16, 200, 90, 0, 0),            # more sequences than the list has places
         "alone": (300, 1, 1, 8, 8, 128, 64, 0, 700, 0, 0),
         "portions": (9, 3, 150, 8, 2, 128, 128, 1000, 200, 0, 0),
         "tokens": (40, 20, 3, 16, 4, 64, 128, 800, 150, 400, 5)}


@pytest.mark.parametrize("name", list(SIZES))
def test_large_batches_against_the_reference(name):
    """Both sides round the same sums once, eps / 2 each, and weights and queries of two bf16 numbers lose 2^-12: 1.0625 eps of the largest output.
    New keys are equal: their norms are taken in 64 bits."""
    from popxl_addons_b200.ops import native

    B, per, T, H, G, d, dv, prefix, most, window, keep = SIZES[name]
    g = torch.Generator(device="cuda").manual_seed(len(name))
    dt, dev = torch.bfloat16, "cuda"

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dt)

    own = torch.randint(0, most + 1, (B,), device=dev, generator=g)
    lead = torch.arange(B, device=dev) // per * per
    pos = (prefix + own).int()
    shared = torch.full((B,), prefix, dtype=torch.int32, device=dev)
    shared[3::7] = prefix // 2  # some left the prefix earlier
    count = torch.full((B,), T, dtype=torch.int32, device=dev)
    count[5::11] = max(0, T - 2)
    room = (prefix + most + T + 7) // 8 * 8
    k, v = rnd(B, G, room, d), rnd(B, G, room, dv)
    proj = rnd(B * T, (H + G) * d + (G + H) * dv)
    wq, wk = 1.5 + 0.2 * torch.randn(d, device=dev, generator=g), 1.2 + 0.2 * torch.randn(d, device=dev, generator=g)
    joint = torch.full((B * T, H * dv), -7.0, dtype=dt, device=dev)
    args = [proj, wq, wk, k, v, pos, count, lead.int(), shared, joint]
    kw = dict(T=T, heads=H, window=window, keep_first=keep, scale=d ** -0.5, sink=0.0, eps=1e-6)
    other = [a.clone() for a in args]
    want = OPS["window_attention_shared_"].impl(*other, **kw)
    for _ in range(2):  # the second time with scratch memory that has been used
        got = OPS["window_attention_shared_"].native["cuda"](*args, **kw)
        torch.cuda.synchronize()
        native.check_gemm_errors()
        assert torch.equal(args[3], other[3]) and torch.equal(args[4], other[4])
        assert torch.equal(got == -7, want == -7)
        top = want[want != -7].abs().max().item()
        assert (got.float() - want.float()).abs().max().item() <= 1.0625 * torch.finfo(dt).eps * top


def test_two_streams_at_a_time():
    """Calls on two streams, each with scratch memory of its own."""
    from popxl_addons_b200.ops import native

    calls = []
    for seed in range(2):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def rnd(*shape):
            return torch.randn(*shape, device="cuda", generator=g).bfloat16()

        B, H, G, d, room = 24, 8, 2, 128, 640
        i32 = dict(dtype=torch.int32, device="cuda")
        args = [rnd(B, (H + G) * d + (G + H) * d), torch.ones(d, device="cuda"), torch.ones(d, device="cuda"), rnd(B, G, room, d), rnd(B, G, room, d),
                torch.full((B,), 600, **i32), torch.ones(B, **i32), torch.zeros(B, **i32), torch.full((B,), 500 - 100 * seed, **i32),
                torch.zeros(B, H * d, device="cuda").bfloat16()]
        calls.append((args, dict(T=1, heads=H, window=0, keep_first=0, scale=d ** -0.5, sink=None, eps=1e-6)))
    op = OPS["window_attention_shared_"].native["cuda"]
    want = [op(*a, **k).clone() for a, k in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for s, (a, k) in zip(streams, calls):
            with torch.cuda.stream(s):
                op(*a, **k)
    torch.cuda.synchronize()
    native.check_gemm_errors()
    assert all(torch.equal(a[-1], w) for (a, _), w in zip(calls, want))
