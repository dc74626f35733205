"""Choices of beams that hang on the last bits of sums over whole rows, against the float64 oracle. CPU backend, and marked `gpu` the kernels in
every type."""
import math

import pytest
import torch

from test_beams_ops import backend, check_beams  # noqa: F401  (fixture and helper)

KINDS = {"normal": 2.5, "wide": 6.0, "flat": 0.25, "rising": 2.5}  # spread of the logits; rising: every chunk of a row has a new maximum


def base_rows(groups, V, kind, dtype):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(groups, V, generator=g) * KINDS[kind]
    return (x.sort(-1).values if kind == "rising" else x).to(dtype)


def three_beams(rows, other, order):
    """Groups of three slots, one of them empty, the others with rows that are alike or nearly so: their first continuations come first, and the third
    place is between their second ones."""
    groups, V = rows.shape
    logits = torch.stack([torch.zeros_like(rows)] + [(rows, other)[i] for i in order], 1).reshape(groups * 3, V)
    scores = torch.full((groups * 3,), -3.25)
    scores[::3] = -math.inf
    return logits, scores, torch.zeros(groups * 3, dtype=torch.int32), torch.full((groups * 3,), 2, dtype=torch.int32)


@pytest.mark.parametrize("V", [50257, 32003, 4099])
@pytest.mark.parametrize("kind", list(KINDS))
def test_equal_rows_of_several_beams(backend, V, kind):  # noqa: F811
    """Rows of an odd length begin at every place of a 16-byte unit: what is alike is worth the same wherever it lies."""
    rows = base_rows(20, V, kind, backend[1])
    check_beams(backend, *three_beams(rows, rows, (0, 1)), 3, None, V, 0.0)
    check_beams(backend, *three_beams(rows, rows, (0, 1)), 3, None, V, 0.7, in_place=True)


@pytest.mark.parametrize("V", [50257, 4099])
@pytest.mark.parametrize("kind", ["normal", "wide", "rising"])
@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_rows_that_differ_in_one_unlikely_token(backend, V, kind, order):  # noqa: F811
    """One row lacks a token of a probability of about 3e-8, and its other tokens are as much more likely: far more than the roundings of 64 bits,
    less than those of 32."""
    rows = base_rows(12, V, kind, backend[1])
    other = rows.clone()
    p = torch.softmax(rows.double(), -1)
    token = (p.log() - math.log(3e-8)).abs().argmin(-1)
    lost = p[torch.arange(len(rows)), token]
    other[torch.arange(len(rows)), token] = -math.inf
    live = (lost > 1e-9) & (lost < 1e-6)  # rows that have such a token
    if not live.any():
        pytest.skip("no token is that unlikely")
    logits, scores, ended, length = three_beams(rows[live], other[live], order)
    for b in range(0, len(scores), 3):  # the oracle sees the difference
        sums = torch.logsumexp(logits[b + 1:b + 3].double(), -1)
        assert 1e-9 < (sums[0] - sums[1]).abs() < 1e-6
    check_beams(backend, logits, scores, ended, length, 3, None, V, 0.0)


def test_ended_beams_next_to_live_ones(backend):  # noqa: F811
    """An ended beam whose sum is the nearest number in 32 bits to that of a live beam's second continuation, where a prompt's beams have unlike lengths
    and sums are divided by them."""
    V, groups, K = 50257, 16, 2
    rows = base_rows(groups, V, "normal", backend[1])
    logits = torch.stack((rows, rows), 1).reshape(groups * K, V)
    ended, length = torch.tensor([0, 1] * groups).int(), torch.tensor([3, 7] * groups).int()
    second = torch.log_softmax(rows.double(), -1).sort(-1, descending=True).values[:, 1] - 1.5
    for penalty in (0.0, 1.0):
        scores = torch.full((groups * K,), -1.5)
        scores[1::2] = (second * (7 / 4) ** penalty).float()
        check_beams(backend, logits, scores, ended, length, K, 5, V, penalty)


def test_many_rows_that_are_alike(backend):  # noqa: F811
    """All beams of all groups alike: every sum is needed to the last bit."""
    groups, K, V = 3, 16, 9001
    rows = base_rows(1, V, "normal", backend[1]).expand(groups * K, V).contiguous()
    ended, length = torch.zeros(groups * K, dtype=torch.int32), torch.ones(groups * K, dtype=torch.int32)
    check_beams(backend, rows, torch.full((groups * K,), -2.0), ended, length, K, None, V, 0.5)
    scores = -torch.arange(groups * K).float() * 2.0 ** -20  # and sums that differ by a few steps
    check_beams(backend, rows, scores, ended, length, K, None, V, 0.0)


def test_slots_without_a_beam_that_are_marked_as_ended(backend):  # noqa: F811
    """They fill up a group whose beams have all ended, at minus infinity, and keep their mark and their number of tokens."""
    V, K = 40, 4
    logits = torch.randn(3 * K, V, generator=torch.Generator().manual_seed(1)).to(backend[1])
    scores = torch.tensor([-math.inf, -3.0, -1.5, -2.0, math.nan, -1.0, math.inf, -math.inf, -2.5, -math.inf, -math.inf, -4.0])
    ended, length = torch.tensor([1, 1, 1, 1, 1, 1, 0, 1, 1, 0, 1, 1]).int(), torch.arange(3 * K).int() + 5
    for end, penalty in ((3, 0.0), (0, 0.8), (None, 0.0)):
        check_beams(backend, logits, scores, ended, length, K, end, V, penalty)
