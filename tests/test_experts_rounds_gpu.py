"""The experts' products past one range of pairs, one tile and one round of
rows, every output against 64 bits within the oracle's bound."""

import pytest
import torch

from tests import expert_sums
from wpt_amd import experts

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


def layer(device, rows, D, E, F, dtype, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=device) * std).to(dtype)

    router = torch.randn(E, D, generator=g, device=device) * D ** -0.5
    return normal(1, rows, D), router, normal(E, 2 * F, D, std=D ** -0.5), normal(E, D, F, std=F ** -0.5)


def within(got, expected, bound):
    worst = float(((got.double() - expected).abs() - bound).amax())
    assert worst <= 0, worst


def test_rounds_of_few_rows_of_wide_outputs(device):
    # a row's terms are 4 MiB: rounds of 128 rows
    rows, D, k = 300, 1 << 17, 8
    x, router, gate_up, down = layer(device, rows, D, 10, 32, BF16)
    y, chosen, gates = experts.mixture(x, router, experts.ExpertWeights(gate_up, down), k)
    within(y[0], *expert_sums.feed_forward(x[0], gate_up, down, chosen[0], gates[0]))


def dirty(*shapes):
    """Leaves NaN in the memory that outputs of these shapes are likely to get."""
    for shape, dtype in shapes:
        torch.full(shape, float("nan"), dtype=dtype, device="cuda")


def check(device, B, T, D, E, k, F, dtype, bias=None):
    """A layer of B texts of T tokens, some of them padding, as y and as terms."""
    print(f"B={B} T={T} D={D} E={E} k={k} F={F} {dtype}", flush=True)
    rows = B * T
    x, router, gate_up, down = layer(device, rows, D, E, F, dtype, seed=rows + F)
    x = x.view(B, T, D)
    counts = torch.linspace(T, T // 2, B).round().long().to(device)  # the last texts read half their tokens
    weights = experts.ExpertWeights(gate_up, down)
    dirty(((B, T, D), dtype), ((k, rows, D), FP32))
    y, chosen, gates = experts.mixture(x, router, weights, k, bias, counts)
    padding = (torch.arange(T, device=device) >= counts[:, None]).view(rows)
    assert bool((chosen.view(rows, k)[padding] == -1).all()) and int((chosen.view(rows, k)[~padding] < 0).sum()) == 0
    expected, bound = expert_sums.feed_forward(x.view(rows, D), gate_up, down, chosen.view(rows, k), gates.view(rows, k))
    within(y.view(rows, D), expected, bound)
    assert bool((y.view(rows, D)[padding] == 0).all())
    dirty(((k, rows, D), FP32), ((B, T, D), dtype))
    parts, again, _ = experts.mixture_parts(x, router, weights, k, bias, counts)
    assert torch.equal(again, chosen)
    within(parts.double().sum(0), expected, bound)
    assert bool((parts[:, padding] == 0).all())
    return chosen


# products of many row blocks over tiles of 64 tokens, by how the pairs are listed
@pytest.mark.parametrize("B, T, D, E, k, F", [
    (10, 20, 1040, 64, 2, 512),   # up to 2048 pairs, the terms of no expert cleared by one list
    (20, 35, 1040, 64, 2, 512),   # and by sixteen
    (25, 40, 1040, 64, 3, 512),   # up to 4096 pairs
    (25, 50, 264, 100, 4, 256),   # more, a tile or less an expert
    (50, 90, 264, 200, 2, 256),   # two ranges of 8192 pairs
    (26, 100, 520, 16, 4, 512)])  # and several tiles an expert
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_tiles_by_how_many_pairs_there_are(device, B, T, D, E, k, F, dtype):
    bias = torch.zeros(E, device=device)
    bias[3], bias[5] = 2.0, float("-inf")  # one expert far ahead, one without tokens
    chosen = check(device, B, T, D, E, k, F, dtype, bias)
    assert int((chosen == 5).sum()) == 0 and int((chosen == 3).sum()) > B * T * k // E


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_terms_past_one_round_of_rows(device, dtype):
    # 4096 rows' terms of 4096 outputs and 8 choices are 512 MiB
    check(device, 44, 100, 4096, 16, 8, 32, dtype)


@pytest.mark.parametrize("B, dtype", [(165, BF16), (83, FP32)])
def test_operands_past_one_round_of_rows(device, B, dtype):
    # 8 choices' 8192 features of 16383 rows (8191 in FP32) are a buffer of 2 GiB; the terms are written into one output
    check(device, B, 100, 64, 16, 8, 8192, dtype)
