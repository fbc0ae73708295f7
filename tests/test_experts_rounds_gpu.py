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
