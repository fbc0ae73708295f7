"""Calls of the experts beside the plain ones: views of every argument."""

import pytest
import torch

from oracle import experts as oracle
from wpt_amd import experts

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def layer(B, T, D, E, F, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    x = normal(B, T, D).to(dtype)
    return x, normal(E, D) * D ** -0.5, (normal(E, 2 * F, D) * D ** -0.5).to(dtype), (normal(E, D, F) * F ** -0.5).to(dtype)


@pytest.mark.parametrize("rows", [3, 40, 600])
def test_given_choices_and_gates_may_both_be_views(device, rows):
    x, router, gate_up, down = (t.to(device) for t in layer(2, rows, 64, 16, 32, BF16, seed=rows))
    weights = experts.ExpertWeights(gate_up, down)
    chosen, gates = experts.route(x, router, 4)
    n = rows - 1
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (chosen, gates)]
    for rows_, c, g in ((x[:, :n], chosen[:, :n], gates[:, :n]),            # a part of the tokens
                        (x, chosen[..., 1:3], gates[..., 1:3]),             # some of the choices
                        (x, turned[0], turned[1]),
                        (x, chosen[:, :1].expand(2, rows, 4), gates[:, :1].expand(2, rows, 4))):
        held = rows_.contiguous(), c.contiguous(), g.contiguous()
        expected = experts.feed_forward(held[0], weights, held[1], held[2])
        parts = experts.feed_forward_parts(held[0], weights, held[1], held[2])
        y, bound = oracle.feed_forward(*(t.cpu() for t in (held[0][:, :2], gate_up, down, held[1][:, :2], held[2][:, :2])))
        assert bool(((expected[:, :2].cpu().double() - y).abs() <= bound).all()) and bool((y.abs().amax(-1) > 0).all())
        for _ in range(3):
            same = torch.equal(experts.feed_forward(rows_, weights, c, g), expected)
            same_parts = torch.equal(experts.feed_forward_parts(rows_, weights, c, g), parts)
            assert same and same_parts
