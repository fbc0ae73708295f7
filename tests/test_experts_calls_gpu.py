"""Calls of the experts beside the plain ones: views of every argument, weights,
logits, biases and padding that are not finite, tangents."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from oracle import experts as oracle
from wpt_amd import experts, kernels, sampling

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
BF16, FP32 = torch.bfloat16, torch.float32


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


@pytest.mark.parametrize("rows, D, E", [(1, 256, 8), (30, 64, 20), (3, 2048, 64), (200, 512, 100)])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_an_expert_taken_out_stays_out_whatever_its_logits(device, rows, D, E, value):
    print(f"route rows={rows} D={D} E={E} {value}", flush=True)
    x, router, _, _ = layer(1, rows, D, E, 8, BF16, seed=E)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(1))
    router[2, 5], bias[2] = value, -INF
    router[E - 1], bias[E - 1] = NAN, -INF
    expected = oracle.route(x, router, 4, bias)
    assert not bool(((expected[0] == 2) | (expected[0] == E - 1)).any()) and bool(expected[1].isfinite().all())
    chosen, gates = experts.route(x.to(device), router.to(device), 4, bias.to(device))
    assert torch.equal(chosen.cpu(), expected[0])
    assert bool(((gates.cpu().double() - expected[1]).abs() <= expected[1] * (2.0 ** -24 + 1e-9)).all())


# the down product of a few tokens over all experts at once (few k-steps, or wide outputs), and the other forms beside it
@pytest.mark.parametrize("rows, D, F", [(2, 256, 64), (3, 4096, 96), (16, 64, 32), (2, 256, 1200), (16, 512, 1200), (17, 256, 64),
                                        (200, 64, 32)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("value", [INF, NAN])
def test_an_expert_that_is_not_finite_reaches_its_own_tokens_alone(device, rows, D, F, dtype, value):
    print(f"rows={rows} D={D} F={F} {dtype} {value}", flush=True)
    E, k = 9, 2
    x, _, gate_up, down = layer(1, rows, D, E, F, dtype, seed=D + F)
    chosen = torch.stack([torch.arange(rows) % 8, torch.full((rows,), 8)], -1).view(1, rows, k).to(torch.int32)
    chosen[0, -1] = 3  # one expert twice
    gates = torch.rand(1, rows, k, generator=torch.Generator().manual_seed(0)) + 0.5
    on = [t.to(device) for t in (x, chosen, gates)]
    finite = experts.ExpertWeights(gate_up.to(device), down.to(device))
    y = experts.feed_forward(on[0], finite, on[1], on[2])
    broken = down.clone()
    broken[1, 5, F // 2] = value  # token 1's, 9's, ...; output 5
    weights = experts.ExpertWeights(gate_up.to(device), broken.to(device))
    got = experts.feed_forward(on[0], weights, on[1], on[2])
    mine = (chosen[0] == 1).any(-1).to(device)
    expected, _ = oracle.feed_forward(x, gate_up, broken, chosen, gates)
    assert torch.equal(got.isnan().cpu(), expected.isnan())
    assert not bool(got[0, mine, 5].isfinite().any())
    got[0, mine, 5] = y[0, mine, 5]
    assert torch.equal(got, y)
    # a gate matrix that is not: every output of its tokens
    broken = gate_up.clone()
    broken[1, 3, 0] = NAN
    got = experts.feed_forward(on[0], experts.ExpertWeights(broken.to(device), down.to(device)), on[1], on[2])
    assert bool(got[0, mine].isnan().all()) and torch.equal(got[0, ~mine], y[0, ~mine])


def test_tangents_are_refused(device):
    x, router, gate_up, down = (t.to(device) for t in layer(1, 3, 64, 8, 32, FP32))
    weights = experts.ExpertWeights(gate_up, down)
    chosen, gates = experts.route(x, router, 2)
    scores, tokens = torch.randn(1, 3, 100, device=device), torch.zeros(1, 3, dtype=torch.long, device=device)
    q, table = torch.randn(1, 3, 2, 64, device=device), torch.randn(1, 9, 128, device=device)
    positions = torch.arange(3, device=device)[None]
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: experts.route(dual(x), router, 2), lambda: experts.route(x, dual(router), 2),
                     lambda: experts.mixture(dual(x), router, weights, 2), lambda: experts.mixture(x, dual(router), weights, 2),
                     lambda: experts.mixture_parts(dual(x), router, weights, 2),
                     lambda: experts.feed_forward(x, weights, chosen, dual(gates)),
                     lambda: experts.feed_forward_parts(dual(x), weights, chosen, gates),
                     lambda: experts.ExpertWeights(gate_up, dual(down)), lambda: sampling.log_probs(dual(scores), tokens),
                     lambda: kernels.verify_attention(dual(q), table[..., :64], table[..., 64:], positions, 0.125)):
            with pytest.raises(NotImplementedError):
                call()
        assert experts.route(x, router, 2)[1].isfinite().all()


@pytest.mark.parametrize("B, T, D, E, k, F", [
    (1, 1, 256, 8, 2, 64), (2, 4, 64, 40, 2, 32),                   # fewer pairs than experts
    (4, 4, 72, 6, 2, 1200), (10, 8, 72, 6, 2, 40),                  # the width shared out
    (4, 2, 4096, 16, 2, 64), (30, 10, 1040, 64, 2, 512)])           # all experts at once; tiles
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_padding_may_hold_anything_and_be_all_there_is(device, B, T, D, E, k, F, dtype):
    print(f"B={B} T={T} D={D} E={E} k={k} F={F} {dtype}", flush=True)
    x, router, gate_up, down = (t.to(device) for t in layer(B, T, D, E, F, dtype, seed=F))
    weights = experts.ExpertWeights(gate_up, down)
    for counts in (torch.arange(B) % (T + 1), torch.zeros(B, dtype=torch.long)):
        counts = counts.to(device)
        padding = torch.arange(T, device=device) >= counts[:, None]
        results = []
        for value in (0.0, NAN, INF):
            held = x.clone()
            held[padding] = value
            for shape, kind in (((B, T, D), dtype), ((k, B * T, D), FP32)):  # what is not written shows
                torch.full(shape, NAN, dtype=kind, device=device)
            y, chosen, gates = experts.mixture(held, router, weights, k, None, counts)
            parts, _, _ = experts.mixture_parts(held, router, weights, k, None, counts)
            assert bool((y[padding] == 0).all()) and bool((parts[:, padding.view(-1)] == 0).all())
            assert bool((chosen[padding] == -1).all()) and bool((gates[padding] == 0).all())
            results.append((y, chosen, gates, parts))
        assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(results[0], other))
