"""The mixture of experts (wptv_route, wptv_experts, wptv_mixture) against plain
64-bit definitions.

The choice is equal: both sides rank in 64 bits.  A gate is a softmax in 64 bits
rounded once to FP32: half a step, 2^-24 of itself (and 1e-9 for the logits' own
64-bit sums).  The blocks' bound is oracle.experts.feed_forward's."""

import math

import pytest
import torch

from oracle import experts as oracle
from wpt_amd import experts

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
BF16, FP32 = torch.bfloat16, torch.float32


def layer(B, T, D, E, F, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    x = normal(B, T, D).to(dtype)
    return x, normal(E, D) * D ** -0.5, (normal(E, 2 * F, D) * D ** -0.5).to(dtype), (normal(E, D, F) * F ** -0.5).to(dtype)


def gates_close(got, expected):
    assert got.dtype == FP32
    assert bool(((got.cpu().double() - expected).abs() <= expected * (2.0 ** -24 + 1e-9)).all())


def check_route(device, x, router, k, bias=None, counts=None):
    on = [None if t is None else t.to(device) for t in (x, router, bias, counts)]
    chosen, gates = experts.route(on[0], on[1], k, on[2], on[3])
    expected = oracle.route(x, router, k, bias, counts)
    assert chosen.dtype == torch.int32 and torch.equal(chosen.cpu(), expected[0])
    gates_close(gates, expected[1])
    return expected


def y_close(got, expected, dtype):
    y, bound = expected
    assert got.dtype == dtype
    assert bool(((got.cpu().double() - y).abs() <= bound).all())


def check_mixture(device, x, router, gate_up, down, k, bias=None, counts=None):
    weights = experts.ExpertWeights(gate_up.to(device), down.to(device))
    on = [None if t is None else t.to(device) for t in (x, router, bias, counts)]
    y, chosen, gates = experts.mixture(on[0], on[1], weights, k, on[2], on[3])
    expected = oracle.route(x, router, k, bias, counts)
    assert torch.equal(chosen.cpu(), expected[0])
    gates_close(gates, expected[1])
    y_close(y, oracle.feed_forward(x, gate_up, down, *expected), x.dtype)
    return weights, on, (y, chosen, gates)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("B, T, D, E, k", [
    (1, 1, 8, 1, 1), (1, 1, 256, 8, 2), (2, 3, 264, 37, 5), (1, 7, 2048, 64, 8), (3, 1, 4096, 128, 16), (1, 2, 24, 512, 16),
    (257, 1, 64, 9, 3), (2, 150, 72, 16, 4), (1, 1, 16, 16, 16)])
def test_the_choice_is_the_sorted_logits(device, B, T, D, E, k, dtype):
    print(f"route B={B} T={T} D={D} E={E} k={k} {dtype}", flush=True)
    x, router, _, _ = layer(B, T, D, E, 8, dtype, seed=D + E)
    check_route(device, x, router, k)
    g = torch.Generator().manual_seed(1)
    check_route(device, x, router, k, torch.randn(E, generator=g), torch.randint(0, T + 1, (B,), generator=g))


def test_more_tokens_than_a_grid_s_dimension(device):
    rows, D, E = (1 << 19) + 1000, 40, 512
    g = torch.Generator(device=device).manual_seed(0)
    x = torch.randn(1, rows, D, generator=g, device=device).to(BF16)
    router = torch.randn(E, D, generator=g, device=device)
    chosen, gates = experts.route(x, router, 2)
    for part in (slice(0, 500), slice((1 << 19) - 500, None)):
        expected = torch.topk(x[0, part].double() @ router.double().T, 2, -1)
        assert torch.equal(chosen[0, part].long(), expected.indices)
        gates_close(gates[0, part], torch.softmax(expected.values, -1).cpu())


def test_equal_logits_and_experts_taken_out(device):
    x, router, _, _ = layer(1, 4, 64, 12, 8, FP32)
    router[3] = router[7] = router[1]  # equal whatever the token
    expected = check_route(device, x, router, 12)
    assert len(set(expected[0][0, 0].tolist())) == 12
    bias = torch.zeros(12)
    bias[[0, 2, 4, 5, 6, 8, 9, 10, 11]] = -INF  # 1, 3 and 7 are left, all equal
    chosen, _ = check_route(device, x, router, 5, bias)
    assert chosen[0, 0].tolist() == [1, 3, 7, -1, -1]
    check_route(device, x, router, 5, torch.full((12,), -INF))
    check_route(device, torch.zeros_like(x), router, 5)  # all logits 0 (or -0)
    check_route(device, -0.0 * x, router, 5)


def test_near_equal_logits_are_ranked_in_64_bits(device):
    # logits 1 + e 2^-40 of experts e: FP32 sums would call all of them equal
    E, D = 20, 64
    x, router = torch.zeros(1, 1, D), torch.zeros(E, D)
    x[0, 0, 0], x[0, 0, 63] = 1.0, 2.0 ** -40
    router[:, 0], router[:, 63] = 1.0, torch.arange(E).float()
    chosen, _ = check_route(device, x, router, 6)
    assert chosen[0, 0].tolist() == [19, 18, 17, 16, 15, 14]


def test_nan_and_infinite_logits(device):
    x, router, gate_up, down = layer(1, 3, 64, 6, 32, FP32)
    router[2, 5], router[4, 6] = NAN, INF
    x[0, 1, 6] = 0.0  # inf * 0
    chosen, gates = experts.route(x.to(device), router.to(device), 3)
    assert chosen[0, :, 0].tolist() == [2, 2, 2] and bool(gates.isnan().all())
    assert chosen[0, 1, 1].item() == 4
    # a row that holds a NaN is NaN, the rows beside it are not touched
    x, router, gate_up, down = layer(1, 5, 64, 6, 32, BF16)
    weights = experts.ExpertWeights(gate_up.to(device), down.to(device))
    whole, _, _ = experts.mixture(x.to(device), router.to(device), weights, 6)
    x[0, 2, 63] = NAN
    y, _, _ = experts.mixture(x.to(device), router.to(device), weights, 6)
    assert bool(y[0, 2].isnan().all())
    keep = [0, 1, 3, 4]
    assert torch.equal(y[0, keep], whole[0, keep])


@pytest.mark.parametrize("B, T, D, E, k", [
    (160, 1, 256, 128, 8), (9, 1, 2048, 16, 2), (3, 1, 64, 500, 4), (3, 2, 64, 130, 3), (1025, 1, 16, 5, 2),
    (1024, 1, 8, 5, 2), (2, 300, 512, 64, 4)])
def test_the_router_s_forms_meet(device, B, T, D, E, k):
    print(f"route B={B} T={T} D={D} E={E} k={k}", flush=True)
    x, router, _, _ = layer(B, T, D, E, 8, BF16, seed=D + E)
    check_route(device, x, router, k, torch.linspace(-1, 1, E))


# long features over few rows of outputs: the down product's columns are cut
@pytest.mark.parametrize("B, T, D, E, k, F, dtype", [
    (1, 1, 40, 16, 2, 1200, BF16), (1, 1, 40, 16, 2, 1200, FP32),  # fewer pairs than experts
    (4, 4, 136, 3, 2, 2100, BF16), (1, 1, 280, 2, 2, 1111, FP32),  # up to 16 rows
    (6, 5, 96, 4, 1, 2500, BF16), (20, 4, 72, 4, 2, 1111, FP32),   # few rows an expert, more of them
    (3, 40, 256, 64, 2, 1050, BF16), (64, 16, 512, 4, 2, 1041, BF16), (64, 16, 1024, 4, 2, 530, FP32)])
def test_long_features_are_cut_and_joined(device, B, T, D, E, k, F, dtype):
    print(f"mixture B={B} T={T} D={D} E={E} k={k} F={F} {dtype}", flush=True)
    x, router, gate_up, down = layer(B, T, D, E, F, dtype, seed=D + F)
    counts = torch.arange(B) % (T + 1)
    counts[0] = T
    weights, on, (y, _, _) = check_mixture(device, x, router, gate_up, down, k, None, counts)
    again, _, _ = experts.mixture(on[0], on[1], weights, k, None, on[3])
    assert torch.equal(again, y)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("B, T, D, E, k, F", [
    (1, 1, 8, 1, 1, 1), (1, 1, 64, 8, 2, 32), (1, 1, 40, 8, 8, 33), (3, 1, 256, 16, 2, 100),   # fewer pairs than experts
    (4, 4, 136, 3, 2, 48), (16, 1, 264, 8, 2, 15),                                           # up to 16 rows
    (5, 5, 72, 11, 3, 50), (8, 5, 96, 40, 8, 31), (2, 60, 64, 16, 2, 64),                     # few rows an expert
    (33, 3, 72, 4, 3, 40), (2, 64, 48, 2, 1, 16), (20, 16, 64, 5, 2, 80), (7, 11, 520, 1, 1, 17)])
def test_a_layer_is_the_gated_sum_of_its_experts(device, B, T, D, E, k, F, dtype):
    print(f"mixture B={B} T={T} D={D} E={E} k={k} F={F} {dtype}", flush=True)
    x, router, gate_up, down = layer(B, T, D, E, F, dtype, seed=D + F)
    g = torch.Generator().manual_seed(2)
    counts = torch.randint(0, T + 1, (B,), generator=g) if B > 1 else None
    check_mixture(device, x, router, gate_up, down, k, 0.3 * torch.randn(E, generator=g), counts)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_many_pairs_are_taken_range_by_range(device, dtype):
    # 2100 tokens of 4 choices: three ranges of pairs, several tiles an expert, one expert far ahead; few row blocks
    # and (E times 512 features) many
    x, router, gate_up, down = layer(3, 700, 32, 6, 16, dtype)
    router[2] += 0.5 * x.float().mean((0, 1))
    check_mixture(device, x, router, gate_up, down, 4, torch.tensor([0.0, 0.0, 5.0, 0.0, 0.0, 0.0]))


@pytest.mark.parametrize("rows, k", [(150, 2), (256, 8), (600, 8)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_tiles_of_tokens_of_many_row_blocks(device, rows, k, dtype):
    # 64 x 512 features, 64 x 1040 outputs: the products over tiles, in one range of pairs and in two, against torch in
    # 64 bits on the GPU within the oracle's bound of one token, taken as the largest
    E, D, F = 64, 1040, 512
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(1, rows, D, generator=g, device=device).to(dtype)
    router = torch.randn(E, D, generator=g, device=device) * D ** -0.5
    gate_up = (torch.randn(E, 2 * F, D, generator=g, device=device) * D ** -0.5).to(dtype)
    down = (torch.randn(E, D, F, generator=g, device=device) * F ** -0.5).to(dtype)
    bias = torch.zeros(E, device=device)
    bias[3] = 2.0  # one expert with several tiles
    weights = experts.ExpertWeights(gate_up, down)
    y, chosen, gates = experts.mixture(x, router, weights, k, bias)
    expected = torch.zeros(rows, D, dtype=torch.float64, device=device)
    for e in range(E):
        token, slot = (chosen[0] == e).nonzero(as_tuple=True)
        h = x[0, token].double() @ gate_up[e].double().T
        act = torch.nn.functional.silu(h[:, :F]) * h[:, F:]
        expected[token] += gates[0, token, slot, None].double() * (act @ down[e].double().T)
    assert int((chosen == 3).sum()) > 64  # more than a tile
    worst = 0.0
    for m in (0, rows // 2, rows - 1):
        _, bound = oracle.feed_forward(x[:, m:m + 1].cpu(), gate_up.cpu(), down.cpu(), chosen[:, m:m + 1].cpu(),
                                       gates[:, m:m + 1].cpu())
        worst = max(worst, float(bound.max()))
    assert float((y[0].double() - expected).abs().max()) <= 2 * worst
    parts, again, _ = experts.mixture_parts(x, router, weights, k, bias)
    assert torch.equal(again, chosen)
    assert float((parts.double().sum(0) - expected).abs().max()) <= 2 * worst


def test_one_expert_may_take_every_row_and_another_none(device):
    for rows in (15, 70, 200):
        x, router, gate_up, down = layer(rows, 1, 64, 9, 40, BF16, seed=rows)
        bias = torch.full((9,), -INF)
        bias[5] = 0.0
        _, _, (_, chosen, gates) = check_mixture(device, x, router, gate_up, down, 2, bias)
        assert chosen[..., 0].unique().tolist() == [5] and chosen[..., 1].unique().tolist() == [-1]


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_fewer_pairs_than_experts_all_of_one(device, dtype):
    # several tiles of an expert that is served by its first pair's workgroups
    for rows, k, E in ((60, 1, 64), (100, 2, 300), (511, 1, 512)):
        x, router, gate_up, down = layer(rows, 1, 72, E, 24, dtype, seed=rows)
        weights = experts.ExpertWeights(gate_up.to(device), down.to(device))
        chosen = torch.full((rows, 1, k), E // 2, dtype=torch.int32)
        chosen[rows // 3, 0, 0], chosen[rows // 2, 0, k - 1] = 5, -1
        gates = torch.rand(rows, 1, k, generator=torch.Generator().manual_seed(1))
        expected = oracle.feed_forward(x, gate_up, down, chosen, gates)
        on = [t.to(device) for t in (x, chosen, gates)]
        for _ in range(3):
            y_close(experts.feed_forward(on[0], weights, on[1], on[2]), expected, dtype)
            parts = experts.feed_forward_parts(on[0], weights, on[1], on[2])
            assert bool(((parts.double().sum(0).cpu() - expected[0].view(rows, -1)).abs() <= expected[1].view(rows, -1)).all())


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_given_choices_may_repeat_an_expert_or_name_none(device, rows):
    x, _, gate_up, down = layer(1, rows, 64, 7, 24, BF16)
    weights = experts.ExpertWeights(gate_up.to(device), down.to(device))
    g = torch.Generator().manual_seed(3)
    chosen = torch.randint(-1, 8, (1, rows, 3), generator=g, dtype=torch.int32)
    chosen[0, 0] = torch.tensor([4, 4, 7])
    chosen[0, -1] = -1
    if rows > 1:
        chosen[0, 1] = torch.tensor([2147483647, -2147483648, 3])
    gates = torch.randn(1, rows, 3, generator=g)
    expected = oracle.feed_forward(x, gate_up, down, chosen, gates)
    on = [t.to(device) for t in (x, chosen, gates)]
    y_close(experts.feed_forward(on[0], weights, on[1], on[2]), expected, BF16)
    parts = experts.feed_forward_parts(on[0], weights, on[1], on[2])
    assert parts.shape == (3, rows, 64) and parts.dtype == FP32
    y, bound = expected
    assert bool(((parts.double().sum(0).cpu() - y[0]).abs() <= bound[0]).all())
    assert bool((parts[:, -1] == 0).all())


def test_parts_are_terms_of_the_same_call(device):
    x, router, gate_up, down = layer(4, 5, 64, 16, 32, BF16)
    weights, on, (y, chosen, gates) = check_mixture(device, x, router, gate_up, down, 4)
    parts, c, g = experts.mixture_parts(on[0], on[1], weights, 4)
    total = parts[0].clone()
    for part in parts[1:]:
        total += part
    assert torch.equal(c, chosen) and torch.equal(g, gates)
    assert torch.equal(total.to(BF16).view_as(y), y)
    assert torch.equal(experts.feed_forward(on[0], weights, chosen, gates), y)


def test_a_row_s_bits_do_not_depend_on_the_rows_beside_it_in_its_tile(device):
    # the sums of one token run over the columns alone
    x, router, gate_up, down = layer(1, 200, 96, 4, 48, BF16)
    weights = experts.ExpertWeights(gate_up.to(device), down.to(device))
    whole, _, _ = experts.mixture(x.to(device), router.to(device), weights, 2)
    order = torch.randperm(200, generator=torch.Generator().manual_seed(0))
    moved, _, _ = experts.mixture(x[:, order].to(device), router.to(device), weights, 2)
    assert torch.equal(moved.cpu(), whole.cpu()[:, order])


def test_strided_inputs_and_empty_batches(device):
    x, router, gate_up, down = layer(3, 4, 64, 5, 20, BF16)
    weights, on, (y, chosen, gates) = check_mixture(device, x, router, gate_up, down, 2)
    wide = torch.zeros(3, 4, 69, dtype=BF16, device=device)
    wide[..., 5:] = on[0]
    odd = torch.empty(3 * 4 * 64 + 1, dtype=BF16, device=device)[1:].view(3, 4, 64)
    odd.copy_(on[0])
    for view in (wide[..., 5:], on[0].transpose(0, 1).contiguous().transpose(0, 1), odd):
        got = experts.mixture(view, on[1], weights, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, (y, chosen, gates)))
    routers = torch.zeros(64, 5, device=device)
    routers.copy_(on[1].T)
    assert torch.equal(experts.mixture(on[0], routers.T, weights, 2)[0], y)
    for shape in ((0, 4, 64), (3, 0, 64)):
        empty = torch.empty(*shape, dtype=BF16, device=device)
        y0, c0, g0 = experts.mixture(empty, on[1], weights, 2)
        assert y0.shape == shape and c0.shape == shape[:2] + (2,) and g0.shape == c0.shape


def test_what_does_not_match_is_refused(device):
    x, router, gate_up, down = (t.to(device) for t in layer(1, 2, 64, 5, 20, BF16))
    weights = experts.ExpertWeights(gate_up, down)
    chosen, gates = experts.route(x, router, 2)
    for call in (lambda: experts.route(x, router.double(), 2), lambda: experts.route(x, router[:, :32], 2),
                 lambda: experts.route(x, router, 6), lambda: experts.route(x, router, 0),
                 lambda: experts.route(x, router, 2, torch.zeros(4, device=device)),
                 lambda: experts.route(x, router, 2, None, torch.zeros(2, dtype=torch.long, device=device)),
                 lambda: experts.route(x, router, 2, None, torch.ones(1, device=device)),
                 lambda: experts.mixture(x, router[:4], weights, 2), lambda: experts.mixture(x.float(), router, weights, 2),
                 lambda: experts.feed_forward(x, weights, chosen.long(), gates),
                 lambda: experts.feed_forward(x, weights, chosen, gates[..., :1]),
                 lambda: experts.feed_forward(x, weights, chosen[..., :0], gates[..., :0]),
                 lambda: experts.route(x, router.cpu(), 2)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        experts.route(x[..., :20].contiguous(), router[:, :20].contiguous(), 2)
    with pytest.raises(NotImplementedError):
        experts.mixture(x.requires_grad_(), router, weights, 2)[0].sum().backward()


def test_a_captured_layer_replays_on_new_inputs_and_beside_another_stream(device):
    x, router, gate_up, down = (t.to(device) for t in layer(8, 5, 128, 16, 96, BF16))
    other = layer(8, 5, 128, 16, 96, BF16, seed=9)[0].to(device)
    weights = experts.ExpertWeights(gate_up, down)
    eager = [experts.mixture(t, router, weights, 4) for t in (x, other)]
    held = x.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        experts.mixture(held, router, weights, 4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = experts.mixture(held, router, weights, 4)
    torch.cuda.current_stream().wait_stream(stream)
    for i in (0, 1, 0, 1):
        held.copy_(x if i == 0 else other)
        graph.replay()
        beside = experts.mixture(other, router, weights, 4)  # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(beside, eager[1]))
    # two streams at once
    with torch.cuda.stream(stream):
        first = [experts.mixture(x, router, weights, 4) for _ in range(5)]
    second = [experts.mixture(other, router, weights, 4) for _ in range(5)]
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a[0], eager[0][0]) and torch.equal(b[0], eager[1][0])


def test_no_gradient_is_lost_in_silence(device):
    x, router, gate_up, down = (t.to(device) for t in layer(1, 3, 64, 8, 32, FP32))
    weights = experts.ExpertWeights(gate_up, down)
    with torch.no_grad():
        chosen, gates = experts.route(x, router, 2)
    x.requires_grad_()
    trained = experts.ExpertWeights(gate_up.requires_grad_(), down)
    for out in (experts.mixture_parts(x, router, weights, 2)[0], experts.feed_forward_parts(x, weights, chosen, gates),
                experts.mixture(x.detach(), router, trained, 2)[0],
                experts.feed_forward(x.detach(), trained, chosen, gates)):
        with pytest.raises(NotImplementedError):
            out.sum().backward()
    with torch.no_grad():
        assert not experts.mixture(x, router, trained, 2)[0].requires_grad
