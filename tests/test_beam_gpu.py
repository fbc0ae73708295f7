"""Beam search's selection (wptv_beam_step) and the reordering of states
(wptv_reorder_rows) against the plain 64-bit definitions.

Parents, tokens and ends are equal: both sides rank in 64 bits.  The totals:
one rounding to FP32, half a step (2^-24 of the value), and the error of
L = log sum exp x, whose terms exp(x - max) are FP32: the argument's rounding
adds 2^-24 |x - max| to a term, weighted by the terms at most log V (their
entropy), the exponential itself at most 2 steps of 2^-23, the FP32 parts of
the sum at most 64 additions of 2^-24."""

import math

import pytest
import torch

from oracle import beam as oracle
from wpt_amd import kernels, sampling

pytestmark = pytest.mark.gpu
INF = math.inf


def totals_close(got, expected, V):
    expected = expected.double()
    finite = torch.isfinite(expected)
    assert torch.equal(torch.isfinite(got), finite)
    assert bool((got[~finite] == -INF).all())
    bound = (expected.abs() + math.log(V) + 4 + 64) * 2.0 ** -24
    assert bool(((got.double() - expected).abs()[finite] <= bound[finite]).all())


def check(device, scores, totals, ended=None, stops=(), beams=None):
    on = [None if x is None else x.to(device) for x in (scores, totals, ended)]
    got = [x.cpu() for x in sampling.beam_step(*on, stops=stops, beams=beams)]
    expected = oracle.beam_step(scores, totals, ended, stops, beams)
    assert got[0].dtype == torch.float32 and got[3].dtype == torch.bool
    for name, a, b in zip(("parents", "tokens", "ended"), got[1:], expected[1:]):
        assert torch.equal(a, b), name
    totals_close(got[0], expected[0], scores.shape[-1])
    return got


def inputs(n, W, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    scores = (3 * torch.randn(n, W, V, generator=g)).to(dtype)
    totals = -30 * torch.rand(n, W, generator=g)
    return scores, totals, torch.rand(n, W, generator=g) < 0.2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, W, V, K", [
    (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 8), (1, 2, 40, 64), (1, 4, 8192, 4), (3, 8, 32768, 8), (2, 16, 50257, 16),
    (1, 64, 300, 64), (4, 5, 1001, 5), (1, 1, 131073, 32), (1, 64, 4099, 64), (40, 3, 4095, 3), (2, 1, 32768, 64),
    (300, 2, 1024, 2), (1, 7, 4097, 1), (256, 2, 2049, 2), (257, 2, 2049, 2), (3, 8, 4096, 8),
    (3, 8, 4097, 8), (5, 9, 100, 9), (1, 1, 32768, 64), (2, 8, 17, 64), (2, 16, 2000, 16)])
def test_the_next_beams_are_those_of_the_sorted_candidates(device, n, W, V, K, dtype):
    print(f"beam_step n={n} W={W} V={V} K={K} {dtype}", flush=True)
    scores, totals, ended = inputs(n, W, V, dtype, seed=n + W + V)
    check(device, scores, totals, beams=K)
    check(device, scores, totals, ended, stops=(V // 2,), beams=K)


@pytest.mark.parametrize("V", [5, 700, 33000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few values", "zeros", "one high", "last"])
def test_ties_and_sorted_scores(device, kind, V):
    n, W = 2, 3
    g = torch.Generator().manual_seed(V)
    ramp = torch.arange(V, dtype=torch.float32) / 64
    scores = {"equal": torch.full((V,), 1.5), "rising": ramp, "falling": -ramp,
              "few values": torch.randint(0, 3, (V,), generator=g).float(),
              "zeros": torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0),
              "one high": torch.where(torch.arange(V) == V // 3, 9.0, 0.0),
              "last": torch.where(torch.arange(V) >= V - 2, 9.0, 0.0)}[kind].expand(n, W, V).contiguous()
    for dtype in (torch.float32, torch.bfloat16):
        for K in (1, 3, 15, 64):
            if K > W * V:
                continue
            print(f"beam_step {kind} V={V} K={K} {dtype}", flush=True)
            # equal totals: equal beams tie with each other; distinct ones do not
            check(device, scores.to(dtype), torch.full((n, W), -2.5), beams=K)
            check(device, scores.to(dtype), torch.tensor([[-1.0, -2.0, -3.0], [-9.0, -2.0, -2.0]]), beams=K)


def test_beams_that_cannot_go_on(device):
    n, W, V = 7, 4, 900
    scores, totals, ended = inputs(n, W, V, torch.float32, seed=3)
    totals[0, 1:] = -INF  # a text's start: one beam
    totals[1] = torch.tensor([INF, math.nan, -4.0, -INF])
    scores[2, 1, 77] = math.nan
    scores[2, 2, 5] = INF
    scores[2, 3] = -INF
    scores[3] = -INF  # nothing in the whole text
    scores[4, :, 3:] = -INF  # three tokens a beam
    ended[5] = True  # every beam has ended: they go on as they are
    totals[6] = -INF
    ended[6] = torch.tensor([True, False, True, False])
    for K in (1, 4, 13):
        print(f"beam_step dead beams K={K}", flush=True)
        check(device, scores, totals, ended, stops=(11, 0), beams=K)
        check(device, scores.to(torch.bfloat16), totals, ended, stops=(899,), beams=K)


@pytest.mark.parametrize("offset", [-30000.0, -900.0, 900.0, 30000.0])
def test_scores_far_from_zero_with_masked_stretches(device, offset):
    scores, totals, ended = inputs(2, 3, 13000, torch.float32, seed=6)
    scores += offset
    scores[0, :, :9000] = -INF  # whole stretches of the vocabulary
    scores[1, 1, 4096:8192] = -INF
    scores[1, 2, 5:] = -INF
    check(device, scores, totals, ended, stops=(3,), beams=6)


def test_ended_beams_of_a_small_vocabulary(device):
    for V, K in ((1, 2), (2, 4), (3, 6)):
        scores, totals, _ = inputs(2, 2, V, torch.float32, seed=V)
        check(device, scores, totals, torch.tensor([[True, False], [True, True]]), stops=(V - 1,), beams=K)


def test_strided_scores_and_totals(device):
    g = torch.Generator().manual_seed(8)
    whole = torch.randn(3, 5, 4, 1003, generator=g)  # the last position of a reading of 4
    totals = torch.randn(5, 3, generator=g).T
    got = [x.cpu() for x in sampling.beam_step(whole.to(device)[:, :, -1], totals.to(device))]
    expected = oracle.beam_step(whole[:, :, -1], totals)
    assert torch.equal(got[1], expected[1]) and torch.equal(got[2], expected[2])
    odd = torch.randn(2, 3, 1500, generator=g).to(torch.bfloat16)
    got = [x.cpu() for x in sampling.beam_step(odd.to(device)[..., 1:1400], totals.to(device)[:2, :3])]
    expected = oracle.beam_step(odd[..., 1:1400], totals[:2, :3])
    assert torch.equal(got[1], expected[1]) and torch.equal(got[2], expected[2])


def test_scores_past_4_gb(device):
    n, W, V = 1100, 16, 131072  # 4.6 GB of bf16: the last texts lie past 2^31 elements
    scores = torch.empty(n, W, V, dtype=torch.bfloat16, device=device)
    for first in range(0, n, 100):
        scores[first:first + 100].normal_(std=3)
    totals = -20 * torch.rand(n, W, device=device)
    got = [x[[0, -1]].cpu() for x in sampling.beam_step(scores, totals)]
    expected = oracle.beam_step(scores[[0, -1]].cpu(), totals[[0, -1]].cpu())
    for a, b in zip(got[1:], expected[1:]):
        assert torch.equal(a, b)
    totals_close(got[0], expected[0], V)


def test_no_texts(device):
    got = sampling.beam_step(torch.empty(0, 3, 10, device=device), torch.empty(0, 3, device=device))
    assert [tuple(x.shape) for x in got] == [(0, 3)] * 4


# ---- reorder_rows ----------------------------------------------------------------


def fill(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 100, shape, generator=g).to(dtype)


@pytest.mark.parametrize("n, W", [(1, 1), (1, 2), (3, 4), (2, 5), (2, 8), (1, 16), (2, 17), (1, 64), (37, 3)])
@pytest.mark.parametrize("ragged", [False, True])
def test_every_beam_takes_over_its_parent(device, n, W, ragged):
    print(f"reorder_rows n={n} W={W} ragged={ragged}", flush=True)
    R, N = n * W, 45
    g = torch.Generator().manual_seed(n * W)
    lengths = torch.randint(0, N + 5, (R,), generator=g) if ragged else None
    shapes = [((R, N, 128), torch.bfloat16), ((R, 16, 256), torch.bfloat16), ((R, N, 1), torch.float32),
              ((R, N, 6), torch.bfloat16), ((R, 7, 3), torch.uint8), ((R, N, 5), torch.bfloat16), ((R, 1, 1), torch.long),
              ((R, N, 24), torch.float32)]
    tables = [fill(*s, seed=i) for i, s in enumerate(shapes)]
    for parents in (torch.randint(0, W, (n, W), generator=g),                       # some beams several times
                    torch.stack([torch.randperm(W, generator=g) for _ in range(n)]),  # cycles
                    torch.arange(W).expand(n, W).contiguous(),                      # nothing moves
                    torch.zeros(n, W, dtype=torch.long),
                    torch.randint(-2, W + 2, (n, W), generator=g)):                 # some that are no beams
        expected = oracle.reorder_rows(tables, parents, lengths)
        got = [t.to(device) for t in tables]
        kernels.reorder_rows(got, parents.to(device), None if lengths is None else lengths.to(device))
        for a, b in zip(got, expected):
            assert torch.equal(a.cpu(), b)


def test_tables_that_are_views_and_more_than_one_launch_of_them(device):
    n, W, N = 2, 3, 9
    g = torch.Generator().manual_seed(1)
    parents = torch.randint(0, W, (n, W), generator=g)
    whole = fill((40, n * W, N + 3, 40), torch.bfloat16, 1)
    moved = whole.to(device)
    kernels.reorder_rows(list(moved[:, :, 1:N + 1, 8:24].unbind(0)), parents.to(device))
    expected = whole.clone()
    expected[:, :, 1:N + 1, 8:24] = torch.stack(oracle.reorder_rows(list(whole[:, :, 1:N + 1, 8:24].unbind(0)), parents))
    assert torch.equal(moved.cpu(), expected)
    rows_first = fill((N, n * W, 16), torch.float32, 2)  # token rows outermost
    moved = rows_first.to(device)
    kernels.reorder_rows(moved.transpose(0, 1), parents.to(device))
    assert torch.equal(moved.cpu().transpose(0, 1), oracle.reorder_rows([rows_first.transpose(0, 1)], parents)[0])


def test_rows_past_the_bound_keep_their_values(device):
    table = fill((2, 50, 8), torch.float32, 3)
    moved = table.to(device)
    kernels.reorder_rows(moved, torch.tensor([[1, 0]], device=device), torch.tensor([20, 13], device=device), rows=20)
    expected = oracle.reorder_rows([table], torch.tensor([[1, 0]]), torch.tensor([20, 13]))[0]
    assert torch.equal(moved.cpu(), expected)


def test_a_table_past_4_gb(device):
    W, N, width = 3, 3000, 512  # 1.5 KB of 1-byte rows would do; the last batch row starts past 2^32 bytes
    stride = 1_500_000_000
    whole = torch.empty(2 * stride + N * width, dtype=torch.uint8, device=device)
    table = whole.as_strided((W, N, width), (stride, width, 1))
    small = fill((W, N, width), torch.uint8, 4)
    table.copy_(small)
    kernels.reorder_rows(table, torch.tensor([[2, 0, 1]], device=device))
    assert torch.equal(table.cpu(), oracle.reorder_rows([small], torch.tensor([[2, 0, 1]]))[0])


def test_on_another_stream_and_in_a_graph(device):
    n, W, V, N = 2, 4, 5003, 33
    scores, totals, ended = (x.to(device) for x in inputs(n, W, V, torch.bfloat16, seed=5))
    table = fill((n * W, N, 24), torch.bfloat16, 6).to(device)

    def step():
        t, p, v, e = sampling.beam_step(scores, totals, ended, stops=(4,))
        kernels.reorder_rows(table, p)
        return t, p, v, e

    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    before = table.clone()
    with torch.cuda.stream(stream):
        side = step()
    stream.synchronize()
    after = table.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        if i:  # new values in place; the first replay repeats the eager run
            scores.copy_(torch.randn(n, W, V, generator=g))
        table.copy_(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured] + [table.clone()]
        table.copy_(before)
        eager = list(step()) + [table]
        for a, b in zip(got, eager):
            assert torch.equal(a, b)
        if i == 0:
            for a, b in zip(got, list(side) + [after]):
                assert torch.equal(a, b)


# ---- values close to each other ----------------------------------------------------


def close_beams(n, W, V, dtype, seed):
    """Texts whose beams' best candidates are equal but for the rounding of the
    totals to FP32, some 1e-8 to 1e-7: the totals level the beams out."""
    g = torch.Generator().manual_seed(seed)
    scores = (3 * torch.randn(n, W, V, generator=g)).to(dtype)
    best = torch.log_softmax(scores.double(), -1).amax(-1)
    totals = (-2.5 - best).float()
    gaps = (totals.double() + best).sort(-1).values.diff(dim=-1)
    # far from 64 bits' own steps, and closer than FP32 sums tell apart
    assert float(gaps[gaps > 0].min()) > 1e-13 and float(gaps.max()) < 1e-6
    return scores, totals


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, W, V, K", [
    (48, 2, 4000, 1), (48, 2, 4000, 2), (48, 5, 1500, 3), (300, 2, 4000, 2), (600, 2, 4000, 1), (600, 2, 4000, 2),
    (40, 4, 33001, 4), (3, 16, 20000, 7), (2, 64, 5000, 64)])
def test_beams_closer_than_fp32_sums_tell_apart(device, n, W, V, K, dtype):
    print(f"beam_step close beams n={n} W={W} V={V} K={K} {dtype}", flush=True)
    scores, totals = close_beams(n, W, V, dtype, seed=n + K)
    check(device, scores, totals, beams=K)
    ended = torch.zeros(n, W, dtype=torch.bool)
    ended[:, 0] = True  # an ended beam's own total beside the others' values
    totals[:, 0] = -2.5
    check(device, scores, totals, ended, stops=(5,), beams=K)


def test_the_beams_of_a_text_do_not_depend_on_the_batch(device):
    scores, totals = close_beams(600, 2, 4000, torch.float32, seed=4)  # other parts of a beam at each size
    scores, totals = scores.to(device), totals.to(device)
    whole = sampling.beam_step(scores, totals)
    for n in (1, 64, 300):
        got = sampling.beam_step(scores[:n], totals[:n])
        for a, b in zip(got[1:], whole[1:]):
            assert torch.equal(a, b[:n])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, V", [(2, 40), (2, 700), (2, 33000), (400, 4100)])
@pytest.mark.parametrize("kind", ["rising", "falling", "mixed", "signs", "far total"])
def test_scores_apart_whose_values_are_equal(device, kind, n, V, dtype):
    """Scores so small, or totals so large, that 64 bits hold the values of many
    of a beam's scores as one: equal values fall to the lowest tokens."""
    W = 3
    g = torch.Generator().manual_seed(V)
    ramp = torch.arange(V, dtype=torch.float32) * 1e-20
    shuffled = ramp[torch.randperm(V, generator=g)]
    scores = {"rising": ramp, "falling": -ramp, "signs": torch.where(torch.rand(V, generator=g) < 0.5, shuffled, -shuffled),
              "mixed": torch.where(torch.rand(V, generator=g) < 4 / V, torch.rand(V, generator=g) + 1, shuffled),
              "far total": 1e-3 * torch.randn(V, generator=g)}[kind].expand(n, W, V).contiguous().to(dtype)
    totals = torch.tensor([-1.0, -2.5, -3.0] if kind != "far total" else [-1e30, -1.5e30, -1e30]).expand(n, W).contiguous()
    totals[0] = totals[0].flip(0)
    totals[1, 1] = totals[1, 0]
    some = slice(0, 3)  # of the larger batch, as many as plain loops read in time
    for K in (1, 3, 15, 64):
        print(f"beam_step {kind} n={n} V={V} K={K} {dtype}", flush=True)
        got = [x.cpu()[some] for x in sampling.beam_step(scores.to(device), totals.to(device), beams=K)]
        expected = oracle.beam_step(scores[some], totals[some], beams=K)
        assert torch.equal(got[1], expected[1]) and torch.equal(got[2], expected[2])
        totals_close(got[0], expected[0], V)


def test_batch_rows_past_4_gb(device):
    W, N, width = 3, 300, 512
    stride = 2_200_000_000  # the last batch row starts past 2^32 bytes
    whole = torch.empty(2 * stride + N * width, dtype=torch.uint8, device=device)
    table = whole.as_strided((W, N, width), (stride, width, 1))
    small = fill((W, N, width), torch.uint8, 5)
    table.copy_(small)
    lengths = torch.tensor([300, 120, 250])
    kernels.reorder_rows(table, torch.tensor([[2, 0, 1]], device=device), lengths.to(device))
    assert torch.equal(table.cpu(), oracle.reorder_rows([small], torch.tensor([[2, 0, 1]]), lengths)[0])


@pytest.mark.parametrize("n, W, V, K", [(3, 4, 3000, 16), (300, 8, 7, 9), (300, 3, 9001, 12), (2, 16, 30001, 64)])
def test_beams_of_the_same_scores_in_another_order(device, n, W, V, K):
    """Their log-sum-exp is one number, whatever the order of its terms: with
    equal totals equal scores fall to the lowest beam and token."""
    print(f"beam_step permuted beams n={n} W={W} V={V} K={K}", flush=True)
    g = torch.Generator().manual_seed(V)
    scores = torch.empty(n, W, V)
    for i in range(n):
        row = 2 * torch.randn(V, generator=g)
        scores[i] = torch.stack([row[torch.randperm(V, generator=g)] for _ in range(W)])
    got = [x.cpu() for x in sampling.beam_step(scores.to(device), torch.full((n, W), -2.5, device=device), beams=K)]
    order = scores.view(n, W * V).sort(dim=-1, descending=True, stable=True).indices[:, :K]
    assert torch.equal(got[1], order // V) and torch.equal(got[2], order % V)
