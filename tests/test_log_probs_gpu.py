"""The written tokens' log-probabilities (wptv_log_probs) against 64 bits.  The
alternatives are equal (ranked by the scores themselves); the values lie within
oracle.log_probs.bounds."""

import math

import pytest
import torch

from oracle import log_probs as oracle
from wpt_amd import sampling

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def close(got, expected, bound):
    same = torch.isnan(expected) == torch.isnan(got)
    finite = torch.isfinite(expected)
    assert bool(same.all()) and bool((got[expected == -INF] == -INF).all())
    assert bool(((got.double() - expected).abs()[finite] <= bound.expand_as(expected)[finite]).all())


def check(device, scores, tokens, top=0, temperature=1.0):
    got = [t.cpu() for t in sampling.log_probs(scores.to(device), tokens.to(device), top, temperature)]
    lp, entropy, ids, best = oracle.log_probs(scores, tokens, top, temperature)
    assert got[0].dtype == got[1].dtype == got[3].dtype == torch.float32 and got[2].dtype == torch.int64
    assert torch.equal(got[2], ids)
    one, slope, spread = oracle.bounds(scores, temperature)
    x = scores.double()
    high = x.amax(-1, keepdim=True)
    at = (x.gather(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None])[..., 0] - high[..., 0]).abs() / temperature
    close(got[0], lp, one + slope * at + 2.0 ** -24 * lp.abs())
    assert bool((got[0][(tokens < 0) | (tokens >= x.shape[-1])] == 0).all())
    close(got[1], entropy, spread + 2.0 ** -24 * entropy.abs())
    close(got[3], best, one[..., None] + slope * (x.gather(-1, ids) - high).abs() / temperature + 2.0 ** -24 * best.abs())
    return got


def inputs(B, T, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    scores = (3 * torch.randn(B, T, V, generator=g)).to(dtype)
    return scores, torch.randint(-1, V, (B, T), generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B, T, V, top", [
    (1, 1, 1, 1), (1, 1, 2, 0), (2, 3, 5, 5), (1, 2, 64, 64), (3, 1, 1000, 7), (1, 1, 8192, 5), (2, 2, 8191, 64),
    (2, 5, 32768, 20), (1, 3, 50257, 8), (1, 1, 131072, 32), (1, 1, 131075, 3), (1, 1, 300001, 64), (70, 4, 513, 2),
    (300, 1, 4099, 1), (2, 2, 65537, 0), (300, 1, 20000, 6), (260, 1, 40001, 3), (1, 2, 600001, 9), (1, 1, 1100003, 5),
    (40, 4, 32768, 2), (1, 1, 7, 7), (1, 3, 8, 8), (1, 2, 9, 4)])
def test_the_values_are_those_of_64_bits(device, B, T, V, top, dtype):
    print(f"log_probs B={B} T={T} V={V} top={top} {dtype}", flush=True)
    scores, tokens = inputs(B, T, V, dtype, seed=V + top)
    check(device, scores, tokens, top)
    check(device, scores, tokens, top, temperature=0.37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, V, top", [(300, 16385, 40), (300, 20480, 6), (300, 20481, 0), (300, 24583, 3), (3, 8200, 9),
                                          (300, 36864, 5), (300, 69633, 4),
                                          (300, 69633, 0), (260, 131073, 0)])
def test_rows_that_fill_a_workgroup_in_part(device, rows, V, top, dtype):
    print(f"log_probs rows={rows} V={V} top={top} {dtype}", flush=True)
    scores, tokens = inputs(rows, 1, V, dtype, seed=V)
    scores[1] = scores[1].round()  # many equal scores
    scores[2] = 1.0
    check(device, scores, tokens, top)


@pytest.mark.parametrize("V", [7, 100, 5000, 30000, 40000, 140000, 600000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_scores_fall_to_the_lowest_tokens(device, V, dtype):
    g = torch.Generator().manual_seed(V)
    few = torch.randint(0, 3, (2, 2, V), generator=g).to(dtype)  # three values, thousands of each
    few[0, 1] = 7.0
    few[1, 0] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    few[1, 1] = 0.0
    few[1, 1, V - 1] = 1.0
    check(device, few, torch.full((2, 2), V - 1), min(V, 40))


def test_banned_tokens_and_rows_without_a_distribution(device):
    for V in (90, 9000, 70000):
        scores, tokens = inputs(3, 4, V, torch.float32, seed=V)
        scores[0, 0, ::2] = -INF
        scores[0, 1] = -INF
        scores[0, 2, 17] = NAN
        scores[0, 3, 40], scores[0, 3, 3] = INF, INF
        scores[1, 0] = -INF
        scores[1, 0, V // 2] = -3.0  # one token is left
        scores[1, 1] = torch.finfo(torch.float32).min
        scores[1, 2, :] = -1e30
        scores[1, 2, 5] = 1e30
        scores[1, 3, 50:] = NAN
        scores[2, 0, 1:] = -INF
        scores[2, 1] = INF
        tokens[0, 0], tokens[1, 0], tokens[1, 2] = 2, V // 2, 6
        got = check(device, scores, tokens, 30)
        assert got[0][1, 0] == 0 and got[1][1, 0] == 0  # certain
        check(device, scores, tokens, 30, temperature=1.3)


def test_a_token_all_but_certain_keeps_its_digits(device):
    # 1 - p of 1e-9: far below a step of FP32 sums
    V = 1024
    scores = torch.full((1, 1, V), 0.0)
    scores[0, 0, 9] = math.log(1e9 * (V - 1))
    lp, entropy, _, _ = sampling.log_probs(scores.to(device), torch.tensor([[9]], device=device))
    expected = oracle.log_probs(scores, torch.tensor([[9]]))
    assert lp.item() == pytest.approx(expected[0].item(), rel=1e-4)
    assert entropy.item() == pytest.approx(expected[1].item(), rel=1e-4)


def test_a_row_cut_in_parts_joins_like_a_whole_one(device):
    # few long rows are read in parts: a part of banned tokens, the maximum in any part, a NaN in one
    V = 130000
    scores, tokens = inputs(6, 1, V, torch.bfloat16)
    scores[0, 0, :V // 2] = -INF
    scores[1, 0, 100:] = -INF
    scores[2, 0, 3], scores[3, 0, V - 1], scores[4, 0, V // 2] = 40.0, 60.0, 50.0
    scores[5, 0, V - 3] = NAN
    tokens[3, 0] = V - 1
    check(device, scores, tokens, 33)
    check(device, scores.float(), tokens, 64, temperature=0.7)


def test_strides_and_empty_batches(device):
    scores, tokens = inputs(3, 4, 1001, torch.bfloat16)
    whole = check(device, scores, tokens, 9)
    wide = torch.full((3, 4, 1013), 50.0, dtype=torch.bfloat16, device=device)
    wide[..., 7:1008] = scores.to(device)
    late = torch.zeros(3, 9, 1001, dtype=torch.bfloat16, device=device)
    late[:, 2:6] = scores.to(device)
    for view in (wide[..., 7:1008], late[:, 2:6], scores.transpose(1, 2).contiguous().to(device).transpose(1, 2),
                 scores.transpose(0, 1).contiguous().to(device).transpose(0, 1)):
        got = sampling.log_probs(view, tokens.to(device), 9)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, whole))
    got = sampling.log_probs(scores.to(device), tokens.T.contiguous().to(device).T, 9)
    assert torch.equal(got[0].cpu(), whole[0])
    for shape in ((0, 4), (3, 0)):
        got = sampling.log_probs(torch.empty(*shape, 50, device=device), torch.empty(*shape, dtype=torch.long, device=device), 3)
        assert got[0].shape == shape and got[2].shape == shape + (3,)


def test_rows_past_4_gb(device):
    # the last rows of a table of 4.3 GB
    V, T = 131072, 16400
    scores = torch.zeros(1, T, V, dtype=torch.bfloat16, device=device)
    scores[0, -1] = torch.randn(V, generator=torch.Generator().manual_seed(0)).to(device)
    tokens = torch.full((1, 2), 77, device=device)
    lp, _, ids, _ = sampling.log_probs(scores[:, -2:], tokens, 4)
    expected = oracle.log_probs(scores[:, -2:].cpu(), tokens.cpu(), 4)
    assert torch.equal(ids.cpu(), expected[2]) and torch.allclose(lp.cpu().double(), expected[0], atol=1e-5)
    whole = sampling.log_probs(scores, torch.full((1, T), 77, device=device), 4)
    assert torch.allclose(whole[0][:, -2:], lp, atol=1e-5) and torch.equal(whole[2][:, -2:], ids)


def test_what_does_not_match_is_refused(device):
    scores, tokens = (t.to(device) for t in inputs(2, 3, 50, torch.float32))
    for call in (lambda: sampling.log_probs(scores, tokens[:, :2]), lambda: sampling.log_probs(scores, tokens.int()),
                 lambda: sampling.log_probs(scores, tokens, 51), lambda: sampling.log_probs(scores, tokens, -1),
                 lambda: sampling.log_probs(scores, tokens, 2, 0.0), lambda: sampling.log_probs(scores, tokens, 2, INF),
                 lambda: sampling.log_probs(scores, tokens, 2, 1e-40), lambda: sampling.log_probs(scores, tokens.cpu()), lambda: sampling.log_probs(scores.half(), tokens)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        sampling.log_probs(torch.zeros(1, 1, 100, device=device), tokens[:1, :1], 65)


def test_captured_and_beside_another_stream(device):
    scores, tokens = (t.to(device) for t in inputs(4, 5, 9000, torch.bfloat16))
    other = inputs(4, 5, 9000, torch.bfloat16, seed=5)[0].to(device)
    eager = [sampling.log_probs(s, tokens, 12) for s in (scores, other)]
    held = scores.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sampling.log_probs(held, tokens, 12)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = sampling.log_probs(held, tokens, 12)
    torch.cuda.current_stream().wait_stream(stream)
    for i in (0, 1, 1, 0):
        held.copy_((scores, other)[i])
        graph.replay()
        beside = sampling.log_probs(other, tokens, 12)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(beside, eager[1]))
