"""The accumulated attention weights (wptv_attention_weights), the choice of
the rows to keep (wptv_choose_kept) and their move (wptv_keep_rows) against
the plain 64-bit definitions.

The lists and the moved rows are equal.  A weight is a sum of terms
exp(scale q . k - lse); each term's argument is off by the FP32 sum of c
products, at most c 2^-24 scale |q| |k|, by the rounding of the scale and of
lse in the base-2 exponent, each at most 2^-23 of its size, and the term by
its exponential, at most 2 steps of 2^-23; the sum of R terms of one sign in
FP32 adds at most log2-many or, in turn, R roundings of 2^-24 of itself: 64
are allowed for, since a wavefront sums in blocks and R here is at most 4096
terms of mixed size (a sum in turn of R equal terms is off by R / 2 steps on a
random walk's square root: 64 at 4096)."""

import math

import pytest
import torch

from oracle import eviction as oracle
from wpt_amd import kernels

pytestmark = pytest.mark.gpu


def reading(B, T, H, c, N, dtype, seed, spare=0):
    """A reading of T tokens of B texts whose tables hold N rows (spare of them
    unused): q, the table, positions, lse, start."""
    g = torch.Generator().manual_seed(seed)
    q = torch.nn.functional.normalize(torch.randn(B, T, H, c, generator=g), dim=-1) * c ** 0.5
    table = torch.randn(B, N, 2 * c, generator=g)
    table[..., :c] = torch.nn.functional.normalize(table[..., :c], dim=-1) * c ** 0.5
    q, table = q.to(dtype), table.to(dtype)
    start = torch.randint(0, N - T - spare + 1, (B,), generator=g)
    start[0] = N - T - spare
    positions = start[:, None] + torch.arange(T)
    lse = oracle.log_sum_exp(q, table[..., :c], positions, c ** -0.5).float()
    return q, table, positions, lse, start


def close(got, expected, old, q, k, lse, scale):
    size = float(q.double().norm(dim=-1).max() * k.double().nan_to_num(0).norm(dim=-1).max()) * scale
    steps = q.shape[-1] * size / 2 + 2 * size + 2 * float(lse.double().abs().nan_to_num(0, 0, 0).max()) + 4 + 64
    bound = (expected.abs() * steps + old.double().abs()) * 2.0 ** -24
    off = (got.double() - expected).abs()
    assert bool((off <= bound).all()), float((off / expected.abs().clamp(min=1e-30)).max())


def check(device, q, table, positions, lse, weights, counts=None, start=None, splits=0):
    c = q.shape[-1]
    k = table[..., :c]
    expected = oracle.attention_weights(q, k, positions, lse, c ** -0.5, weights, counts, start)
    on = table.to(device)
    runs = []
    for _ in range(2):
        held = weights.to(device)
        got = kernels.add_attention_weights(q.to(device), on[..., :c], positions.to(device), lse.to(device), c ** -0.5,
                                            held, counts=None if counts is None else counts.to(device),
                                            start=None if start is None else start.to(device), splits=splits)
        assert got is held
        runs.append(held.cpu())
    assert torch.equal(*runs)  # the sums' order is fixed
    close(runs[0], expected, weights, q, k, lse, c ** -0.5)
    return runs[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B, T, H, c, N", [
    (1, 1, 1, 64, 1), (1, 1, 16, 128, 300), (3, 5, 16, 128, 517), (2, 7, 4, 64, 1029), (2, 3, 12, 128, 65),
    (1, 9, 32, 64, 255), (2, 1, 8, 64, 64), (1, 70, 16, 128, 70), (2, 130, 8, 64, 200), (1, 64, 16, 64, 1000),
    (2, 4, 3, 96, 130), (1, 2, 5, 33, 77), (5, 20, 16, 64, 129), (3, 21, 16, 128, 257), (70, 1, 4, 64, 4000), (1, 3, 2, 256, 100), (2, 33, 128, 64, 40), (1, 2, 200, 16, 30)])
def test_the_weights_of_a_reading(device, B, T, H, c, N, dtype):
    print(f"attention weights B={B} T={T} H={H} c={c} N={N} {dtype}", flush=True)
    q, table, positions, lse, start = reading(B, T, H, c, N, dtype, seed=B + T + H + N)
    g = torch.Generator().manual_seed(1)
    weights = 3 * torch.rand(B, N, generator=g)
    got = check(device, q, table, positions, lse, weights, start=start)
    # every query head gives weight 1 in all: the new weights sum to T H a text
    fresh = check(device, q, table, positions, lse, torch.zeros(B, N))
    assert torch.allclose(fresh.double().sum(1), torch.full((B,), float(T * H), dtype=torch.double), rtol=1e-3)
    counts = torch.randint(0, T + 1, (B,), generator=g)
    check(device, q, table, positions, lse, weights, counts=counts, start=start)


@pytest.mark.parametrize("T, H, c, N", [(300, 16, 128, 1100), (257, 4, 64, 257)])
@pytest.mark.parametrize("splits", [0, 1, 3, 7])
def test_the_queries_of_a_prompt_in_parts(device, T, H, c, N, splits):
    print(f"attention weights of a prompt T={T} H={H} c={c} N={N} splits={splits}", flush=True)
    for dtype in (torch.bfloat16, torch.float32):
        q, table, positions, lse, start = reading(2, T, H, c, N, dtype, seed=T)
        weights = torch.rand(2, N, generator=torch.Generator().manual_seed(2))
        check(device, q, table, positions, lse, weights, start=start, splits=splits)
        check(device, q, table, positions, lse, weights, counts=torch.tensor([T // 2, 0]), start=start, splits=splits)


@pytest.mark.parametrize("dtype, c", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64),
                                      (torch.float32, 128), (torch.bfloat16, 40)])
def test_nothing_unseen_reaches_the_weights(device, dtype, c):
    B, T, H, N, spare = 3, 6, 8, 150, 30
    q, table, positions, lse, start = reading(B, T, H, c, N, dtype, seed=9, spare=spare)
    counts = torch.tensor([T, 4, 0])
    weights = torch.rand(B, N, generator=torch.Generator().manual_seed(3))
    for b in range(B):
        table[b, int(positions[b, -1]) + 1:] = math.nan  # rows that no query sees
        table[b, :, c:] = math.inf  # the values are not read
        q[b, int(counts[b]):] = math.nan  # queries that are not counted
        lse[b, int(counts[b]):] = math.nan
        if counts[b] < T:
            table[b, int(positions[b, 0]) + int(counts[b]):] = math.nan
    got = check(device, q.nan_to_num(0), table.nan_to_num(0, 0, 0), positions, lse.nan_to_num(0), weights, counts, start)
    held = weights.to(device)
    kernels.add_attention_weights(q.to(device), table.to(device)[..., :c], positions.to(device), lse.to(device),
                                  c ** -0.5, held, counts=counts.to(device), start=start.to(device))
    assert torch.equal(held.cpu(), got)
    assert torch.equal(got[2], weights[2])  # nothing counted: untouched
    for b in range(2):
        assert torch.equal(got[b, int(start[b]) + int(counts[b]):], weights[b, int(start[b]) + int(counts[b]):])


def test_queries_that_see_nothing_or_past_the_table(device):
    B, T, H, c, N = 2, 4, 16, 128, 90
    q, table, positions, lse, start = reading(B, T, H, c, N, torch.bfloat16, seed=4)
    positions = torch.tensor([[-1, 3, 500, -7], [-1, -1, -1, -1]])
    lse = oracle.log_sum_exp(q, table[..., :c], positions, c ** -0.5).float()  # -inf where nothing is seen
    weights = torch.rand(B, N, generator=torch.Generator().manual_seed(5))
    got = check(device, q, table, positions, lse, weights)
    assert torch.equal(got[1], weights[1])


def test_strides_and_unaligned_tables(device):
    B, T, H, c, N = 2, 5, 16, 64, 140
    q, table, positions, lse, start = reading(B, T, H, c, N, torch.bfloat16, seed=6)
    weights = torch.rand(B, 2 * N, generator=torch.Generator().manual_seed(6))
    expected = oracle.attention_weights(q, table[..., :c], positions, lse, c ** -0.5, weights[:, 3:3 + N])
    wide = torch.zeros(B, N, 2 * c + 1, dtype=torch.bfloat16, device=device)  # rows of an odd stride
    wide[..., 1:1 + c] = table[..., :c].to(device)
    rows_first = table[..., :c].transpose(0, 1).contiguous().to(device).transpose(0, 1)
    for k in (wide[..., 1:1 + c], rows_first):
        held = weights.to(device)
        kernels.add_attention_weights(q.to(device).transpose(1, 2).contiguous().transpose(1, 2), k, positions.to(device),
                                      lse.to(device), c ** -0.5, held[:, 3:3 + N])
        close(held.cpu()[:, 3:3 + N], expected, weights[:, 3:3 + N], q, table[..., :c], lse, c ** -0.5)
        assert torch.equal(held.cpu()[:, :3], weights[:, :3]) and torch.equal(held.cpu()[:, 3 + N:], weights[:, 3 + N:])


def test_a_table_past_4_gb(device):
    T, H, c, N = 3, 16, 128, 200
    q, table, positions, lse, start = reading(2, T, H, c, N, torch.bfloat16, seed=7)
    stride = 40_000_000  # elements between rows: the last starts past 2^33 bytes
    whole = torch.empty(N * stride // 2, dtype=torch.bfloat16, device=device)
    k = whole.as_strided((1, N // 2, c), (0, stride, 1))
    k.copy_(table[:1, :N // 2, :c])
    positions = (N // 2 - T + torch.arange(T))[None]
    lse = oracle.log_sum_exp(q[:1], table[:1, :N // 2, :c], positions, c ** -0.5).float()
    expected = oracle.attention_weights(q[:1], table[:1, :N // 2, :c], positions, lse, c ** -0.5, torch.zeros(1, N // 2))
    held = torch.zeros(1, N // 2, device=device)
    kernels.add_attention_weights(q[:1].to(device), k, positions.to(device), lse.to(device), c ** -0.5, held)
    close(held.cpu(), expected, torch.zeros(1, N // 2), q, table[..., :c], lse, c ** -0.5)


# ---- choose_kept, keep_rows --------------------------------------------------------


def choose(device, weights, lengths, keep, first, recent):
    expected = oracle.choose_kept(weights, lengths, keep, first, recent)
    got = kernels.choose_kept(weights.to(device), lengths.to(device), keep, first, recent)
    assert torch.equal(got[0].cpu(), expected[0]) and torch.equal(got[1].cpu(), expected[1])
    return got


@pytest.mark.parametrize("L, B, N, keep, first, recent", [
    (1, 1, 1, 1, 0, 0), (2, 3, 40, 10, 2, 3), (1, 4, 300, 256, 4, 128), (3, 2, 1029, 200, 0, 0), (2, 2, 4100, 2048, 4, 128),
    (1, 3, 5000, 133, 4, 128), (1, 2, 257, 256, 0, 256), (2, 1, 100, 8, 8, 0), (1, 2, 9000, 8999, 1, 1),
    (1, 2, 20000, 3000, 4, 64), (1, 1, 70001, 40000, 0, 1), (2, 2, 30, 50, 4, 20)])
@pytest.mark.parametrize("kind", ["random", "equal", "few values", "special"])
def test_the_rows_kept(device, L, B, N, keep, first, recent, kind):
    print(f"choose_kept L={L} B={B} N={N} keep={keep} first={first} recent={recent} {kind}", flush=True)
    g = torch.Generator().manual_seed(N + keep)
    weights = 1 / (1e-4 + torch.rand(L, B, N, generator=g))
    if kind == "equal":
        weights.fill_(0.25)
    elif kind == "few values":
        weights = torch.randint(0, 3, (L, B, N), generator=g).float()
    elif kind == "special":
        pick = torch.randint(0, 8, (L, B, N), generator=g)
        values = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1.0, 2.0])
        weights = values[pick]
        weights[0, 0, ::7] = -math.nan  # a NaN with the sign bit set
    lengths = torch.randint(0, N + 1, (B,), generator=g)
    lengths[0] = N
    if B > 1:
        lengths[1] = min(keep + 1, N)
    choose(device, weights, lengths, keep, first, recent)


def test_lengths_outside_the_table_and_strided_weights(device):
    weights = torch.rand(2, 3, 60, generator=torch.Generator().manual_seed(1))
    choose(device, weights, torch.tensor([-5, 1000, 60]), 20, 1, 2)
    wide = torch.zeros(2, 3, 80, device=device)
    wide[..., 7:67] = weights.to(device)
    expected = oracle.choose_kept(weights, torch.tensor([60, 50, 21]), 20, 1, 2)
    for view in (wide[..., 7:67], weights.permute(2, 0, 1).contiguous().to(device).permute(1, 2, 0)):
        got = kernels.choose_kept(view, torch.tensor([60, 50, 21], device=device), 20, 1, 2)
        assert torch.equal(got[0].cpu(), expected[0]) and torch.equal(got[1].cpu(), expected[1])


@pytest.mark.parametrize("L, B, N, keep", [(1, 1, 2, 1), (2, 3, 40, 17), (1, 2, 1029, 700), (3, 1, 333, 300), (1, 5, 4100, 2049),
                                           (35, 2, 50, 20), (2, 40, 90, 31)])
def test_the_kept_rows_move_together(device, L, B, N, keep):
    print(f"keep_rows L={L} B={B} N={N} keep={keep}", flush=True)
    g = torch.Generator().manual_seed(N)
    weights = torch.rand(L, B, N, generator=g)
    lengths = torch.randint(0, N + 1, (B,), generator=g)
    lengths[0] = N
    kept, counts = choose(device, weights, lengths, keep, 0, keep // 3)
    for width, dtype in ((256, torch.bfloat16), (1, torch.float32), (5, torch.bfloat16), (3, torch.uint8), (33, torch.float32),
                         (128, torch.float32), (2, torch.long)):
        tables = [torch.randint(0, 100, (B, N, width), generator=g).to(dtype) for _ in range(2 * L if L < 5 else L)]
        expected = oracle.keep_rows(tables, kept.cpu(), counts.cpu())
        got = [t.to(device) for t in tables]
        kernels.keep_rows(got, kept, counts)
        for a, b in zip(got, expected):
            assert torch.equal(a.cpu(), b)


def test_tables_that_are_views_move_in_place(device):
    B, N, keep = 2, 70, 31
    g = torch.Generator().manual_seed(2)
    kept, counts = choose(device, torch.rand(1, B, N, generator=g), torch.tensor([N, 40]), keep, 2, 9)
    whole = torch.randint(0, 100, (B, N + 5, 48), generator=g).to(torch.bfloat16)
    moved = whole.to(device)
    kernels.keep_rows(moved[:, 2:N + 2, 8:40], kept, counts)
    expected = whole.clone()
    expected[:, 2:N + 2, 8:40] = oracle.keep_rows([whole[:, 2:N + 2, 8:40]], kept.cpu(), counts.cpu())[0]
    assert torch.equal(moved.cpu(), expected)
    rows_first = torch.randint(0, 100, (N, B, 16), generator=g).float()
    moved = rows_first.to(device)
    kernels.keep_rows(moved.transpose(0, 1), kept, counts)
    assert torch.equal(moved.cpu().transpose(0, 1),
                       oracle.keep_rows([rows_first.transpose(0, 1)], kept.cpu(), counts.cpu())[0])


def test_kept_rows_past_4_gb(device):
    B, N, width, keep = 3, 500, 512, 200
    kept, counts = choose(device, torch.rand(1, B, N, generator=torch.Generator().manual_seed(3)), torch.tensor([N] * B),
                          keep, 1, 5)
    stride = 2_200_000_000
    whole = torch.empty(2 * stride + N * width, dtype=torch.uint8, device=device)
    table = whole.as_strided((B, N, width), (stride, width, 1))
    small = torch.randint(0, 100, (B, N, width), generator=torch.Generator().manual_seed(4)).to(torch.uint8)
    table.copy_(small)
    kernels.keep_rows(table, kept, counts)
    assert torch.equal(table.cpu(), oracle.keep_rows([small], kept.cpu(), counts.cpu())[0])


def test_lists_that_name_no_row_move_nothing_out_of_range(device):
    table = torch.arange(20.0).view(1, 10, 2)
    kept = torch.tensor([[[0, 3, -1, 99, 7, 8]]])
    moved = table.to(device)
    kernels.keep_rows(moved, kept.to(device), torch.tensor([6], device=device))
    expected = table.clone()
    expected[0, 1], expected[0, 4], expected[0, 5] = table[0, 3], table[0, 7], table[0, 8]
    assert torch.equal(moved.cpu(), expected)


def test_a_list_that_names_a_row_twice(device):
    table = torch.randint(0, 100, (1, 3000, 8), generator=torch.Generator().manual_seed(1)).float()
    rows = torch.sort(torch.randint(0, 3000, (1, 1, 1400), generator=torch.Generator().manual_seed(2))).values
    rows = torch.maximum(rows, torch.arange(1400))  # not below their places
    moved = table.to(device)
    kernels.keep_rows(moved, rows.to(device), torch.tensor([1400], device=device))
    assert torch.equal(moved.cpu(), oracle.keep_rows([table], rows, torch.tensor([1400]))[0])


def test_two_streams_at_once(device):
    B, T, H, c, N, keep = 2, 40, 16, 64, 600, 200
    sets, streams = [], [torch.cuda.Stream(device) for _ in range(2)]
    for seed in range(2):
        q, table, positions, lse, start = (x.to(device) for x in reading(B, T, H, c, N, torch.bfloat16, seed=seed))
        sets.append((q, table, positions, lse, start, torch.rand(1, B, N, device=device)))

    def step(q, table, positions, lse, start, weights):
        table, weights = table.clone(), weights.clone()
        kernels.add_attention_weights(q, table[..., :c], positions, lse, c ** -0.5, weights[0], start=start)
        kept, counts = kernels.choose_kept(weights, positions[:, -1] + 1, keep, 2, 16)
        kernels.keep_rows(table, kept, counts)
        return weights, kept, table

    expected = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, expected[i]))


def test_in_a_graph_on_another_stream(device):
    L, B, T, H, c, N, keep = 2, 2, 3, 16, 128, 200, 64
    q, table, positions, lse, start = reading(B, T, H, c, N, torch.bfloat16, seed=8)
    table, q, positions, lse, start = (x.to(device) for x in (table, q, positions, lse, start))
    weights = torch.zeros(L, B, N, device=device)
    tables = [table.clone() for _ in range(L)]
    lengths = positions[:, -1] + 1

    def step():
        for i in range(L):
            kernels.add_attention_weights(q, tables[i][..., :c], positions, lse, c ** -0.5, weights[i], start=start)
        kept, counts = kernels.choose_kept(weights, lengths, keep, 2, 16)
        kernels.keep_rows(tables, kept, counts)
        return kept, counts

    def reset(seed):
        fresh = torch.rand(L, B, N, generator=torch.Generator().manual_seed(seed))
        weights.copy_(fresh)
        for t in tables:
            t.copy_(table)

    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    reset(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        side = [x.clone() for x in step()] + [weights.clone()] + [t.clone() for t in tables]
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        reset(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured] + [weights.clone()] + [t.clone() for t in tables]
        reset(i)
        eager = list(step()) + [weights] + tables
        for a, b in zip(got, eager):
            assert torch.equal(a, b)
        if i == 0:
            for a, b in zip(got, side):
                assert torch.equal(a, b)


@pytest.mark.parametrize("B, splits", [(13, 5), (11, 7), (67, 2)])
def test_parts_that_do_not_divide_over_the_xcds(device, B, splits):
    """64 chunks of a batch row and a part or more, and no multiple of 8."""
    assert B * splits >= 64 and B * splits % 8
    q, table, positions, lse, start = reading(B, 20, 16, 64, 300, torch.bfloat16, seed=B)
    weights = torch.rand(B, 300, generator=torch.Generator().manual_seed(B))
    check(device, q, table, positions, lse, weights, start=start, splits=splits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("c", [64, 128, 96])
def test_the_weights_to_their_last_bits(device, dtype, c):
    """Queries and keys of -1, 0 and 1 and a scale of 2^-4: the products are
    exact, so what is left of a term exp(s - lse) are, in steps of 2^-24, the
    rounding of log2 e (0.22) on |s|, with its product's (1.22) on |lse|, that of
    the difference on |s - lse|, the exponential's 2; and the sum's R additions of
    terms of one sign, no more than R / 4 + 8 in turn in any form, and the last."""
    B, T, H, N = 3, 5, 16, 420
    g = torch.Generator().manual_seed(c)
    q, k = (torch.randint(-1, 2, shape, generator=g).to(dtype) for shape in ((B, T, H, c), (B, N, c)))
    positions = torch.tensor([N - T, 200, 17])[:, None] + torch.arange(T)
    lse = oracle.log_sum_exp(q, k, positions, 2.0 ** -4).float()
    old = torch.zeros(B, N)
    expected = oracle.attention_weights(q, k, positions, lse, 2.0 ** -4, old)
    held = old.to(device)
    kernels.add_attention_weights(q.to(device), k.to(device), positions.to(device), lse.to(device), 2.0 ** -4, held)
    s = float((torch.matmul(q.float().reshape(B, T * H, c), k.float().transpose(1, 2)) * 2.0 ** -4).abs().max())
    high = float(lse.abs().max())
    steps = 0.22 * s + 1.22 * high + (s + high) + 2 + T * H / 4 + 8 + 1
    assert steps < 64
    assert bool(((held.cpu().double() - expected).abs() <= expected * steps * 2.0 ** -24).all())
