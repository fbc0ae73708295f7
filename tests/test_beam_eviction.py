"""What the beam and eviction operators refuse, checked on the host before
anything is launched (no GPU is needed), and their 64-bit definitions on small
cases done by hand."""

import ctypes

import pytest
import torch

from oracle import beam as beam_oracle
from oracle import eviction as eviction_oracle
from wpt_amd import _lib, kernels, sampling

A = 1 << 20  # an address that is never read: every call here ends on the host


def message():
    return _lib.lib().wptv_last_error().decode()


def longs(*values):
    return (ctypes.c_int64 * len(values))(*values)


def beam(n=1, W=2, V=10, K=2, dtype=_lib.WPTV_F32, stops=(), ended=None, n_stops=None, size=1 << 20, scores=A):
    return _lib.lib().wptv_beam_step(scores, W * V, V, dtype, A, ended, longs(*stops), len(stops) if n_stops is None else
                                     n_stops, n, W, V, K, A, A, A, A, A, size, None)


@pytest.mark.parametrize("status, text, arguments", [
    (-1, "bad shape", {"n": -1}), (-1, "bad shape", {"W": 0}), (-1, "bad shape", {"V": 0}), (-1, "bad shape", {"K": 0}),
    (-1, "bad shape", {"K": 21}), (-3, "at most 64", {"W": 65}), (-3, "at most 64", {"W": 64, "K": 65}),
    (-3, "neither", {"dtype": 7}), (-1, "outside", {"stops": (10,)}), (-1, "outside", {"stops": (1, -1)}),
    (-1, "0 to 16", {"n_stops": 17}), (-1, "stop token", {"ended": A}), (-1, "workspace", {"V": 100000, "size": 8}),
    (-1, "NULL", {"scores": None}), (-3, "too large", {"n": 1 << 30, "W": 4})])
def test_beam_step_refuses(status, text, arguments):
    assert beam(**arguments) == status
    assert text in message()


def test_no_texts_is_no_work():
    assert beam(n=0) == 0


def reorder(base=A, sb=640, sn=64, capacity=10, row=64, count=1, n=1, W=2, parents=2 * A, lengths=None, rows=10):
    return _lib.lib().wptv_reorder_rows((ctypes.c_void_p * 1)(base), longs(sb), longs(sn), longs(capacity), longs(row), count,
                                        parents, lengths, rows, n, W, None)


@pytest.mark.parametrize("status, text, arguments", [
    (-1, "bad shape", {"W": 0}), (-1, "bad shape", {"n": -1}), (-1, "bad shape", {"rows": -1}), (-3, "at most 64", {"W": 65}),
    (-3, "65535", {"n": 65536}), (-1, "overlap", {"sn": 63}), (-1, "overlap", {"sb": 0}), (-1, "overlap", {"sb": 600}),
    (-1, "capacity", {"capacity": -1}), (-1, "capacity", {"row": 0}), (-1, "NULL", {"base": None}),
    (-1, "parents", {"parents": None}), (-1, "list of rows", {"parents": A}), (-1, "list of rows", {"lengths": A})])
def test_reorder_rows_refuses(status, text, arguments):
    assert reorder(**arguments) == status
    assert text in message()


def test_a_table_given_twice_is_refused():
    two = [(ctypes.c_void_p * 2)(A, A), longs(640, 640), longs(64, 64), longs(10, 10), longs(64, 64), 2]
    assert _lib.lib().wptv_reorder_rows(*two, 2 * A, None, 10, 1, 2, None) == -1 and "the same" in message()
    assert _lib.lib().wptv_keep_rows(*two, 2 * A, 1, 4, 3 * A, 1, None) == -1 and "the same" in message()


def keep(base=A, sb=640, sn=64, capacity=10, row=64, count=1, lists=1, kept=2 * A, keep=4, B=2):
    return _lib.lib().wptv_keep_rows((ctypes.c_void_p * 3)(base, 4 * A, 5 * A), longs(sb, sb, sb), longs(sn, sn, sn),
                                     longs(capacity, capacity, capacity), longs(row, row, row), count, kept, lists, keep,
                                     3 * A, B, None)


@pytest.mark.parametrize("status, text, arguments", [
    (-1, "list of rows", {"base": 2 * A}), (-1, "list of rows", {"base": 3 * A}),
    (-1, "3 tables for 2", {"count": 3, "lists": 2}), (-1, "for 0 lists", {"lists": 0}), (-1, "B=-1", {"B": -1}),
    (-3, "65535", {"B": 65536}), (-1, "overlap", {"sb": 639}), (-1, "overlap", {"sn": 32}), (-1, "kept", {"kept": None})])
def test_keep_rows_refuses(status, text, arguments):
    assert keep(**arguments) == status
    assert text in message()


@pytest.mark.parametrize("text, arguments", [
    ("must hold", (0, 0, 0)), ("must hold", (4, 3, 2)), ("must hold", (4, -1, 2)), ("must hold", (4, 1, -1))])
def test_choose_kept_refuses(text, arguments):
    assert _lib.lib().wptv_choose_kept(A, 10, 10, A, 1, 1, 10, *arguments, A, A, None) == -1
    assert text in message()


def test_choose_kept_takes_at_least_one_layer_and_texts_that_fit_its_counts():
    assert _lib.lib().wptv_choose_kept(A, 10, 10, A, 0, 1, 10, 4, 1, 1, A, A, None) == -1 and "bad shape" in message()
    assert _lib.lib().wptv_choose_kept(A, 10, 10, A, 1, 1, (1 << 30) + 1, 4, 1, 1, A, A, None) == -3
    assert "too large" in message()
    assert _lib.lib().wptv_choose_kept(A, 10, 10, A, 1, 0, 10, 4, 1, 1, A, A, None) == 0


@pytest.mark.parametrize("status, text, arguments", [
    (-3, "too large", {"N": (1 << 30) + 1}), (-3, "too large", {"T": 1 << 29, "H": 2}),
    (-1, "bad shape", {"H": 0}), (-1, "bad shape", {"N": 0}), (-3, "dtype", {"dtype": 3}), (-3, "width", {"c": 257}),
    (-1, "overlap", {"stride": 100}), (-1, "overlap", {"row": 63}), (-1, "NULL", {"q": None}), (-1, "splits", {"splits": -1})])
def test_attention_weights_refuse(status, text, arguments):
    a = dict(q=A, row=64, dtype=_lib.WPTV_BF16, B=2, T=3, H=4, c=64, N=101, splits=1, stride=101) | arguments
    assert _lib.lib().wptv_attention_weights(a["q"], A, 6464, a["row"], a["dtype"], A, A, None, None, a["B"], a["T"], a["H"],
                                             a["c"], a["N"], 0.125, a["splits"], A, a["stride"], None, 0, None) == status
    assert text in message()


def test_the_python_entry_points_refuse_what_is_not_theirs():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(kernels.KernelUnavailable):
        sampling.beam_step(x, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="dimensions"):
        sampling.beam_step(x[0], torch.zeros(2, 3))
    with pytest.raises(ValueError, match="bfloat16"):
        sampling.beam_step(x.half(), torch.zeros(2, 3))
    with pytest.raises(kernels.KernelUnavailable):
        kernels.reorder_rows(x, torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(ValueError, match="whole numbers"):
        kernels.reorder_rows(x, torch.zeros(1, 2))
    with pytest.raises(ValueError, match="texts, beams"):
        kernels.reorder_rows(x, torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="each table"):
        kernels.reorder_rows(x[0], torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(ValueError, match="no table"):
        kernels.reorder_rows([], torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(kernels.KernelUnavailable):
        kernels.keep_rows(x, torch.zeros(1, 2, 2, dtype=torch.long), torch.ones(2, dtype=torch.long))
    with pytest.raises(ValueError, match="layers, B, keep"):
        kernels.keep_rows(x, torch.zeros(2, 2, dtype=torch.long), torch.ones(2, dtype=torch.long))
    with pytest.raises(kernels.KernelUnavailable):
        kernels.choose_kept(x, torch.ones(3, dtype=torch.long), 2, 0, 1)
    with pytest.raises(ValueError, match="FP32"):
        kernels.choose_kept(x.double(), torch.ones(3, dtype=torch.long), 2, 0, 1)
    with pytest.raises(kernels.KernelUnavailable):
        kernels.add_attention_weights(torch.zeros(1, 1, 2, 8), x[:1], torch.zeros(1, 1, dtype=torch.long),
                                      torch.zeros(1, 1, 2), 1.0, torch.zeros(1, 3))


def test_the_definition_of_the_next_beams():
    scores = torch.log(torch.tensor([[[0.5, 0.3, 0.2], [0.1, 0.8, 0.1]]]))
    totals = torch.tensor([[0.0, -0.1]])
    t, p, v, e = beam_oracle.beam_step(scores, totals, stops=(1,), beams=3)
    assert p.tolist() == [[1, 0, 0]] and v.tolist() == [[1, 0, 1]] and e.tolist() == [[True, False, True]]
    assert torch.allclose(t.exp(), torch.tensor([[0.8 * torch.tensor(-0.1).exp().item(), 0.5, 0.3]], dtype=torch.double))
    # an ended beam stays as it is; equal values to the lowest beam, then token
    t, p, v, e = beam_oracle.beam_step(torch.zeros(1, 2, 4), torch.tensor([[-1.0, -1.0]]), torch.tensor([[True, False]]),
                                       stops=(2,), beams=4)
    assert p.tolist() == [[0, 1, 1, 1]] and v.tolist() == [[2, 0, 1, 2]] and e.tolist() == [[True, False, False, True]]


def test_the_definition_of_eviction():
    weights = torch.tensor([[[9.0, 1.0, 3.0, 2.0, 3.0, 0.0]]])
    kept, counts = eviction_oracle.choose_kept(weights, torch.tensor([6]), 4, 1, 1)
    assert kept.tolist() == [[[0, 2, 4, 5]]] and counts.tolist() == [4]
    table = torch.arange(6.0).view(1, 6, 1)
    assert eviction_oracle.keep_rows([table], kept, counts)[0].flatten().tolist() == [0, 2, 4, 5, 4, 5]
    q = torch.ones(1, 2, 1, 1)
    got = eviction_oracle.attention_weights(q, torch.zeros(1, 3, 1), torch.tensor([[1, 2]]), torch.tensor([[[0.0], [0.0]]]),
                                            1.0, torch.tensor([[5.0, 5.0, 5.0]]), start=torch.tensor([1]))
    assert got.tolist() == [[7.0, 2.0, 1.0]]


def test_tables_that_take_a_gradient_are_refused():
    x = torch.zeros(2, 3, 8, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        kernels.reorder_rows([torch.zeros(2, 3, 8, requires_grad=True)], torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(ValueError, match="gradient"):
        kernels.keep_rows(x, torch.zeros(1, 2, 2, dtype=torch.long), torch.ones(2, dtype=torch.long))


def two_tables(first, second, parents=1 << 40, n=1, W=2):
    """(status of reorder_rows, of keep_rows) of two tables (address, batch stride, row stride, capacity, row bytes)."""
    arrays = [(ctypes.c_void_p * 2)(first[0], second[0])] + [longs(a, b) for a, b in zip(first[1:], second[1:])] + [2]
    # a part of the moves that launches nothing: one beam a text, lists of no rows
    return (_lib.lib().wptv_reorder_rows(*arrays, parents, None, 10, n * W, 1, None),
            _lib.lib().wptv_keep_rows(*arrays, parents, 1, 0, 1 << 41, n * W, None))


@pytest.mark.parametrize("overlap, first, second", [
    (True, (A, 640, 64, 10, 64), (A + 63, 640, 64, 10, 64)), (True, (A, 640, 64, 10, 64), (A + 640, 640, 64, 10, 64)),
    (False, (A, 640, 64, 10, 64), (A + 1280, 640, 64, 10, 64)),
    (True, (A, 640, 64, 10, 64), (A + 1279, 640, 64, 10, 64)),
    # the two halves of each row, and one byte more
    (False, (A, 640, 64, 10, 32), (A + 32, 640, 64, 10, 32)), (True, (A, 640, 64, 10, 33), (A + 32, 640, 64, 10, 32)),
    (False, (A + 32, 640, 64, 10, 32), (A, 640, 64, 10, 32)), (True, (A + 32, 640, 64, 10, 32), (A, 640, 64, 10, 33)),
    # the halves again, the second a row further: its first row beside the other's second
    (False, (A, 1000, 64, 10, 32), (A + 96, 1000, 64, 10, 32)), (True, (A, 1000, 64, 10, 32), (A + 90, 1000, 64, 10, 32)),
    # in each batch row's block one table behind the other, of other rows
    (False, (A, 1000, 64, 10, 64), (A + 640, 1000, 36, 10, 36)), (True, (A, 1000, 64, 10, 64), (A + 620, 1000, 36, 10, 36)),
    # the end of one batch row's block and the start of the next one's
    (True, (A, 1000, 64, 10, 64), (A + 650, 1000, 36, 10, 36)), (False, (A, 1010, 64, 10, 64), (A + 650, 1010, 36, 10, 36)),
    # token rows outermost
    (False, (A, 64, 128, 10, 32), (A + 32, 64, 128, 10, 32)), (True, (A, 64, 128, 10, 32), (A + 31, 64, 128, 10, 32)),
    (True, (A, 64, 128, 10, 32), (A + 32, 1280, 128, 10, 32)),  # one nested each way: not told apart
    # a table of one row, and an empty one
    (False, (A, 640, 64, 10, 60), (A + 60, 640, 1, 1, 4)), (True, (A, 640, 64, 10, 60), (A + 59, 640, 1, 1, 4)),
    (False, (A, 640, 64, 10, 64), (A, 640, 64, 0, 64)), (False, (A, 640, 64, 0, 64), (A, 640, 64, 10, 64))])
def test_tables_that_overlap_are_refused(overlap, first, second):
    for status in two_tables(first, second):
        assert status == (-1 if overlap else 0), message()
    if overlap:
        assert "overlap" in message()


def test_lists_within_a_table_are_refused():
    # lists of 16 bytes: in a row, between two rows, behind the last
    for at, status in ((A + 8, -1), (A + 40, 0), (A + 50, -1), (A + 616, 0), (A + 1280, 0), (A - 8, -1), (A - 16, 0)):
        assert reorder(row=32, parents=at, W=2, n=1) == status if status else True
        assert reorder(row=32, parents=at, W=1, n=2) == status, (at - A, message())
    assert reorder(lengths=A + 700) == -1 and "list of rows" in message()
    assert keep(kept=A + 100, keep=0) == 0 and keep(kept=A + 100) == -1 and "list of rows" in message()


def test_overlapping_tables_by_their_bytes():
    """Random small tables against the sets of their bytes: every overlap is
    refused, and where the strides are the same nothing else."""
    import random
    rng = random.Random(0)

    def places(table, rows_b):
        base, sb, sn, capacity, row = table
        rows = [base + b * sb + n * sn for b in range(rows_b) for n in range(capacity)]
        got = {x + i for x in rows for i in range(row)}
        return got if len(got) == len(rows) * row else None

    seen = [0, 0]
    for _ in range(4000):
        rows_b, row, capacity = rng.randint(1, 3), rng.randint(1, 5), rng.randint(0, 4)
        sn = rng.randint(row, 12)
        sb = rng.choice([sn * capacity + rng.randint(0, 30), rng.randint(1, 40)])
        first = (A, sb, sn, capacity, row)
        same = rng.random() < 0.7
        second = (A + rng.randint(-150, 150), sb if same else rng.randint(1, 80), sn if same else rng.randint(1, 12),
                  rng.randint(0, 4), rng.randint(1, 5))
        a, b = places(first, rows_b), places(second, rows_b)
        nested = [t[3] <= 1 or rows_b <= 1 or t[1] >= (t[3] - 1) * t[2] + t[4] or t[2] >= (rows_b - 1) * t[1] + t[4]
                  for t in (first, second)]
        if a is None or b is None or not all(nested):
            continue
        for status in two_tables(first, second, n=1, W=rows_b):
            if a & b:
                assert status == -1, (first, second, rows_b)
            elif same:
                assert status == 0, (first, second, rows_b, message())
            seen[bool(a & b)] += 1
    assert min(seen) > 500


def test_more_texts_than_the_join_s_grid_holds_are_not_cut_in_parts():
    size = ctypes.c_size_t(0)
    for B, asked, given in ((65535, 2, 2), (65536, 2, 1), (65536, 0, 1)):
        parts = ctypes.c_int(asked)
        assert _lib.lib().wptv_attention_weights_workspace(B, 2, 16, 64, 64, _lib.WPTV_BF16, ctypes.byref(parts),
                                                           ctypes.byref(size)) == 0
        assert parts.value == given and (size.value == 0) == (given == 1)
