"""A weighted cache's deferred readings on the host alone: what is added when,
and what is refused (the kernels and the capture are stood in for; no GPU is
needed)."""

import pytest
import torch

from wpt_amd import cache as module
from wpt_amd.cache import Cache


@pytest.fixture
def host(monkeypatch):
    """The kernels recorded in a list, and whether the stream captures."""
    class Host:
        capturing = False
        added = []

    def lengths(held, before, counts, undo):
        if before is not None and not undo:
            before.copy_(held)
        held.copy_((before if undo else held) + counts)

    state = Host()
    state.added = []
    monkeypatch.setattr(module, "_lengths", lengths)
    monkeypatch.setattr(module.kernels, "add_attention_weights",
                        lambda q, k, positions, lse, scale, weights, counts=None, start=None:
                        state.added.append((int(q.flatten()[0]), counts.tolist(), start.tolist())))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    return state


def read(cache, name, tokens, undoable):
    """A reading of `tokens` tokens, as the decoder's extend makes it."""
    cache.settle()
    cache.reserve(cache.bound + tokens)
    counts = torch.full((cache.rows,), tokens)
    for layer in cache.growing:
        cache.weigh(layer, torch.full((cache.rows, tokens, 1, 4), float(name)), None, None, 1.0, counts, undoable)
    cache.finish(counts, undoable, tokens)


def weighted(rows=2, layers=2):
    return Cache(rows, layers, 8, torch.float32, "cpu", capacity=16, weighted=True)


def test_a_reading_is_added_when_it_is_known_what_stays(host):
    cache = weighted()
    read(cache, 1, 3, undoable=False)
    assert host.added == [(1, [3, 3], [0, 0])] * 2
    read(cache, 2, 4, undoable=True)
    assert len(host.added) == 2
    cache.undo(torch.tensor([1, 4]))
    assert host.added[2:] == [(2, [1, 4], [3, 3])] * 2 and cache.lengths.tolist() == [4, 7]
    read(cache, 3, 2, undoable=True)
    read(cache, 4, 1, undoable=False)  # the reading before stays whole
    assert host.added[4:] == [(3, [2, 2], [4, 7])] * 2 + [(4, [1, 1], [6, 9])] * 2


def test_rows_are_not_copied_moved_or_evicted_while_a_reading_is_pending(host):
    cache = weighted()
    read(cache, 1, 3, undoable=True)
    for move in (lambda: cache.select([0]), lambda: cache.reorder(torch.tensor([[1, 0]])), lambda: cache.evict(2, 0, 1)):
        with pytest.raises(ValueError, match="pending"):
            move()
    assert not host.added


def test_a_pending_reading_is_not_added_in_a_capture_it_was_not_made_in(host):
    cache = weighted()
    read(cache, 1, 3, undoable=True)
    host.capturing = True
    with pytest.raises(RuntimeError, match="before capturing"):
        read(cache, 2, 1, undoable=False)
    with pytest.raises(RuntimeError, match="before capturing"):
        cache.undo(torch.tensor([1, 1]))
    assert not host.added and cache.lengths.tolist() == [3, 3]
    host.capturing = False
    cache.undo(torch.tensor([1, 1]))
    assert host.added == [(1, [1, 1], [0, 0])] * 2 and cache.lengths.tolist() == [1, 1]
    host.capturing = True  # a captured reading with its undo, or with the reading after it
    read(cache, 3, 2, undoable=True)
    cache.undo(torch.tensor([2, 0]))
    read(cache, 4, 2, undoable=True)
    read(cache, 5, 1, undoable=False)
    assert [x[0] for x in host.added[2:]] == [3, 3, 4, 4, 5, 5]


def test_a_captured_reading_is_not_added_outside_its_capture(host):
    cache = weighted()
    host.capturing = True
    read(cache, 1, 3, undoable=True)
    host.capturing = False
    with pytest.raises(RuntimeError, match="captured together"):
        cache.undo(torch.tensor([1, 1]))
    with pytest.raises(RuntimeError, match="captured together"):
        read(cache, 2, 1, undoable=False)
    assert not host.added


def test_a_reading_that_failed_half_way_leaves_nothing_to_add(host):
    cache = weighted()
    read(cache, 1, 3, undoable=False)
    counts = torch.tensor([2, 2])
    cache.weigh(0, torch.full((2, 2, 1, 4), 9.0), None, None, 1.0, counts, True)  # an error before the next layer
    read(cache, 2, 1, undoable=False)
    assert [x[0] for x in host.added] == [1, 1, 2, 2]
    cache.weigh(0, torch.full((2, 2, 1, 4), 9.0), None, None, 1.0, counts, True)
    read(cache, 3, 2, undoable=True)
    cache.undo(torch.tensor([1, 1]))
    assert [x[0] for x in host.added[4:]] == [3, 3]
    read(cache, 4, 2, undoable=True)
    cache.settle()  # the next reading begins: the one before is whole
    cache.weigh(0, torch.full((2, 2, 1, 4), 9.0), None, None, 1.0, counts, True)
    with pytest.raises(ValueError, match="not here"):
        cache.undo(torch.tensor([1, 1]))
    assert [x[0] for x in host.added[6:]] == [4, 4]


def test_the_rows_that_sparse_layers_read_are_not_evicted(host):
    cache = Cache(2, 2, 8, torch.float32, "cpu", capacity=16, bare=(1,), weighted=True, recent=16)
    for held in (cache, cache.select([1, 0])):
        with pytest.raises(ValueError, match="sparse layers read the last 16"):
            held.evict(20, 2, 15)
