"""Whether a Writer's captured reading may be replayed, off the GPU: its graph is
bound to the memory that it was captured over."""

import gc
import types
import weakref

import pytest
import torch

from wpt_amd import writer
from wpt_amd.cache import Cache


@pytest.mark.parametrize("kinds, room", [(dict(), 16), (dict(rings=(0, 1)), None), (dict(rings=(0, 1), routes=3), 16),
                                         (dict(rings=(1,), routes=3), 16), (dict(bare=(1,)), 16)])
def test_a_cache_s_room_is_what_reserve_goes_by(monkeypatch, kinds, room):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    cache = Cache(2, 2, 8, torch.float32, "cpu", capacity=16, ring_rows=16, **kinds)
    assert cache.room == room
    tables = cache.tables
    cache.reserve(16)
    assert cache.tables is tables
    cache.reserve(17)
    assert cache.room == (None if room is None else 32)
    assert (cache.tables is tables) == (room is None)
    assert cache.routes is None or cache.routes.shape[2] == 32


class Captured(writer._CapturedRead):
    """A captured reading without its graph: what it was captured over."""

    made = 0

    def __init__(self, of, L):
        rows, V, width = of.cache.rows, 8, L + 1
        self.ids, self.drafts = torch.zeros(rows, width, dtype=torch.long), torch.zeros(rows, L, dtype=torch.long)
        self.q, self.state = torch.zeros(rows, L, V), torch.zeros(16, dtype=torch.uint8)
        of.cache.reserve(of.cache.bound + width * self.ROUNDS)
        self.limit, self.tables = of.cache.room, of.cache.tables
        self.read, self.tokens, self.counts = (None,), None, None
        self.graph = types.SimpleNamespace(replay=lambda: None)
        Captured.made += 1


@pytest.mark.parametrize("grown_by", ["another length", "an eager reading", "the program"])
def test_a_reading_captured_over_replaced_tables_is_not_replayed(monkeypatch, grown_by):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(writer, "_CapturedRead", Captured)
    monkeypatch.setattr(writer.sampling, "generator_state", lambda *a: torch.zeros(16, dtype=torch.uint8))
    monkeypatch.setattr(writer.sampling, "set_offset", lambda *a: None)
    monkeypatch.setattr(Captured, "made", 0)
    of = object.__new__(writer.Writer)
    of.cache, of.generator, of.device, of._reads = Cache(2, 1, 8, torch.float32, "cpu", capacity=256, routes=2), None, "cpu", {}
    of._rows = [types.SimpleNamespace(unread=[1]) for _ in range(2)]

    def round_(L):
        of._captured_round(torch.zeros(2, L, dtype=torch.long), torch.zeros(2, L, 8), L)

    for _ in range(40):
        round_(4)
    assert Captured.made == 1 and of.cache.bound == 200 and of.cache.room == 512
    if grown_by == "another length":  # 64 more rounds of 6 tokens do not fit
        round_(5)
    elif grown_by == "an eager reading":
        of.cache.reserve(of.cache.bound + 400)
    else:
        of.cache.reserve(5000)
    assert of.cache.room > 512
    before = Captured.made
    of._reads[2] = stale = Captured(of, 2)  # of a length that does not come again, over tables that the next growth replaces
    before += 1
    of.cache.reserve(of.cache.room + 1)
    held = weakref.ref(stale.tables[0])
    del stale
    round_(4)  # 211 of 512 tokens, but of the tables before
    assert Captured.made == before + 1
    gc.collect()
    assert held() is None  # the tables that are gone are not kept
    round_(4)
    assert Captured.made == before + 1
