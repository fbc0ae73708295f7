"""How far a Writer's captured reading may be replayed, off the GPU: its graph is
bound to the memory that it was captured over."""

import pytest
import torch

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
