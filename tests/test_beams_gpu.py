"""Beam search and the bounded cache as they are used: the decoder's cache
reordered in place and evicted from, readings of a weighted cache, and the
BeamWriter's run of all of them."""

import math

import pytest
import torch

from oracle import beam as beam_oracle
from wpt_amd import kernels, sampling
from wpt_amd.beams import BeamWriter
from wpt_amd.decoder import EXACT, SPARSE, WINDOW, DecoderConfig, MQADecoder, random_weights
from wpt_amd.step import VerifyStep

pytestmark = pytest.mark.gpu

EXACTS = DecoderConfig(layers=3, d_model=256, heads=4, head_dim=64, ffn=256, vocab=512)
MIXED = DecoderConfig(layers=5, d_model=256, heads=4, head_dim=64, ffn=256, vocab=512,
                      kinds=(WINDOW, EXACT, WINDOW, EXACT, SPARSE), window=16, top_k=8)


def decoder(device, config=EXACTS, dtype=torch.float32, seed=0, std=0.08, silent=()):
    weights = random_weights(config, seed=seed, std=std)
    for i in silent:  # a layer whose attention adds nothing
        weights[f"layers.{i}.out"].zero_()
    return MQADecoder(config, weights, dtype, device)


def tokens(*shape, seed=0, vocab=512):
    return torch.randint(0, vocab, shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("config", [EXACTS, MIXED], ids=["exact", "mixed"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reordered_rows_go_on_as_copies_of_their_parents(device, config, dtype):
    model = decoder(device, config, dtype)
    for length in (5, 70):  # within the rings and past their end
        cache = model.new_cache(6, capacity=16, widest=16, weighted=True)
        ids = tokens(6, length, seed=length)
        counts = torch.tensor([length, length - 3, length, 1, length, 2])
        model.extend(ids, cache, counts)
        parents = torch.tensor([[2, 0, 0], [1, 1, 5 - 3]], device=device)
        copy = cache.select([2, 0, 0, 4, 4, 5])
        model.reorder(cache, parents)
        assert torch.equal(cache.lengths, copy.lengths)
        for b, n in enumerate(cache.lengths.tolist()):
            assert torch.equal(cache.weights[:, b, :n], copy.weights[:, b, :n])
        after = tokens(6, 3, seed=1)
        a, b = model.extend(after, cache)[0], model.extend(after, copy)[0]
        assert torch.equal(a, b)
        with pytest.raises(ValueError, match="parents"):
            model.reorder(cache, torch.zeros(2, 2, dtype=torch.long))
        model.extend(after, cache, undoable=True)
        with pytest.raises(ValueError, match="pending"):
            model.reorder(cache, parents)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_weights_of_a_decoder_s_readings(device, dtype):
    model = decoder(device, MIXED, dtype)
    ids = tokens(3, 60, seed=2)
    counts = torch.tensor([60, 37, 0])
    whole = model.new_cache(3, widest=16, weighted=True)  # wider than the rings: read in pieces
    model.extend(ids, whole, counts)
    # each of a token's 4 query heads gives weight 1 in all, in each exact layer
    assert torch.allclose(whole.weights.sum(-1).cpu(), 4.0 * counts.float().expand(2, 3), rtol=1e-3)
    parts = model.new_cache(3, widest=16, weighted=True)
    for start, end in ((0, 20), (20, 60)):
        model.extend(ids[:, start:end], parts, (counts - start).clamp(0, end - start))
    undone = model.new_cache(3, widest=64, weighted=True)  # drafts read and taken back leave nothing
    for start, end in ((0, 20), (20, 41), (41, 60)):
        kept = (counts - start).clamp(0, end - start)
        model.extend(torch.cat([ids[:, start:end], tokens(3, 5, seed=9)], 1), undone, undoable=True)
        model.undo(undone, kept)
    kept_all = model.new_cache(3, widest=64, weighted=True)  # undoable, but followed by another reading
    model.extend(ids[:, :20], kept_all, counts.clamp(0, 20), undoable=True)
    model.extend(ids[:, 20:], kept_all, (counts - 20).clamp(0, 40))
    # the readings differ in the order of the decoder's sums: bf16's step is 2^-8, and layers pass it on
    bound = 1e-3 if dtype == torch.float32 else 0.2
    for cache in (parts, undone, kept_all):
        assert torch.equal(cache.lengths, whole.lengths)
        for b, n in enumerate(counts.tolist()):
            off = (cache.weights[:, b, :n] - whole.weights[:, b, :n]).norm()
            assert float(off) <= bound * float(whole.weights[:, b, :n].norm()) + 1e-30


def test_evicted_rows_are_gone_and_the_others_go_on(device):
    keep, first, recent = 24, 2, 7
    model = decoder(device)
    ids = tokens(3, 50, seed=3)
    counts = torch.tensor([50, 20, 30])
    cache = model.new_cache(3, weighted=True)
    model.extend(ids, cache, counts)
    tables = [t.clone() for t in cache.tables]
    weights, lengths = cache.weights.clone(), cache.lengths.clone()
    kept = model.evict(cache, keep, first, recent)
    assert cache.lengths.tolist() == [24, 20, 24] and cache.evicted.tolist() == [26, 0, 6] and cache.bound == keep
    expected, _ = kernels.choose_kept(weights, lengths, keep, first, recent)
    assert torch.equal(kept, expected)
    # a cache made by hand of the same rows goes on with the same scores and weights
    other = model.new_cache(3, weighted=True)
    for i, t in enumerate(tables):
        for b, n in enumerate(cache.lengths.tolist()):
            other.tables[i][b, :n] = t[b, kept[i, b, :n]]
            other.weights[i, b, :n] = weights[i, b, kept[i, b, :n]]
    other.lengths.copy_(cache.lengths)
    other.bound = cache.bound
    after = tokens(3, 4, seed=4)
    a, b = model.extend(after, cache)[0], model.extend(after, other)[0]
    assert torch.equal(a, b)
    for b, n in enumerate(cache.lengths.tolist()):
        assert torch.equal(cache.weights[:, b, :n], other.weights[:, b, :n])
    # every row within the budget: nothing happens
    model.evict(cache, 60, first, recent)
    assert cache.lengths.tolist() == [28, 24, 28] and cache.evicted.tolist() == [26, 0, 6]


def test_window_layers_keep_their_places_after_an_eviction(device):
    # the exact layer's attention adds nothing to the stream: what is evicted from it cannot be seen, unless a
    # window layer's ring loses its tokens' places
    config = DecoderConfig(layers=3, d_model=256, heads=4, head_dim=64, ffn=256, vocab=512, kinds=(WINDOW, EXACT, WINDOW),
                           window=16)
    model = decoder(device, config, silent=(1,))
    ids = tokens(2, 45, seed=5)
    plain, bounded = model.new_cache(2, widest=16), model.new_cache(2, widest=16, weighted=True)
    for cache in (plain, bounded):
        model.extend(ids, cache)
    model.evict(bounded, 20, 2, 8)
    for step in range(3):
        after = tokens(2, 3, seed=6 + step)
        a, b = model.extend(after, plain)[0], model.extend(after, bounded)[0]
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
        a = model.extend(after, plain, undoable=True)[0]
        b = model.extend(after, bounded, undoable=True)[0]
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
        for cache in (plain, bounded):
            model.undo(cache, torch.tensor([1, 0]))
        model.evict(bounded, 20, 2, 8)
    assert torch.equal(plain.lengths, bounded.starts())
    for layer in (0, 2):
        assert torch.allclose(plain.tail(layer, 15), bounded.tail(layer, 15), rtol=1e-5, atol=1e-5)


def test_what_eviction_refuses(device):
    model = decoder(device, MIXED)
    cache = model.new_cache(1)
    with pytest.raises(ValueError, match="weighted"):
        model.evict(cache, 100)
    cache = model.new_cache(1, weighted=True)
    model.extend(tokens(1, 40), cache)
    with pytest.raises(ValueError, match="sparse layers"):
        model.evict(cache, 30, 2, 15)
    with pytest.raises(ValueError, match="must hold"):
        model.evict(cache, 30, 20, 16)
    model.extend(tokens(1, 2), cache, undoable=True)
    with pytest.raises(ValueError, match="pending"):
        model.evict(cache, 30, 2, 16)
    with pytest.raises(ValueError, match="undo\\(\\)"):
        cache.undo_on_device()
    model.undo(cache, [1])
    model.evict(cache, 30, 2)
    assert cache.lengths.tolist() == [30]


def test_verify_steps_on_a_weighted_cache(device):
    model = decoder(device, EXACTS, torch.bfloat16)
    caches = []
    for captured in (False, True):
        cache = model.new_cache(2, capacity=128, weighted=True)
        model.extend(tokens(2, 9, seed=1), cache)
        step = VerifyStep(model, cache, k=3, greedy=True)
        step.feeds.copy_(tokens(2, 4, seed=2))
        if captured:
            step.capture()  # two eager steps before it
            for _ in range(3):
                torch.cuda.synchronize()
                step.replay()
        else:
            for _ in range(5):
                step.run()
        torch.cuda.synchronize()
        copy = cache.select([1, 0])  # a cache whose host bound the replays have not raised
        model.reorder(cache, torch.tensor([[1, 0]]))
        assert torch.equal(cache.lengths, copy.lengths)
        for b, n in enumerate(cache.lengths.tolist()):
            assert all(torch.equal(x[b, :n], y[b, :n]) for x, y in zip(cache.tables, copy.tables))
        caches.append(cache)
        assert torch.allclose(cache.weights.sum(-1), 4.0 * cache.lengths.float().expand(3, 2), rtol=1e-2)
    assert torch.equal(caches[0].lengths, caches[1].lengths)
    for b, n in enumerate(caches[0].lengths.tolist()):
        assert torch.equal(caches[0].weights[:, b, :n], caches[1].weights[:, b, :n])


def plain_search(model, prompt, beams, steps, stops):
    """Beam search that reads every beam's whole text at every step."""
    texts, totals, ended = [list(prompt)], torch.tensor([[0.0]]), torch.tensor([[False]])
    for _ in range(steps):
        scores = torch.stack([model(torch.tensor([t]))[0, -1] for t in texts])[None].cpu()
        totals, parents, picks, ended = beam_oracle.beam_step(scores, totals, ended if stops else None, stops, beams)
        texts = [texts[p] + [t] for p, t in zip(parents[0].tolist(), picks[0].tolist())]
    return [t[len(prompt):] for t in texts], totals[0].tolist()


@pytest.mark.parametrize("config", [EXACTS, MIXED], ids=["exact", "mixed"])
@pytest.mark.parametrize("beams, stops", [(1, ()), (4, ()), (5, (3, 7, 100, 200, 300))])
def test_the_beams_written_are_those_of_a_plain_search(device, config, beams, stops):
    model = decoder(device, config, std=0.12)
    prompts = [tokens(n, seed=n).tolist() for n in (7, 1, 30)]
    writer = BeamWriter(model, prompts, beams, stops=stops)
    got = writer.write(9)
    for prompt, found in zip(prompts, got):
        texts, totals = plain_search(model, prompt, beams, len(writer._steps), stops)
        cut = [t[:1 + min([t.index(s) for s in stops if s in t], default=len(t))] for t in texts]
        assert [t for t, _ in found] == cut
        assert [x for _, x in found] == pytest.approx(totals, abs=1e-3)


def test_a_search_of_ended_beams_stops(device):
    model = decoder(device)
    writer = BeamWriter(model, [[1, 2], [3]], 3, stops=iter((7,)))
    writer.ended.fill_(True)
    writer.totals.copy_(torch.tensor([[-1.0, -2.0, -float("inf")], [-1.0, -1.5, -3.0]]))
    assert [[t for t, _ in beams] for beams in writer.write(50)] == [[[], []], [[], [], []]]
    assert not writer._steps


def test_beam_search_on_a_bounded_cache(device):
    model = decoder(device, MIXED, torch.bfloat16)
    prompts = [tokens(n, seed=n).tolist() for n in (90, 3, 41)]
    unbounded = BeamWriter(model, prompts, 4, stops=(5,)).write(20)
    wide = BeamWriter(model, prompts, 4, stops=(5,), keep=400, first=2).write(20)  # never reached
    assert wide == unbounded
    writer = BeamWriter(model, prompts, 4, stops=(5,), keep=40, first=2)
    got = writer.write(20)
    assert int(writer.cache.lengths.max()) <= 45
    assert (writer.cache.lengths + writer.cache.evicted).tolist() == [len(p) - 1 + 20 for p in prompts for _ in range(4)]
    for beams in got:
        assert len(beams) == 4 and all(math.isfinite(x) for _, x in beams)
        assert [x for _, x in beams] == sorted((x for _, x in beams), reverse=True)
        assert len({tuple(t) for t, _ in beams}) == 4
    # a text's own beams do not depend on the texts beside it but for the last bits of its scores
    assert writer.cache.weights.shape[:2] == (2, 12)


def test_what_the_beam_writer_refuses(device):
    model = decoder(device)
    for arguments in (([], 2), ([[]], 2), ([[1]], 0), ([[1]], 65)):
        with pytest.raises(ValueError):
            BeamWriter(model, *arguments)
    with pytest.raises(ValueError, match="keep"):
        BeamWriter(model, [[1]], 2, keep=3, first=4)
    with pytest.raises(ValueError, match="16 tokens"):
        BeamWriter(model, [[1]], 2, stops=range(17))
    with pytest.raises(ValueError, match="sparse layers"):
        BeamWriter(decoder(device, MIXED), [[1]], 2, keep=17, first=2)
    for prompts, stops in (([[1, 512]], ()), ([[-1]], ()), ([[1]], (512,))):
        with pytest.raises(IndexError):
            BeamWriter(model, prompts, 2, stops=stops)


def test_a_captured_beam_step(device):
    model = decoder(device, EXACTS, torch.bfloat16)
    n, W = 2, 3
    cache = model.new_cache(n * W, capacity=64, weighted=True)
    ids = tokens(n, 6, seed=1).repeat_interleave(W, 0)
    model.extend(ids, cache)
    start = [x.clone() for x in cache.tables] + [cache.weights.clone(), cache.lengths.clone()]
    last, totals = tokens(n * W, 1, seed=2).to(device), torch.zeros(n, W, device=device)
    first_last = last.clone()

    def step():
        scores = model.extend(last, cache, logits=True)[0].view(n, W, -1)
        t, parents, picks, _ = sampling.beam_step(scores, totals)
        model.reorder(cache, parents)
        totals.copy_(t)
        last.copy_(picks.view(n * W, 1))

    def reset():
        for x, y in zip(cache.tables + [cache.weights, cache.lengths], start):
            x.copy_(y)
        last.copy_(first_last)
        totals.zero_()

    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream(device).wait_stream(stream)
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    results = []
    for replayed in (True, False):
        reset()
        cache.bound = 6
        for _ in range(5):
            torch.cuda.synchronize()
            graph.replay() if replayed else step()
            cache.bound += 1 if replayed else 0
        torch.cuda.synchronize()
        results.append([totals.clone(), last.clone(), cache.lengths.clone(), cache.weights[..., :11].clone()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_the_cache_itself_knows_what_the_sparse_layers_read(device):
    cache = decoder(device, MIXED).new_cache(1, weighted=True)
    with pytest.raises(ValueError, match="sparse layers read the last 16"):
        cache.evict(30, 2, 15)
    decoder(device).new_cache(1, weighted=True).evict(30, 2, 0)  # no sparse layers


def test_evictions_in_a_captured_step(device):
    model = decoder(device, MIXED, torch.bfloat16)
    prompt = tokens(3, 30, seed=1)
    cache = model.new_cache(3, capacity=64, widest=16, weighted=True)
    model.extend(prompt, cache, torch.tensor([30, 22, 9]))
    last = tokens(3, 2, seed=2).to(device)
    state = [t for t in cache.tables if t is not None] + [cache.weights, cache.lengths, cache.evicted]
    start, bound = [x.clone() for x in state], cache.bound

    def step():
        scores = model.extend(last, cache)[0]
        kept = model.evict(cache, 24, 2, 16)
        last.copy_(scores.argmax(-1))
        return kept

    def reset():
        for x, y in zip(state, start):
            x.copy_(y)
        last.copy_(tokens(3, 2, seed=2))
        cache.bound = bound

    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream(device).wait_stream(stream)
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    runs = [[], []]
    for run, replayed in zip(runs, (True, False)):
        reset()
        for _ in range(5):
            torch.cuda.synchronize()
            kept = step() if not replayed else (graph.replay(), captured)[1]
            torch.cuda.synchronize()
            run.append([kept.clone(), last.clone(), cache.lengths.clone(), cache.evicted.clone()])
        run.append([t[:, :24].clone() for t in state[:-3]] + [cache.weights[..., :20].clone()])
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert cache.lengths.tolist() == [24, 24, 19] and cache.evicted.tolist() == [16, 8, 0]


def test_prompts_of_several_chunks_on_a_bounded_cache(device):
    # the exact layer's attention adds nothing to the stream: evictions while the prompts are read change nothing
    config = DecoderConfig(layers=3, d_model=256, heads=4, head_dim=64, ffn=256, vocab=512, kinds=(WINDOW, EXACT, WINDOW),
                           window=16)
    model = decoder(device, config, std=0.12, silent=(1,))
    prompts = [tokens(n, seed=n).tolist() for n in (2300, 1100, 40)]
    plain = BeamWriter(model, prompts, 3).write(6)
    writer = BeamWriter(model, prompts, 3, keep=200, first=4, recent=50)
    got = writer.write(6)
    assert [[t for t, _ in beams] for beams in got] == [[t for t, _ in beams] for beams in plain]
    for a, b in zip(got, plain):
        assert [x for _, x in a] == pytest.approx([x for _, x in b], abs=1e-3)
    assert int(writer.cache.lengths.max()) <= 225
    assert writer.cache.starts().tolist() == [len(p) - 1 + 6 for p in prompts for _ in range(3)]
