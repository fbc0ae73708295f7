"""Decoders whose feed-forward blocks are mixtures of experts, against the
oracle: read in pieces and through undo, their routes recorded, written by a
Writer and scored by log_probs, captured, and reordered by a beam search.

FP32: the routes are equal and the scores within 1e-5 of their largest, as the
dense decoder's.  bf16: the choice is made on the GPU's own bf16 stream, so that
near ties may fall the other way than the oracle's; the oracle then takes the
recorded routes, whose logits on its own stream must come within 5e-2 of its k-th
largest, and the scores lie within 2e-2."""

import pytest
import torch

from oracle.decoder import Decoder as Oracle
from wpt_amd import beams, sampling
from wpt_amd.decoder import EXACT, SPARSE, WINDOW, DecoderConfig, MQADecoder, random_weights
from wpt_amd.step import VerifyStep
from wpt_amd.writer import Writer

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
SMALL = DecoderConfig(layers=2, d_model=128, heads=4, head_dim=64, ffn=40, vocab=512, experts=10, experts_per_token=3)
MIXED = DecoderConfig(layers=4, d_model=256, heads=2, head_dim=128, ffn=64, vocab=512, kinds=(WINDOW, EXACT, SPARSE, EXACT),
                      window=16, rope_dims=32, top_k=8, experts=6, experts_per_token=2)


def models(config, dtype, seed=0, std=0.05, bias=False):
    w = random_weights(config, seed=seed, std=std)
    if bias:
        g = torch.Generator().manual_seed(seed + 1)
        for i in range(config.layers):
            w[f"layers.{i}.router_bias"] = 0.1 * torch.randn(config.experts, generator=g)
    rounded = {n: v if dtype == FP32 or n.endswith(("norm", "sink", "router", "router_bias")) else v.to(dtype).float()
               for n, v in w.items()}
    ora = Oracle(rounded, config.layers, config.heads, config.head_dim, config.kinds, config.window, config.rope_dims,
                 config.rope_base, config.top_k, experts_per_token=config.experts_per_token)
    return MQADecoder(config, w, dtype=dtype), ora


def close(got, expected, share):
    return float((got.cpu().double() - expected.double()).abs().max() / expected.abs().max()) <= share


@pytest.mark.parametrize("config", [SMALL, MIXED])
def test_fp32_readings_in_pieces_and_through_undo_match_the_oracle(device, config):
    model, ora = models(config, FP32, bias=config is SMALL)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, config.vocab, (3, 40), generator=g)
    cache, rows = model.new_cache(3, routes=True, capacity=16), ora.new_cache(3)
    seen = {i: [[] for _ in range(3)] for i in range(config.layers)}
    at = 0
    for n, counts, kept in ((9, (9, 4, 7), None), (5, (5, 5, 5), (2, 5, 0)), (1, (1, 1, 1), None), (12, (12, 3, 12), (1, 3, 12))):
        piece = ids[:, at:at + n]
        at += n
        got = model.extend(piece, cache, torch.tensor(counts), undoable=kept is not None)[0]
        expected = ora.extend(piece, rows, torch.tensor(counts), undoable=kept is not None)[0]
        live = torch.arange(n) < torch.tensor(counts)[:, None]
        assert close(got.cpu()[live], expected[live], 1e-5)
        if kept is not None:
            model.undo(cache, torch.tensor(kept))
            ora.undo(rows, torch.tensor(kept))
        for i in range(config.layers):
            for b in range(3):
                seen[i][b] += ora.routed[i][0][b, :counts[b] if kept is None else kept[b]].tolist()
    for i in range(config.layers):
        for b, length in enumerate(cache.lengths.tolist()):
            assert cache.routes[i, b, :length].tolist() == seen[i][b], (i, b)


@pytest.mark.parametrize("B, T", [(2, 5), (7, 30), (3, 200), (1, 1)])
def test_bf16_readings_on_every_product_match_the_oracle(device, B, T):
    # 10 rows and 210 (fm products), 600 (row-major ones), one
    config = DecoderConfig(layers=2, d_model=256, heads=4, head_dim=64, ffn=96, vocab=512, experts=12, experts_per_token=4)
    model, ora = models(config, BF16)
    ids = torch.randint(0, config.vocab, (B, T), generator=torch.Generator().manual_seed(B))
    cache = model.new_cache(B, routes=True, capacity=T)
    scores, _ = model.extend(ids, cache)
    for i in range(config.layers):
        ora.given_routes[i] = cache.routes[i, :, :T].cpu()
    expected = ora.extend(ids, ora.new_cache(B))[0]
    for i in range(config.layers):
        own, x = ora.routed[i]
        logits = x.double() @ ora.w[f"layers.{i}.router"].double().T
        last = logits.gather(-1, own.long()).amin(-1)
        assert bool((logits.gather(-1, ora.given_routes[i].long()).amin(-1) >= last - 5e-2).all())
    assert close(scores, expected, 2e-2)


def test_a_writer_records_routes_and_log_probs_score_what_it_wrote(device):
    # the operators as a rollout uses them: written tokens, their routes, their log-probabilities
    model, _ = models(SMALL, BF16, seed=4)
    g = torch.Generator(device=device).manual_seed(1)
    writer = Writer(model, [3, 5, 7], rows=4, generator=g, top_k=None, temperature=1.0, routes=True)
    for _ in range(6):
        writer.write({}, {i: 1 for i in range(4)})
    text = torch.tensor(writer.histories, device=device)
    assert text.shape == (4, 9)
    cache = model.new_cache(4, routes=True)
    scores = model.extend(text, cache, logits=True)[0]
    read = int(writer.cache.lengths.min())
    assert read >= 8
    same = (writer.routes[:, :, :8] == cache.routes[:, :, :8]).float().mean()
    assert float(same) > 0.9  # readings of 1 and of 9 tokens sum in other orders: near ties only
    lp, entropy, ids, best = sampling.log_probs(scores[:, :-1], text[:, 1:], top=5)
    plain = torch.log_softmax(scores[:, :-1].double(), -1)
    assert torch.allclose(lp.double(), plain.gather(-1, text[:, 1:, None])[..., 0], atol=1e-5)
    assert torch.allclose(entropy.double(), -(plain.exp() * plain).sum(-1), atol=1e-5)
    assert torch.allclose(best.double(), plain.topk(5, -1).values, atol=1e-5)
    assert bool((lp <= best[..., 0]).all()) and bool((entropy >= 0).all())


def test_a_captured_step_of_experts_replays_as_the_eager_one(device):
    config = DecoderConfig(layers=2, d_model=256, heads=4, head_dim=64, ffn=96, vocab=512, experts=8, experts_per_token=2)
    w = random_weights(config, seed=7, std=0.05)
    k, B = 3, 4
    prompt = torch.randint(0, config.vocab, (B, 20), generator=torch.Generator().manual_seed(2))

    def start(step_cls):
        model = MQADecoder(config, w, dtype=BF16)
        cache = model.new_cache(B, routes=True, capacity=128)
        model.extend(prompt, cache)
        step = step_cls(model, cache, k, greedy=True)
        step.feeds.copy_(prompt[:, :k + 1])
        return step, cache

    eager, eager_cache = start(VerifyStep)
    taken = [tuple(t.clone() for t in eager.run()) for _ in range(8)]
    replayed, cache = start(VerifyStep)
    replayed.capture(warmup=2)
    for i in range(2, 8):
        tokens, counts = replayed.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, taken[i][0]) and torch.equal(counts, taken[i][1])
    assert torch.equal(cache.lengths, eager_cache.lengths)
    for b, length in enumerate(cache.lengths.tolist()):
        assert torch.equal(cache.routes[:, b, :length], eager_cache.routes[:, b, :length])


def test_beams_carry_their_routes_and_a_weighted_cache_has_none(device):
    model, _ = models(SMALL, FP32, seed=5)
    ids = torch.randint(0, SMALL.vocab, (4, 6), generator=torch.Generator().manual_seed(0))
    cache = model.new_cache(4, routes=True)
    model.extend(ids, cache, torch.tensor([6, 3, 5, 6]))
    before = cache.routes.clone()
    model.reorder(cache, torch.tensor([[1, 1], [0, 0]]))
    assert torch.equal(cache.routes[:, 0, :3], before[:, 1, :3]) and torch.equal(cache.routes[:, 3, :5], before[:, 2, :5])
    assert cache.lengths.tolist() == [3, 3, 5, 5]
    copy = cache.select([3, 0])
    assert torch.equal(copy.routes, cache.routes[:, [3, 0]])
    with pytest.raises(ValueError):
        model.new_cache(2, routes=True, weighted=True)
    found = beams.BeamWriter(model, [[1, 2, 3]], 3, stops=(0,), keep=40).write(5)
    assert len(found[0]) == 3


def test_window_layers_alone_read_a_long_prompt(device):
    config = DecoderConfig(layers=2, d_model=128, heads=2, head_dim=64, ffn=32, vocab=128, kinds=(WINDOW, WINDOW), window=8,
                           rope_dims=32, experts=4, experts_per_token=2)
    model, _ = models(config, BF16)
    ids = torch.randint(0, config.vocab, (3, 250), generator=torch.Generator().manual_seed(1))
    whole = model.new_cache(3, widest=250, routes=True, capacity=8)
    scores = model.extend(ids, whole)[0]
    pieces = model.new_cache(3, widest=250, routes=True)
    parts = torch.cat([model.extend(ids[:, a:a + 50], pieces)[0] for a in range(0, 250, 50)], 1)
    assert whole.routes.shape[2] >= 250 and int((whole.routes[:, :, :250] < 0).sum()) == 0
    same = (whole.routes[:, :, :250] == pieces.routes[:, :, :250]).all(-1).all(0)  # (3, 250): no near tie fell the other way
    assert float(same.float().mean()) > 0.9
    assert float((scores - parts).abs()[same].max()) <= 2e-2 * float(parts.abs().max())


def test_a_dense_decoder_records_no_routes(device):
    config = DecoderConfig(layers=1, d_model=64, heads=1, head_dim=64, ffn=32, vocab=64)
    with pytest.raises(NotImplementedError):
        MQADecoder(config, random_weights(config), dtype=BF16).new_cache(1, routes=True)
