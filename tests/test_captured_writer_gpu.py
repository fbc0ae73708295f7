"""Writers whose steady rounds replay HIP graphs, against the same Writers read
eagerly: past the growth of what the cache holds."""

import pytest
import torch

from wpt_amd.decoder import WINDOW, DecoderConfig, MQADecoder, random_weights
from wpt_amd.writer import Writer

pytestmark = pytest.mark.gpu


class Guesses:
    """Drafts whose every token has the same probability; a few of them are taken."""

    def draft(self, model, texts, context, draft, probabilities, generator):
        V = model.config.vocab
        tokens = torch.tensor([[(7 * t[-1] + 3 * j + len(t)) % V for j in range(draft)] for t in texts], device=model.device)
        return tokens, torch.full((len(texts), draft, V), 1.0 / V, device=model.device), None


def written(config, w, lengths, rounds, capture, device, routes, reserved={}):
    model = MQADecoder(config, w, dtype=torch.bfloat16)
    g = torch.Generator(device=device).manual_seed(2)
    writer = Writer(model, [3, 5, 7], 3, temperature=1.0, top_k=None, generator=g, drafter=Guesses(), routes=routes,
                    capture=capture)
    for i in range(rounds):
        writer.draft = lengths[i % len(lengths)]
        if i in reserved:
            writer.cache.reserve(reserved[i])
        writer.write({}, {r: writer.draft + 1 for r in range(3)})
    return writer


@pytest.mark.parametrize("routes", [True, False])
def test_a_captured_writer_of_window_layers_alone(device, routes):
    config = DecoderConfig(layers=2, d_model=128, heads=2, head_dim=64, ffn=32, vocab=64, kinds=(WINDOW, WINDOW), window=8,
                           rope_dims=32, experts=4, experts_per_token=2)
    w = random_weights(config, seed=1, std=0.05)
    eager, captured = (written(config, w, (4,), 130, c, device, routes) for c in (False, True))
    assert captured._reads and captured.histories == eager.histories
    if routes:
        assert captured.routes.shape[2] > 512
        for b, length in enumerate(eager.cache.lengths.tolist()):
            assert torch.equal(captured.routes[:, b, :length], eager.routes[:, b, :length])
            assert int(captured.routes[:, b, :length].min()) >= 0


@pytest.mark.parametrize("experts", [0, 4])
def test_captured_readings_of_several_lengths_share_a_cache_that_grows(device, experts):
    # the tables that the graphs were captured over are replaced in between (both Writers' at the same rounds: how the
    # attention is cut over workgroups goes by the tables' size)
    config = DecoderConfig(layers=2, d_model=128, heads=2, head_dim=64, ffn=64, vocab=64, experts=experts,
                           experts_per_token=min(experts, 2))
    w = random_weights(config, seed=1, std=0.05)
    eager, captured = (written(config, w, (4, 3, 4, 5), 150, c, device, bool(experts), {0: 512, 40: 1500, 90: 3100})
                       for c in (False, True))
    assert len(captured._reads) == 3 and captured.cache.capacity == 3100
    assert captured.histories == eager.histories
    assert torch.equal(captured.cache.lengths, eager.cache.lengths)
    for b, length in enumerate(eager.cache.lengths.tolist()):
        for mine, theirs in zip(captured.cache.tables, eager.cache.tables):
            assert torch.equal(mine[b, :length], theirs[b, :length])
        if experts:
            assert torch.equal(captured.routes[:, b, :length], eager.routes[:, b, :length])
