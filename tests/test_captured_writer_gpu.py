"""Writers whose steady rounds replay HIP graphs, against the same Writers read
eagerly: past the growth of what the cache holds."""

import pytest
import torch

from wpt_amd.decoder import WINDOW, DecoderConfig, MQADecoder, random_weights
from wpt_amd.writer import Writer

pytestmark = pytest.mark.gpu


class Guesses:
    """Drafts of so many tokens a round, in turn, each token's probability the
    same; a few of them are taken."""

    def __init__(self, lengths):
        self.lengths, self.round = lengths, 0

    def draft(self, model, texts, context, draft, probabilities, generator):
        L = self.lengths[self.round % len(self.lengths)]
        self.round += 1
        V = model.config.vocab
        tokens = torch.tensor([[(7 * t[-1] + 3 * j + len(t)) % V for j in range(L)] for t in texts], device=model.device)
        return tokens, torch.full((len(texts), L, V), 1.0 / V, device=model.device), None


def written(config, w, lengths, rounds, capture, device, routes):
    model = MQADecoder(config, w, dtype=torch.bfloat16)
    g = torch.Generator(device=device).manual_seed(2)
    writer = Writer(model, [3, 5, 7], 3, temperature=1.0, top_k=None, generator=g, drafter=Guesses(lengths), draft=max(lengths),
                    routes=routes, capture=capture)
    for _ in range(rounds):
        writer.write({}, {r: max(lengths) + 1 for r in range(3)})
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
