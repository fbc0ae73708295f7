"""A decoder of experts over mixed layers in bf16 against the oracle, and the
log-probabilities of what a captured verify step writes, from its own scores."""

import pytest
import torch

from oracle.decoder import Decoder as Oracle
from wpt_amd import sampling
from wpt_amd.decoder import EXACT, WINDOW, DecoderConfig, MQADecoder, random_weights
from wpt_amd.step import VerifyStep

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
CONFIG = DecoderConfig(layers=4, d_model=256, heads=4, head_dim=64, ffn=96, vocab=512, kinds=(WINDOW, EXACT, EXACT, WINDOW),
                       window=16, rope_dims=32, experts=12, experts_per_token=4)


@pytest.mark.parametrize("B, T", [(2, 5), (7, 30), (3, 120), (1, 1)])
def test_bf16_readings_over_mixed_layers_match_the_oracle(device, B, T):
    # tolerances as the exact layers' decoders of experts have them: the oracle takes the recorded routes, whose logits on
    # its own stream come within 5e-2 of its k-th largest; scores within 2e-2 of their largest
    w = random_weights(CONFIG, seed=3, std=0.05)
    rounded = {n: v if n.endswith(("norm", "sink", "router")) else v.to(BF16).float() for n, v in w.items()}
    ora = Oracle(rounded, CONFIG.layers, CONFIG.heads, CONFIG.head_dim, CONFIG.kinds, CONFIG.window, CONFIG.rope_dims,
                 CONFIG.rope_base, CONFIG.top_k, experts_per_token=CONFIG.experts_per_token)
    model = MQADecoder(CONFIG, w, dtype=BF16)
    ids = torch.randint(0, CONFIG.vocab, (B, T), generator=torch.Generator().manual_seed(B))
    cache = model.new_cache(B, routes=True, capacity=T)
    scores, _ = model.extend(ids, cache)
    for i in range(CONFIG.layers):
        ora.given_routes[i] = cache.routes[i, :, :T].cpu()
        assert int(ora.given_routes[i].min()) >= 0
    expected = ora.extend(ids, ora.new_cache(B))[0]
    for i in range(CONFIG.layers):
        own, x = ora.routed[i]
        logits = x.double() @ ora.w[f"layers.{i}.router"].double().T
        last = logits.gather(-1, own.long()).amin(-1)
        assert bool((logits.gather(-1, ora.given_routes[i].long()).amin(-1) >= last - 5e-2).all())
    assert float((scores.cpu().double() - expected.double()).abs().max()) <= 2e-2 * float(expected.abs().max())


def test_a_captured_step_s_scores_give_what_it_wrote(device):
    B, k, temperature = 4, 3, 0.8
    model = MQADecoder(CONFIG, random_weights(CONFIG, seed=7, std=0.05), dtype=BF16)
    cache = model.new_cache(B, routes=True, capacity=256)
    prompt = torch.randint(0, CONFIG.vocab, (B, 20), generator=torch.Generator().manual_seed(2))
    model.extend(prompt, cache)
    step = VerifyStep(model, cache, k, temperature=temperature)
    step.feeds.copy_(prompt[:, :k + 1])
    step.capture(warmup=1)
    for _ in range(5):
        before = cache.lengths.clone()
        tokens, counts = step.replay()
        lp, entropy, _, _ = sampling.log_probs(step.scores, tokens, temperature=temperature)
        plain = torch.log_softmax(step.scores.double() / temperature, -1)
        written = torch.arange(k + 1, device=device) < counts[:, None]
        assert bool((tokens[written] >= 0).all()) and bool((tokens[~written] == -1).all())
        at = plain.gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
        assert torch.allclose(lp.double(), torch.where(written, at, 0.0), atol=1e-5)
        assert torch.allclose(entropy.double(), -(plain.exp() * plain).sum(-1), atol=1e-5)
        assert torch.equal(cache.lengths, before + counts)
        for b, length in enumerate(cache.lengths.tolist()):  # the routes of what stays
            assert int(cache.routes[:, b, :length].min()) >= 0
