"""The mixture of experts and the log-probabilities off the GPU: their oracles by
hand, and what the entry points refuse before anything runs."""

import ctypes
import json
import math

import pytest
import torch

from oracle import experts as oracle
from oracle import log_probs as oracle_log_probs
from wpt_amd import _lib, experts, folder, sampling
from wpt_amd.decoder import DecoderConfig, random_weights

INF, NAN = math.inf, math.nan


def test_the_oracle_chooses_and_shares_as_worked_by_hand():
    x = torch.tensor([[[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]]])
    router = torch.tensor([[0.0, 1.0], [math.log(3), 1.0], [-5.0, 1.0]])
    chosen, gates = oracle.route(x, router, 2)
    assert chosen.tolist() == [[[1, 0], [0, 1], [1, 0]]]  # the second token's three logits are equal
    assert gates[0, 0].tolist() == pytest.approx([0.75, 0.25]) and gates[0, 1].tolist() == [0.5, 0.5]
    # a bias moves the choice, not the gates; -inf takes an expert out; padding chooses none
    chosen, gates = oracle.route(x, router, 2, torch.tensor([0.0, -INF, 0.0]), torch.tensor([2]))
    assert chosen.tolist() == [[[0, 2], [0, 2], [-1, -1]]]
    assert gates[0, 0].tolist() == pytest.approx([1 / (1 + math.exp(-5)), 1 / (1 + math.exp(5))])
    assert gates[0, 2].tolist() == [0, 0]
    chosen, _ = oracle.route(x, router, 2, torch.tensor([-INF, -INF, 0.0]))
    assert chosen[0, 0].tolist() == [2, -1]
    chosen, _ = oracle.route(torch.tensor([[[NAN, 0.0]]]), router, 2)
    assert chosen.tolist() == [[[0, 1]]]


def test_the_oracle_s_blocks_are_their_formula():
    g = torch.Generator().manual_seed(0)
    x, gate_up, down = (torch.randn(*s, generator=g) for s in ((1, 2, 8), (3, 10, 8), (3, 8, 5)))
    chosen, gates = torch.tensor([[[2, 0], [-1, 1]]], dtype=torch.int32), torch.tensor([[[0.5, 0.25], [0.0, 1.0]]])

    def block(e, row):
        h = gate_up[e].double() @ row.double()
        return down[e].double() @ (torch.nn.functional.silu(h[:5]) * h[5:])

    y, bound = oracle.feed_forward(x, gate_up, down, chosen, gates)
    assert torch.allclose(y[0, 0], 0.5 * block(2, x[0, 0]) + 0.25 * block(0, x[0, 0]), atol=1e-14)
    assert torch.allclose(y[0, 1], block(1, x[0, 1]), atol=1e-14)
    assert bool((bound > 0).all()) and float(bound.max()) < 1e-4


def test_the_oracle_s_log_probabilities_by_hand():
    scores = torch.tensor([[[0.0, math.log(2), 0.0, -INF], [1.0, NAN, INF, NAN], [-INF] * 4, [3.0, -0.0, 0.0, 3.0]]])
    tokens = torch.tensor([[1, 0, 0, -1]])
    lp, entropy, ids, best = oracle_log_probs.log_probs(scores, tokens, top=3)
    assert lp[0, 0].item() == pytest.approx(math.log(0.5)) and lp[0, 3].item() == 0
    assert math.isnan(lp[0, 1]) and math.isnan(lp[0, 2]) and math.isnan(entropy[0, 1]) and math.isnan(entropy[0, 2])
    assert entropy[0, 0].item() == pytest.approx(1.5 * math.log(2))
    assert ids.tolist() == [[[1, 0, 2], [1, 3, 2], [0, 1, 2], [0, 3, 1]]]
    assert best[0, 0].tolist() == pytest.approx([math.log(0.5), math.log(0.25), math.log(0.25)])
    lp, entropy, _, _ = oracle_log_probs.log_probs(scores[:, :1], tokens[:, :1], temperature=0.5)
    assert lp.item() == pytest.approx(math.log(4 / 6))


def packed(*arguments):
    sizes = ctypes.c_size_t(0), ctypes.c_size_t(0)
    status = _lib.lib().wptv_experts_packed(*arguments, *map(ctypes.byref, sizes))
    return status, sizes[0].value, sizes[1].value


def test_the_packed_sizes_hold_the_padded_matrices():
    assert packed(2048, 704, _lib.WPTV_BF16) == (0, 2 * 704 * 2048 * 2, 2048 * 704 * 2)
    # features to the products' 32 columns (FP32: 16), inputs to 32 (16), outputs to 32
    assert packed(40, 33, _lib.WPTV_BF16) == (0, 2 * 64 * 64 * 2, 64 * 64 * 2)
    assert packed(40, 33, _lib.WPTV_F32) == (0, 2 * 48 * 48 * 4, 64 * 48 * 4)


@pytest.mark.parametrize("arguments, status", [
    ((36, 8, 1), -3), ((0, 8, 1), -1), ((64, 0, 1), -1), ((64, 8, 7), -3), ((64, (1 << 20) + 1, 0), -3)])
def test_weights_of_shapes_without_a_kernel_are_refused(arguments, status):
    assert packed(*arguments)[0] == status


@pytest.mark.parametrize("B, T, D, E, k, dtype, status", [
    (-1, 1, 64, 4, 2, 1, -1), (1, 1, 60, 4, 2, 1, -3), (1, 1, 64, 4, 5, 1, -1), (1, 1, 64, 4, 0, 1, -1),
    (1, 1, 64, 513, 2, 1, -3), (1, 1, 64, 40, 17, 1, -3), (1, 1, 64, 4, 2, 5, -3), (4097, 4097, 64, 4, 2, 1, -3)])
def test_routes_of_shapes_without_a_kernel_are_refused(B, T, D, E, k, dtype, status):
    library = _lib.lib()
    assert library.wptv_route(16, dtype, 16, None, None, B, T, D, E, k, 16, 16, 16, 1 << 40, None) == status
    assert library.wptv_mixture(16, dtype, 16, None, None, B, T, D, E, k, 64, 16, 16, 16, 16, None, 16, 16, 1 << 40,
                                None) == status


@pytest.mark.parametrize("D, E, k, F", [(448, 37, 4, 2395), (64, 8, 2, 4000), (2048, 64, 8, 704), (9000, 16, 1, 40)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_a_workspace_is_enough_for_fewer_rows(D, E, k, F, dtype):
    library, size = _lib.lib(), ctypes.c_size_t()
    last = [0, 0]
    for rows in [*range(0, 700), *range(700, 40000, 997)]:
        assert library.wptv_experts_workspace(rows, D, F, k, dtype, 0, ctypes.byref(size)) == 0
        assert size.value >= last[0]
        last[0] = size.value
        assert library.wptv_route_workspace(rows, D, E, ctypes.byref(size)) == 0
        assert size.value >= last[1]
        last[1] = size.value


def test_null_and_misaligned_pointers_and_small_workspaces_are_refused():
    library = _lib.lib()
    assert library.wptv_route(None, 1, 16, None, None, 1, 1, 64, 4, 2, 16, 16, 16, 0, None) == -1
    assert library.wptv_route(8, 1, 16, None, None, 1, 1, 64, 4, 2, 16, 16, 16, 0, None) == -1
    assert b"16-byte" in library.wptv_last_error()
    assert library.wptv_route(16, 1, 16, None, None, 1, 1, 2048, 64, 2, 16, 16, 16, 63, None) == -1
    assert library.wptv_route(16, 1, 16, None, None, 1, 1, 2048, 64, 2, 16, 16, None, 1 << 40, None) == -1
    assert b"workspace" in library.wptv_last_error()

    def products(parts=None, y=16, workspace=16, size=1 << 30, x=16, F=64, rows=3):
        return library.wptv_experts(x, 1, 16, 16, 16, 16, rows, 64, 4, 2, F, parts, y, workspace, size, None)

    assert products(parts=16) == -1 and products(y=None) == -1  # one of the two results
    assert products(x=None) == -1 and products(x=24) == -1 and products(F=0) == -1
    assert products(workspace=None) == -1 and products(size=100) == -1
    assert b"workspace" in library.wptv_last_error()
    assert products(rows=0) == 0
    assert library.wptv_pack_experts(16, None, 4, 64, 64, 1, 16, 16, None) == -1


@pytest.mark.parametrize("B, T, V, top, status", [
    (1, 1, 10, 11, -1), (1, 1, 0, 0, -1), (1, 1, 100, 65, -3), (-1, 1, 10, 0, -1), (1, 1, (1 << 24) + 1, 0, -3),
    (70000, 70000, 10, 0, -3), (1, 1, 10, -1, -1)])
def test_log_probs_of_shapes_without_a_kernel_are_refused(B, T, V, top, status):
    size = ctypes.c_size_t(0)
    library = _lib.lib()
    assert library.wptv_log_probs_workspace(B, T, V, top, ctypes.byref(size)) == status
    assert library.wptv_log_probs(16, V, V, 0, 16, 1.0, B, T, V, top, 16, 16, 16, 16, None, 0, None) == status


def test_log_probs_refuses_temperatures_types_and_null_pointers():
    library = _lib.lib()

    def call(dtype=0, temperature=1.0, ids=16, tokens=16, B=1):
        return library.wptv_log_probs(16, 10, 10, dtype, tokens, temperature, B, 1, 10, 2, 16, 16, ids, 16, None, 0, None)

    assert call(temperature=0.0) == -1 and call(temperature=-1.0) == -1
    assert call(temperature=NAN) == -1 and call(temperature=INF) == -1
    assert call(dtype=3) == -3 and call(ids=None) == -1 and call(tokens=None) == -1
    assert call(B=0) == 0


def test_tensors_off_the_gpu_and_mismatched_ones_are_refused():
    x, router = torch.zeros(1, 2, 64), torch.zeros(4, 64)
    with pytest.raises(_lib.KernelUnavailable):
        experts.route(x, router, 2)
    with pytest.raises(_lib.KernelUnavailable):
        experts.ExpertWeights(torch.zeros(2, 16, 64), torch.zeros(2, 64, 8))
    with pytest.raises(ValueError):
        experts.ExpertWeights(torch.zeros(2, 15, 64), torch.zeros(2, 64, 8))
    with pytest.raises(ValueError):
        experts.ExpertWeights(torch.zeros(2, 16, 64), torch.zeros(2, 64, 9))
    with pytest.raises(ValueError):
        experts.route(x[0], router, 2)
    with pytest.raises(NotImplementedError):
        experts.route(x.half(), router, 2)
    with pytest.raises(_lib.KernelUnavailable):
        sampling.log_probs(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(ValueError):
        sampling.log_probs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long))


@pytest.mark.parametrize("experts_, per_token", [(-1, 0), (4, 0), (0, 2), (4, 5), (20, 9)])
def test_a_decoder_s_experts_are_whole(experts_, per_token):
    with pytest.raises(ValueError):
        DecoderConfig(layers=1, d_model=64, heads=1, head_dim=64, ffn=32, vocab=64, experts=experts_,
                      experts_per_token=per_token)


def test_a_folder_keeps_a_decoder_s_experts(tmp_path):
    config = DecoderConfig(layers=2, d_model=64, heads=1, head_dim=64, ffn=24, vocab=64, experts=5, experts_per_token=2)
    weights = random_weights(config, dtype=torch.bfloat16)
    assert weights["layers.1.gate_up"].shape == (5, 48, 64) and weights["layers.0.router"].dtype == torch.float32
    folder.save_folder(config, weights, tmp_path, b"{}", "test version 1")
    folder.save_drafter_record(tmp_path)
    loaded_config, loaded = folder.load_weights(tmp_path)
    assert loaded_config == config and all(torch.equal(weights[k], loaded[k]) for k in weights)
    # a folder written before there were experts
    fields = json.loads((tmp_path / folder.CONFIG_NAME).read_text())
    del fields["experts"], fields["experts_per_token"]
    (tmp_path / folder.CONFIG_NAME).write_text(json.dumps(fields))
    assert folder.load_weights(tmp_path)[0].experts == 0
