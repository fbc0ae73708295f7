"""A mixture of experts on the GPU (libwptv's wptv_route, wptv_experts and
wptv_mixture, include/wptv.h): a linear router's choice of experts for each
token, and the chosen experts' SwiGLU blocks, for the few rows of a verify step
(any number is taken).

    chosen, gates = route(x, router, k)             each token's k experts and their shares
    y = feed_forward(x, weights, chosen, gates)     the gated sum of their blocks
    y, chosen, gates = mixture(x, router, weights, k)   both in one call

The decoder's layers with experts call mixture_parts, whose terms the residual
add + norm sums (decoder.DecoderConfig.experts).  These forms are forward-only,
as the attention's."""

import ctypes

import torch

from . import _lib
from ._lib import KernelUnavailable, check, ptr
from .kernels import _forward_only, _index, _no_tangents

__all__ = ["ExpertWeights", "route", "feed_forward", "feed_forward_parts", "mixture", "mixture_parts"]


def _input(x, what):
    """x (B, T, D) as the kernels read it, and (B, T, D)."""
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be (B, T, D); got {tuple(x.shape)}")
    dtype = _lib.dtype_code(x.dtype)
    if x.device.type != "cuda":
        raise KernelUnavailable(f"the HIP experts run on a GPU; x is on {x.device}")
    x = x.contiguous()
    if x.data_ptr() % 16:  # a slice of a larger tensor: rows start on 16 bytes
        x = x.clone()
    return x, dtype, x.shape


def _router(router, bias, counts, x, k):
    """(router, bias, counts) checked and laid out, and the experts' count."""
    B, T, D = x.shape
    if router.dim() != 2 or router.shape[1] != D or router.dtype != torch.float32 or router.device != x.device:
        raise ValueError(f"router must be FP32 (E, D={D}) on {x.device}; got {router.dtype} {tuple(router.shape)}")
    E = router.shape[0]
    if not 1 <= k <= E:
        raise ValueError(f"k = {k} of {E} experts")
    router = router.contiguous()
    if router.data_ptr() % 16:
        router = router.clone()
    if bias is not None:
        if bias.shape != (E,) or bias.dtype != torch.float32 or bias.device != x.device:
            raise ValueError(f"bias must be FP32 (E={E},) on {x.device}; got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    if counts is not None:
        if counts.is_floating_point() or counts.dtype == torch.bool:
            raise ValueError(f"counts are whole numbers; got {counts.dtype}")
        counts = _index(counts, (B,), "counts", x.device)
    return router, bias, counts, E


class ExpertWeights:
    """E experts' SwiGLU blocks, laid out once in the order the products read
    them (wptv_pack_experts): gate_up (E, 2F, D), each expert's F gate rows and
    then its F up rows, and down (E, D, F), bf16 or FP32 on the GPU.  The
    matrices themselves are not kept."""

    def __init__(self, gate_up, down):
        if gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[1] % 2:
            raise ValueError(f"gate_up must be (E, 2F, D) and down (E, D, F); got {tuple(gate_up.shape)}, "
                             f"{tuple(down.shape)}")
        E, F2, D = gate_up.shape
        F = F2 // 2
        if down.shape != (E, D, F) or down.dtype != gate_up.dtype:
            raise ValueError(f"down must be (E={E}, D={D}, F={F}) in gate_up's {gate_up.dtype}; got {down.dtype} "
                             f"{tuple(down.shape)}")
        dtype = _lib.dtype_code(gate_up.dtype)
        device = gate_up.device
        if device.type != "cuda" or down.device != device:
            raise KernelUnavailable(f"the HIP experts run on one GPU; the weights are on {device} and {down.device}")
        self.experts, self.width, self.features, self.dtype, self.device = E, D, F, gate_up.dtype, device
        # stands for matrices that ask for gradients, which no backward pass of these forms gives
        self.trained = torch.empty(0, requires_grad=True) if gate_up.requires_grad or down.requires_grad else None
        _no_tangents(gate_up, down)
        gate_up, down = gate_up.detach().contiguous(), down.detach().contiguous()
        sizes = ctypes.c_size_t(0), ctypes.c_size_t(0)
        check(_lib.lib().wptv_experts_packed(D, F, dtype, ctypes.byref(sizes[0]), ctypes.byref(sizes[1])),
              "ExpertWeights")
        with _lib.on(device):
            self.gate_up = torch.empty(E * sizes[0].value, dtype=torch.uint8, device=device)
            self.down = torch.empty(E * sizes[1].value, dtype=torch.uint8, device=device)
            check(_lib.lib().wptv_pack_experts(ptr(gate_up), ptr(down), E, D, F, dtype, ptr(self.gate_up),
                                               ptr(self.down), _lib.stream(device)), "ExpertWeights")


def route(x, router, k, bias=None, counts=None):
    """Each token's k experts: (chosen (B, T, k) int32, gates (B, T, k) FP32).

    x (B, T, D) bf16 or FP32; router (E, D) FP32.  The logits l = x . router^T
    are formed and ranked in 64 bits: the k largest l + bias (bias (E,) FP32, a
    load-balanced router's; -inf takes an expert out, whatever its l), largest
    first, equal ones the lowest expert, a NaN the largest.  gates: the softmax of the chosen
    experts' l, without the bias.  counts (B,): the tokens read of each row, the
    others padding (None: all).  Where no expert is chosen (padding, or fewer
    than k above -inf) chosen is -1 and the gate 0."""
    k = int(k)
    x_, dtype, (B, T, D) = _input(x, "route")
    router, bias, counts, E = _router(router, bias, counts, x_, k)
    chosen = torch.empty(B, T, k, dtype=torch.int32, device=x.device)
    gates = torch.empty(B, T, k, dtype=torch.float32, device=x.device)
    with _lib.on(x.device):
        _, size = _lib.plan("wptv_route_workspace", "route", B * T, D, E)
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        check(_lib.lib().wptv_route(ptr(x_), dtype, ptr(router), ptr(bias), ptr(counts), B, T, D, E, k,
                                    ptr(chosen), ptr(gates), ptr(workspace), size, _lib.stream(x.device)), "route")
    return chosen, _forward_only(gates, x, router)


def _match(x, weights, what):
    if weights.dtype != x.dtype or weights.device != x.device or weights.width != x.shape[2]:
        raise ValueError(f"{what}: x must be (B, T, {weights.width}) {weights.dtype} on {weights.device} as the experts "
                         f"are; got {tuple(x.shape)} {x.dtype} on {x.device}")


def _result(x, size, k, parts):
    """(parts, y, workspace) of a call on x."""
    B, T, D = x.shape
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    if parts:
        return torch.empty(k, B * T, D, dtype=torch.float32, device=x.device), None, workspace
    return None, torch.empty(B, T, D, dtype=x.dtype, device=x.device), workspace


def _feed_forward(x, weights, chosen, gates, parts):
    x_, dtype, (B, T, D) = _input(x, "feed_forward")
    _match(x_, weights, "feed_forward")
    k = chosen.shape[-1]
    for name, t, kind in (("chosen", chosen, torch.int32), ("gates", gates, torch.float32)):
        if t.shape != (B, T, k) or t.dtype != kind or t.device != x.device or k == 0:
            raise ValueError(f"{name} must be {kind} (B={B}, T={T}, k) on {x.device}; got {t.dtype} {tuple(t.shape)}")
    chosen_, gates_ = chosen.contiguous(), gates.contiguous()  # copies of views, held over the call
    with _lib.on(x.device):
        _, size = _lib.plan("wptv_experts_workspace", "feed_forward", B * T, D, weights.features, k, dtype, int(parts))
        out, y, workspace = _result(x_, size, k, parts)
        check(_lib.lib().wptv_experts(ptr(x_), dtype, ptr(weights.gate_up), ptr(weights.down), ptr(chosen_),
                                      ptr(gates_), B * T, D, weights.experts, k, weights.features, ptr(out), ptr(y),
                                      ptr(workspace), size, _lib.stream(x.device)), "feed_forward")
    return _forward_only(out if parts else y, x, gates, weights.trained)


def feed_forward(x, weights, chosen, gates):
    """The gated sum of each token's experts: y (B, T, D) in x's dtype, the sum
    over j of gates[..., j] down_e (silu(gate_e x) * (up_e x)), e = chosen[..., j]
    (route's; a choice outside 0 .. E - 1 adds nothing).  weights: ExpertWeights.
    FP32 sums; gates silu(g) u is rounded once to the dtype between the products."""
    return _feed_forward(x, weights, chosen, gates, False)


def feed_forward_parts(x, weights, chosen, gates):
    """feed_forward's terms, (k, B T, D) FP32, for layers.add_rms_norm_parts
    (k <= 8), which adds them to the residual stream."""
    return _feed_forward(x, weights, chosen, gates, True)


def _mixture(x, router, weights, k, bias, counts, parts):
    k = int(k)
    x_, dtype, (B, T, D) = _input(x, "mixture")
    _match(x_, weights, "mixture")
    router_, bias, counts, E = _router(router, bias, counts, x_, k)
    if E != weights.experts:
        raise ValueError(f"the router chooses among {E} experts; the weights hold {weights.experts}")
    device = x.device
    chosen = torch.empty(B, T, k, dtype=torch.int32, device=device)
    gates = torch.empty(B, T, k, dtype=torch.float32, device=device)
    with _lib.on(device):
        _, size = _lib.plan("wptv_mixture_workspace", "mixture", B * T, D, E, weights.features, k, dtype, int(parts))
        out, y, workspace = _result(x_, size, k, parts)
        check(_lib.lib().wptv_mixture(ptr(x_), dtype, ptr(router_), ptr(bias), ptr(counts), B, T, D, E, k,
                                      weights.features, ptr(weights.gate_up), ptr(weights.down), ptr(chosen), ptr(gates),
                                      ptr(out), ptr(y), ptr(workspace), size, _lib.stream(device)), "mixture")
    return _forward_only(out if parts else y, x, router, weights.trained), chosen, _forward_only(gates, x, router)


def mixture(x, router, weights, k, bias=None, counts=None):
    """A whole mixture-of-experts layer: route, then feed_forward on its choice,
    in one call.  Returns (y (B, T, D), chosen (B, T, k), gates (B, T, k))."""
    return _mixture(x, router, weights, k, bias, counts, False)


def mixture_parts(x, router, weights, k, bias=None, counts=None):
    """mixture with the terms (k, B T, D) FP32 in y's place (feed_forward_parts)."""
    return _mixture(x, router, weights, k, bias, counts, True)
