"""Selection of experts: scores by softmax or sigmoid, a balance bias that only selects, groups, top-k, renormalised and
scaled weights; and the gradient of the weights.

``select_experts`` is the router of the families whose scores are not a plain softmax (the GLM layer calls it through
``ss::select_experts``); ``ops/moe.py: route`` is the narrower form that the softmax families' fused expert layer uses.
What it returns goes to ``moe.Layout`` and the grouped products as it is. Reference: sigmoid scores with a selection bias in
packages/workloads/src/shadowspill_workloads/models/shared/glm/moe.py:9-47.
"""
from __future__ import annotations

import torch

from . import _lib, reference
from . import functional as F

_P, _I, _L, _F = _lib.c_p, _lib.c_int, _lib.c_ll, _lib.c_f
_lib.register("ss_select_experts", [_P, _I, _L, _P, _I, _I, _I, _I, _I, _I, _I, _F, _P, _P, _P, _P])
_lib.register("ss_select_experts_bwd", [_P, _I, _L, _P, _P, _I, _I, _I, _I, _I, _F, _P, _P])

MAX_EXPERTS, MAX_GROUPS = 512, 32                     # as the kernels have them
_SIGMOID = {"softmax": 0, "sigmoid": 1}


def _check(logits, k, scoring, groups=1, keep_groups=1):
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"router logits are [T, E] in fp32 or bf16, got {tuple(logits.shape)} {logits.dtype}")
    E = logits.shape[1]
    if scoring not in _SIGMOID:
        raise ValueError(f"unknown scoring {scoring!r}; known: {tuple(_SIGMOID)}")
    if not (1 <= groups <= MAX_GROUPS and E % groups == 0 and 1 <= keep_groups <= groups):
        raise ValueError(f"{E} experts do not fall into {groups} groups of which {keep_groups} are kept")
    if not (1 <= k <= keep_groups * (E // groups) and E <= MAX_EXPERTS):
        raise ValueError(f"cannot pick {k} of {keep_groups * (E // groups)} experts (of at most {MAX_EXPERTS})")


def select_experts(logits: torch.Tensor, k: int, *, scoring: str = "softmax", bias: torch.Tensor | None = None,
                   groups: int = 1, keep_groups: int = 1, renormalize: bool = True, scale: float = 1.0):
    """Logits [T,E] (fp32 or bf16) -> (ids int32 [T,k], weights fp32 [T,k], counts int32 [E]).

    The picks are the ``k`` largest ``score + bias`` among the ``keep_groups`` groups of consecutive experts whose two
    largest sum highest, in decreasing order, ties to the lowest index; they are those of keys in 64 bits. Experts whose key is
    -inf or NaN come last, so that the ids of a token are always ``k`` different experts. The weights are the picks' scores
    (without the bias), divided by their sum (+ 1e-20) if ``renormalize``, times ``scale``; a token whose logits are all -inf
    gets weights of zero under softmax, one with a NaN or +inf gets NaN. At most 512 experts; ``k`` has no bound of its own (above 32 the
    picks are made one by one in 64 bits, which takes several times as long)."""
    host = F._host(logits)
    if host is not None:
        got = host.select_experts(logits, k, _SIGMOID.get(scoring, -1), bias, groups, keep_groups, bool(renormalize), scale)
        if got is not NotImplemented:
            return got
    _check(logits, k, scoring, groups, keep_groups)
    T, E = logits.shape
    if bias is not None and (bias.shape != (E,) or bias.dtype != torch.float32 or bias.device != logits.device):
        raise ValueError("the selection bias is fp32 [E] on the logits' device")
    if not F._cuda(logits):
        return reference.select_experts(logits, k, scoring, bias, groups, keep_groups, renormalize, scale)
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    dev = logits.device
    ids = torch.empty((T, k), dtype=torch.int32, device=dev)
    weights = torch.empty((T, k), dtype=torch.float32, device=dev)
    counts = torch.empty(E, dtype=torch.int32, device=dev)
    with F._device_of(logits):
        _lib.check(_lib.lib().ss_select_experts(
            logits.data_ptr(), int(logits.dtype == torch.bfloat16), max(logits.stride(0), E), F._ptr(bias), T, E, k, groups,
            keep_groups, _SIGMOID[scoring], int(renormalize), float(scale), ids.data_ptr(), weights.data_ptr(),
            counts.data_ptr(), _lib.stream_ptr()), "ss_select_experts")
    return ids, weights, counts


def select_experts_bwd(logits: torch.Tensor, ids: torch.Tensor, dweights: torch.Tensor, *, scoring: str = "softmax",
                       renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``select_experts``'s weights (``dweights`` fp32 [T,k]) as a gradient of the logits, in their type; the
    picks and the bias are constants."""
    host = F._host(logits)
    if host is not None:
        got = host.select_experts_bwd(logits, ids, dweights, _SIGMOID.get(scoring, -1), bool(renormalize), scale)
        if got is not NotImplemented:
            return got
    if ids.dim() != 2 or ids.dtype != torch.int32 or dweights.shape != ids.shape or ids.shape[0] != logits.shape[0]:
        raise ValueError("ids are int32 [T, k] and dweights has their shape")
    if ids.device != logits.device or dweights.device != logits.device:
        raise ValueError("logits, ids and dweights are on one device")
    _check(logits, ids.shape[1], scoring)
    if not F._cuda(logits):
        return reference.select_experts_bwd(logits, ids, dweights, scoring, renormalize, scale)
    T, E = logits.shape
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    ids, dweights = ids.contiguous(), dweights.float().contiguous()
    out = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    with F._device_of(logits):
        _lib.check(_lib.lib().ss_select_experts_bwd(
            logits.data_ptr(), int(logits.dtype == torch.bfloat16), max(logits.stride(0), E), ids.data_ptr(),
            dweights.data_ptr(), T, E, ids.shape[1], _SIGMOID[scoring], int(renormalize), float(scale), out.data_ptr(),
            _lib.stream_ptr()), "ss_select_experts_bwd", int(T > 0))
    return out
