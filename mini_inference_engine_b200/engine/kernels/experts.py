"""Routed feed-forwards: the choice of every token's experts (``csrc/expert_routing.cu``) and the experts' products
(``csrc/expert_mlp.cu``)."""

from __future__ import annotations

import functools

import torch

from ... import _lib
from .linear import MAX_PRODUCT, activation_code, check_rows, check_sizes, check_status, check_tangents

MAX_EXPERTS = 1024  # MIE_MAX_EXPERTS
MAX_TOP_K = 32      # MIE_MAX_TOP_K
MAX_GROUPS = 32
MAX_PAIRS = 1 << 30  # of tokens and their experts
SCORES = {"softmax": 0, "sigmoid": 1}  # MIE_SCORES_*


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(tokens: int, top_k: int, experts: int, width: int, ff: int) -> int:
    return int(_lib.load().mie_expert_scratch_bytes(tokens, top_k, experts, width, ff))


def _check_choice(experts: int, top_k: int, groups: int, top_groups: int, group_best: int) -> None:
    """What the library refuses too, ahead of the results' allocation and of calls without tokens."""

    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"routing takes up to {MAX_EXPERTS} experts, not {experts}")
    if not 1 <= groups <= MAX_GROUPS or experts % groups or not 1 <= top_groups <= groups:
        raise ValueError(f"{experts} experts cannot be chosen from {top_groups} of {groups} groups")
    size = experts // groups
    if not 1 <= group_best <= min(2, size):
        raise ValueError("groups are judged by their best one or two")
    if not 1 <= top_k <= min(MAX_TOP_K, top_groups * size):
        raise ValueError(f"cannot choose {top_k} experts from {top_groups} groups of {size}")


def route_experts(logits: torch.Tensor, top_k: int, *, scores: str = "softmax", bias: torch.Tensor | None = None,
                  groups: int = 1, top_groups: int = 1, group_best: int = 1, renormalize: bool = True,
                  scale: float = 1.0, status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(ids int32 [tokens, top_k], weights fp32 [tokens, top_k])`` of router logits ``[tokens, experts]`` (bf16, fp16 or
    fp32).

    ``s = softmax(logits)`` or ``sigmoid(logits)``; the choice goes by ``s + bias`` (fp32 ``[experts]``, for balance), the
    weights are ``s`` of the chosen, over their sum with ``renormalize``, times ``scale``.  With ``groups`` the experts are
    that many equal runs, of which the ``top_groups`` whose ``group_best`` (1 or 2) best choices add up to most are chosen
    from.  Best first, equal choices by their index.  Without ``bias``, and without groups or with ``group_best`` 1, the order
    is that of the logits; otherwise that of the choices in 64 bits (in which sigmoids of 40 and 41, for instance, are equal).
    A logit of ``-inf`` masks an expert: it comes after all others, with weight 0.  A NaN logit makes the token's weights
    NaN."""

    del status  # every input is valid on the device
    check_tangents(logits, bias)
    check_sizes(*logits.shape, top_k, groups, top_groups, group_best)
    if logits.ndim != 2 or logits.dtype not in _lib.DTYPE_CODES:
        raise ValueError("route_experts takes CUDA logits [tokens, experts] in bf16, fp16 or fp32")
    if scores not in SCORES:
        raise ValueError(f"unknown scores {scores!r}: one of {', '.join(SCORES)}")
    (tokens, experts), top_k = logits.shape, int(top_k)
    _check_choice(experts, top_k, groups, top_groups, group_best)
    if not logits.is_cuda:
        raise ValueError("route_experts takes CUDA logits [tokens, experts] in bf16, fp16 or fp32")
    if experts > 1 and logits.stride(1) != 1 or tokens > 1 and logits.stride(0) < experts:
        raise ValueError(f"logits need dense rows that do not overlap, not strides {list(logits.stride())}")
    if bias is not None and (bias.dtype is not torch.float32 or tuple(bias.shape) != (experts,) or
                             not bias.is_contiguous() or bias.device != logits.device):
        raise ValueError(f"bias must be dense fp32 [{experts}] on the logits' device")
    if torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError("route_experts has no gradient")
    device = logits.device
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    if tokens == 0:
        return ids, weights
    with _lib.on_device(device):
        _lib.check(_lib.load().mie_route_experts(
            logits.data_ptr(), logits.stride(0) if tokens > 1 else experts, _lib.DTYPE_CODES[logits.dtype],
            None if bias is None else bias.data_ptr(), SCORES[scores], tokens, experts, top_k, groups, top_groups,
            group_best, int(renormalize), float(scale), ids.data_ptr(), weights.data_ptr(), _lib.stream_arg(device)))
    return ids, weights


def expert_mlp(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor, *,
               activation: str = "silu", residual: torch.Tensor | None = None, status: torch.Tensor) -> torch.Tensor:
    """``residual + sum_j weights[:, j] down_e (act(gate_e x) * (up_e x))``, ``e = ids[:, j]``, of bf16 rows ``x [tokens,
    width]``.

    ``gate_up [experts, 2 ff, width]`` holds an expert's gates and then its ups, ``down [experts, width, ff]``; ``ids``
    (int32 or int64) and ``weights`` (fp32) are ``[tokens, top_k]``, as ``route_experts`` gives them.  An id of -1 is no
    expert (padding rows); another outside the pool is skipped and reported through ``status``.  An expert may be named
    twice by a token."""

    if x.ndim != 2 or gate_up.ndim != 3 or down.ndim != 3 or ids.ndim != 2:
        raise ValueError("expert_mlp takes x [tokens, width], ids [tokens, top_k], gate_up [experts, 2 ff, width] and "
                         "down [experts, width, ff]")
    check_tangents(x, weights, gate_up, down, residual)
    code, device = activation_code(activation), x.device
    (tokens, width), (experts, double_ff, _), top_k = x.shape, gate_up.shape, int(ids.shape[1])
    ff = double_ff // 2
    check_sizes(tokens, width, experts, double_ff, top_k, most=MAX_PRODUCT)
    if not (1 <= experts <= MAX_EXPERTS and 1 <= top_k <= MAX_TOP_K and width >= 1 and ff >= 1):
        raise ValueError(f"expert_mlp takes up to {MAX_EXPERTS} experts, {MAX_TOP_K} of them a token, and rows of one entry or "
                         f"more, not {top_k} of {experts} experts of {width} x {ff}")
    if tokens * top_k >= MAX_PAIRS:
        raise ValueError(f"too many (token, expert) pairs: {tokens} x {top_k}")
    ldx, _ = check_rows("x", x, (tokens, width), device)
    gate_up_row, gate_up_expert = check_rows("gate_up", gate_up, (experts, 2 * ff, width), device)
    down_row, down_expert = check_rows("down", down, (experts, width, ff), device)
    ldr = 0 if residual is None else check_rows("residual", residual, (tokens, width), device)[0]
    if ids.dtype not in (torch.int32, torch.int64) or ids.shape[0] != tokens or ids.device != device:
        raise ValueError(f"ids must be int32 or int64 [{tokens}, top_k] on the device of x")
    if weights.dtype is not torch.float32 or weights.shape != ids.shape or weights.device != device or \
            not weights.is_contiguous():
        raise ValueError(f"weights must be dense fp32 {list(ids.shape)} on the device of x")
    if weights.requires_grad and torch.is_grad_enabled():
        raise ValueError("weights requires a gradient: this operator has none")
    check_status(status, device)
    out = torch.empty((tokens, width), dtype=torch.bfloat16, device=device)
    if tokens == 0:
        return out
    with _lib.on_device(device):
        scratch = torch.empty(_scratch_bytes(tokens, top_k, experts, width, ff), dtype=torch.uint8, device=device)
        _lib.check(_lib.load().mie_expert_mlp(
            x.data_ptr(), ldx, _lib.index_arg(ids), weights.data_ptr(), gate_up.data_ptr(), gate_up_row, gate_up_expert,
            down.data_ptr(), down_row, down_expert, None if residual is None else residual.data_ptr(), ldr, out.data_ptr(),
            width, tokens, top_k, experts, width, ff, code, scratch.data_ptr(), scratch.numel(), status.data_ptr(),
            _lib.stream_arg(device)))
    return out


__all__ = ["MAX_EXPERTS", "MAX_TOP_K", "SCORES", "expert_mlp", "route_experts"]
