"""Fused projections and routed feed-forwards in 64 bits, with a bound on what the kernels' arithmetic may be off by.

Sums of k products in fp32 (in any order, roundings or truncations) are off by at most k 2^-23 of the terms' magnitude; the
activations are Lipschitz with 1.13 and off by a few roundings of the exponential's argument, 2^-21 (4 + 4 |argument|)
relative; a rounding to bf16 is off by 2^-8 of the value, one to fp16 by 2^-11.
"""

from __future__ import annotations

import math

import torch

BF16, FP16, FP32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -23
TINY = 1e-30


def activate(z, kind):
    """Value and error bound of the activation of exact ``z``."""

    if kind == "none":
        return z, torch.zeros_like(z)
    if kind == "relu":
        return z.clamp(min=0), torch.zeros_like(z)
    argument = z if kind == "silu" else 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
    value = z * torch.sigmoid(argument)
    return value, value.abs() * 2.0 ** -21 * (4.0 + 4.0 * argument.abs()) + TINY


def product(x, w, bias=None):
    """``x w^T + bias`` and its error bound, of 64-bit operands."""

    z = x @ w.t()
    error = w.shape[1] * FP32 * (x.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias
        error = error + FP32 * z.abs()
    return z, error


def gated(z, error, kind, is_gated):
    gate, up = z.chunk(2, dim=1) if is_gated else (z, None)
    gate_error, up_error = error.chunk(2, dim=1) if is_gated else (error, None)
    value, off = activate(gate, kind)
    off = off + 1.13 * gate_error
    if is_gated:
        off = off * up.abs() + value.abs() * up_error + off * up_error + FP32 * (value * up).abs()
        value = value * up
    return value, off


def fused_linear(x, w, bias, kind, is_gated, residual):
    """Exact result and bound of ``fused_linear``."""

    double = lambda t: None if t is None else t.double()  # noqa: E731
    value, off = gated(*product(double(x), double(w), double(bias)), kind, is_gated)
    if residual is not None:
        value = value + residual.double()
    off = off + FP32 * value.abs()
    return value, off + BF16 * (value.abs() + off) + TINY


def expert_mlp(x, ids, weights, gate_up, down, kind, residual):
    """Exact result and bound of ``expert_mlp``: a pair's weighted hidden row is rounded to bf16 and its row of the down
    product, before the sum over the pairs, to fp16 with the row's scale."""

    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device) if residual is None else residual.double()
    bound = torch.zeros_like(y)
    for e in range(gate_up.shape[0]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if not token.numel():
            continue
        hidden, off = gated(*product(x[token].double(), gate_up[e].double()), kind, True)
        factor = weights[token, slot, None].double()
        hidden, off = hidden * factor, off * factor.abs()
        off = off + FP32 * hidden.abs()
        off = off + BF16 * (hidden.abs() + off) + TINY
        row, sums = product(hidden, down[e].double())
        sums = sums * (1 + BF16) + off @ down[e].double().abs().t()
        sums = sums + FP16 * (row.abs() + sums) + 2.0 ** -23 * row.abs().amax(dim=1, keepdim=True)
        y.index_add_(0, token, row)
        bound.index_add_(0, token, sums + FP32 * row.abs())
    bound = bound + ids.shape[1] * FP32 * y.abs()
    return y, bound + BF16 * (y.abs() + bound) + TINY


def assert_within(out, exact, bound):
    off = (out.double() - exact).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} times the bound"
