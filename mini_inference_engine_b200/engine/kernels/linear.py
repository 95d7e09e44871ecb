"""bf16 projections: of decode-sized batches (``linear``, ``csrc/linear.cu``; everything else goes to the library product),
and of any number of rows with bias, activation or gate, and residual in the epilogue (``fused_linear``,
``csrc/fused_linear.cu``)."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ... import _lib

MAX_ROWS = 128  # MIE_LINEAR_MAX_ROWS


def linear_supported(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> bool:
    """Whether ``mie_linear`` takes the product: a few bf16 rows that do not overlap, 16-byte aligned, whole 16-byte
    groups, nothing that autograd follows."""

    if not (x.ndim == weight.ndim == 2 and 0 < x.shape[0] <= MAX_ROWS and x.dtype == weight.dtype == torch.bfloat16):
        return False
    (n, k), operands = weight.shape, [x, weight]
    if bias is not None:
        operands.append(bias)
        if bias.dtype != torch.bfloat16 or tuple(bias.shape) != (n,) or not bias.is_contiguous():
            return False
    return bool(x.is_cuda and x.shape[1] == k and n > 0 and k > 0 and k % 8 == 0
                and all(t.device == x.device for t in operands)
                and x.stride(1) == weight.stride(1) == 1 and x.stride(0) >= k and weight.stride(0) >= k
                and x.stride(0) % 8 == 0 and weight.stride(0) % 8 == 0
                and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0
                and not (torch.is_grad_enabled() and any(t.requires_grad for t in operands)))


def prefers_own_kernel(rows: int, n: int, k: int) -> bool:
    """Where the kernels of ``csrc/linear.cu`` beat the library product inside a launch chain (a norm before each
    product, weights from HBM; us, library / this): up to 8 rows everywhere (2048 x 2048 9.8 / 5.2, 4096 x 12288
    37.7 / 21.1; at worst even, 12288 x 2048 of 8 rows 13.2 / 13.4); up to 16 rows also small outputs (4096 x 2048
    8.9 / 7.8, but 16384 x 2048 16.3 / 17.0); up to 64 rows long sums (4096 x 12288 28.7 / 24.9, 256 x 4096 10.6 / 8.0,
    12288 x 4096 24.9 / 22.7, but 4096 x 2048 7.9 / 9.2), where the library cuts K too little.  At 128 rows reading the
    activations once per weight tile costs more than it saves (7.6 / 14)."""

    return rows <= 8 or (rows <= 16 and n <= 4096) or (rows <= 64 and k >= 4096)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, status: torch.Tensor,
           kernel: int = 0) -> torch.Tensor:
    """``x [rows, k] @ weight [n, k]^T (+ bias)`` for weights that no queued kernel of this library writes (a model's
    parameters).  ``kernel``: 0 picks, 1 / 2 name one of the two kernels."""

    if not linear_supported(x, weight, bias):
        return torch.nn.functional.linear(x, weight, bias)
    (rows, k), n = x.shape, int(weight.shape[0])
    if not (kernel or prefers_own_kernel(rows, n, k)):
        return torch.nn.functional.linear(x, weight, bias)
    out = torch.empty(rows, n, dtype=x.dtype, device=x.device)
    _lib.check(_lib.load().mie_linear(_lib.ptr(x), x.stride(0), _lib.ptr(weight), weight.stride(0), _lib.ptr(bias),
                                      _lib.ptr(out), n, rows, n, k, kernel, _lib.ptr(status),
                                      _lib.stream_arg(x.device)))
    return out


ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "relu": 3}  # MIE_ACT_*; gelu is its tanh form


def activation_code(name: str | None) -> int:
    code = ACTIVATIONS.get("none" if name is None else name)
    if code is None:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return code


def check_rows(name: str, tensor: torch.Tensor, shape: tuple[int, ...], device: torch.device) -> tuple[int, int]:
    """A bf16 CUDA tensor of ``shape`` whose rows are dense and do not overlap, and that autograd does not follow.  Returns
    the strides of a row and, of three dimensions, of a matrix; of dimensions with one entry, those of rows without gaps."""

    width = shape[-1]
    matrix = width * shape[-2] if len(shape) > 1 else width
    if (tensor.dtype is torch.bfloat16 and tensor.shape == shape and tensor.is_contiguous() and tensor.device == device
            and tensor.is_cuda and not tensor.requires_grad):
        return width, matrix
    if tensor.dtype is not torch.bfloat16 or tuple(tensor.shape) != shape:
        raise ValueError(f"{name} must be bf16 {list(shape)}, not {tensor.dtype} {list(tensor.shape)}")
    if tensor.device != device or device.type != "cuda":
        raise ValueError(f"{name} must be on the CUDA device of the other operands, not {tensor.device}")
    if tensor.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: this operator has none")
    strides = tensor.stride()
    dense, extent, leading = width == 1 or strides[-1] == 1, width, []
    for size, stride in zip(shape[-2::-1], strides[-2::-1]):
        if size > 1:
            dense, extent = dense and stride >= extent, stride * size
            leading.append(stride)
        else:
            leading.append(extent)
    if not dense:
        raise ValueError(f"{name} needs rows that are dense and do not overlap, not strides {list(strides)}")
    return leading[0] if leading else width, leading[1] if len(leading) > 1 else matrix


MAX_PRODUCT = (1 << 31) - 4096  # MIE_MAX_PRODUCT


def check_sizes(*sizes: int, most: int = (1 << 31) - 1) -> None:
    """The library takes sizes of 32 bits, of products up to ``MAX_PRODUCT``."""

    if max(sizes) > most or min(sizes) < -1 << 31:
        raise ValueError(f"sizes up to {most}, not {max(sizes, key=abs)}")


def check_tangents(*operands: torch.Tensor | None) -> None:
    """Refuses what forward-mode differentiation follows: its tangent would be lost.  There are none outside its levels."""

    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands):
        raise ValueError("an operand carries a forward-mode derivative: this operator has none")


def check_status(status: torch.Tensor, device: torch.device) -> None:
    if status.dtype is not torch.int32 or status.device != device or status.numel() < 1:
        raise ValueError(f"status must be an int32 word on {device}")


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str | None = None, gated: bool = False, residual: torch.Tensor | None = None,
                 status: torch.Tensor) -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` in one launch, for ``x [rows, k]`` and ``weight [n, k]``; with ``gated``,
    ``weight`` and ``bias`` have ``2 n`` rows, gates first, and the result is
    ``act(x gates^T + bias_g) * (x ups^T + bias_u) + residual``.  bf16 with fp32 sums, rounded once."""

    if x.ndim != 2 or weight.ndim != 2:
        raise ValueError("fused_linear takes rows [rows, k] and a weight [n, k]")
    check_tangents(x, weight, bias, residual)
    code, device = activation_code(activation), x.device
    rows, k = x.shape
    n = weight.shape[0]
    check_sizes(rows, n, k, most=MAX_PRODUCT)
    ldx, _ = check_rows("x", x, (rows, k), device)
    ldw, _ = check_rows("weight", weight, (n, k), device)
    if bias is not None:
        check_rows("bias", bias, (n,), device)
    if gated:
        if n % 2:
            raise ValueError(f"a gated weight has as many gates as ups, not {n} rows")
        n //= 2
    if n < 1 or k < 1:
        raise ValueError("fused_linear needs at least one column and one weight row")
    ldr = 0 if residual is None else check_rows("residual", residual, (rows, n), device)[0]
    check_status(status, device)
    out = torch.empty((rows, n), dtype=torch.bfloat16, device=device)
    if rows == 0:
        return out
    with _lib.on_device(device):
        _lib.check(_lib.load().mie_fused_linear(
            x.data_ptr(), ldx, weight.data_ptr(), ldw, None if bias is None else bias.data_ptr(),
            None if residual is None else residual.data_ptr(), ldr, out.data_ptr(), n, rows, n, k, code, gated,
            status.data_ptr(), _lib.stream_arg(device)))
    return out


__all__ = ["ACTIVATIONS", "MAX_ROWS", "fused_linear", "linear", "linear_supported", "prefers_own_kernel"]
