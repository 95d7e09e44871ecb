"""What the fused projection refuses, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mini_inference_engine_b200 import _lib, build
from mini_inference_engine_b200.engine.kernels.linear import fused_linear


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def rows(r, c, dtype=torch.bfloat16):
    return torch.zeros(r, c, dtype=dtype)


@pytest.mark.parametrize("x,w,options,message", [
    (rows(2, 8), rows(4, 8), {}, "CUDA device"),
    (rows(2, 8), rows(4, 8), {"activation": "swish"}, "unknown activation"),
    (rows(2, 8, torch.float32), rows(4, 8), {}, "must be bf16"),
    (rows(2, 8).view(1, 2, 8), rows(4, 8), {}, "takes rows"),
    (rows(1, 1).expand(1 << 32, 1), rows(4, 1), {}, "sizes up to"),
])
def test_refusals_of_the_operator(x, w, options, message):
    with pytest.raises(ValueError, match=message):
        fused_linear(x, w, status=torch.zeros(1, dtype=torch.int32), **options)


def call(lib, m=4, n=8, k=8, ldx=8, ldw=8, ldr=8, ldy=8, activation=0, gated=0, x=4096, residual=None):
    p = ctypes.c_void_p(4096)
    return lib.mie_fused_linear(ctypes.c_void_p(x), ldx, p, ldw, None, residual, ldr, p, ldy, m, n, k, activation, gated,
                                None, None)


def test_refusals_of_the_c_entry(lib):
    assert call(lib, m=0) == 0  # nothing to do
    residual = ctypes.c_void_p(4096)
    for wrong in ({"x": 0}, {"m": -1}, {"n": 0}, {"k": 0}, {"ldx": 7}, {"ldw": 7}, {"ldy": 7}, {"activation": 4},
                  {"activation": -1}, {"residual": residual, "ldr": 7}):
        assert call(lib, **{"m": 0, **wrong}) == -1, wrong


def test_sizes_whose_tiles_pass_32_bits_are_refused(lib):
    """Tiles are counted in 32 bits, past the last row, column and block of k."""

    most = (1 << 31) - 4096
    for wrong in ({"m": most + 1}, {"m": (1 << 31) - 1}, {"k": most + 1, "ldx": most + 1, "ldw": most + 1},
                  {"k": (1 << 31) - 1, "ldx": 1 << 31, "ldw": 1 << 31}, {"n": (1 << 30) + 1, "ldy": 1 << 31}):
        assert call(lib, **wrong) == -1, wrong
    assert call(lib, m=0, k=most, ldx=most, ldw=most) == 0


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_tangents_are_refused(which):
    """Forward-mode derivatives would be lost."""

    from torch.autograd import forward_ad

    given = {"x": rows(2, 8), "weight": rows(4, 8), "bias": rows(1, 4)[0], "residual": rows(2, 4)}
    with forward_ad.dual_level():
        given[which] = forward_ad.make_dual(given[which], torch.ones_like(given[which]))
        with pytest.raises(ValueError, match="derivative"):
            fused_linear(**given, status=torch.zeros(1, dtype=torch.int32))
