"""What routing and the routed feed-forward refuse, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mini_inference_engine_b200 import _lib, build
from mini_inference_engine_b200.engine.kernels.experts import expert_mlp, route_experts


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def test_refusals_of_the_operators():
    with pytest.raises(ValueError, match="CUDA logits"):
        route_experts(torch.zeros(2, 8), 2)
    x, ids, weights = torch.zeros(2, 16).bfloat16(), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    gate_up, down, status = torch.zeros(4, 16, 16).bfloat16(), torch.zeros(4, 16, 8).bfloat16(), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        expert_mlp(x, ids, weights, gate_up, down, status=status)
    with pytest.raises(ValueError, match="unknown activation"):
        expert_mlp(x, ids, weights, gate_up, down, activation="swish", status=status)
    with pytest.raises(ValueError, match="takes x"):
        expert_mlp(x, ids, weights, gate_up[0], down, status=status)
    long = torch.zeros(1, 1).bfloat16().expand(1 << 31, 1)
    with pytest.raises(ValueError, match="sizes up to"):
        route_experts(long, 1)
    with pytest.raises(ValueError, match="sizes up to"):
        route_experts(torch.zeros(2, 8), (1 << 32) + 1)
    with pytest.raises(ValueError, match="sizes up to"):
        expert_mlp(long, ids, weights, gate_up, down, status=status)
    with pytest.raises(ValueError, match="must be bf16"):
        expert_mlp(x.float(), ids, weights, gate_up, down, status=status)


def route(lib, ld=16, dtype=2, scores=0, tokens=0, experts=16, top_k=2, groups=1, top_groups=1, group_best=1, logits=4096):
    p = ctypes.c_void_p(4096)
    return lib.mie_route_experts(ctypes.c_void_p(logits), ld, dtype, None, scores, tokens, experts, top_k, groups,
                                 top_groups, group_best, 1, 1.0, p, p, None)


def test_refusals_of_routing(lib):
    assert route(lib) == 0 and route(lib, groups=4, top_groups=2, group_best=2, top_k=8) == 0
    for wrong in ({"logits": 0}, {"ld": 15}, {"dtype": 3}, {"scores": 2}, {"tokens": -1}, {"experts": 0},
                  {"experts": 1025, "ld": 1025}, {"top_k": 0}, {"top_k": 17}, {"top_k": 33, "experts": 64, "ld": 64},
                  {"groups": 3}, {"groups": 0}, {"groups": 4, "top_groups": 5}, {"groups": 4, "top_groups": 0},
                  {"groups": 4, "top_groups": 1, "top_k": 5}, {"groups": 64, "experts": 64, "ld": 64},
                  {"group_best": 3}, {"groups": 16, "top_groups": 4, "group_best": 2}):
        assert route(lib, **wrong) == -1, wrong


def experts_call(lib, **changes):
    given = {"x": 4096, "ldx": 16, "ids": 4096, "weights": 4096, "gate_up": 4096, "gate_up_row": 16, "down": 4096,
             "down_row": 8, "residual": None, "ldr": 16, "y": 4096, "ldy": 16, "tokens": 0, "top_k": 2, "experts": 4,
             "width": 16, "ff": 8, "activation": 1, "scratch": 4096, "scratch_bytes": 1 << 20, **changes}
    p = lambda name: ctypes.c_void_p(given[name])  # noqa: E731
    return lib.mie_expert_mlp(
        p("x"), given["ldx"], _lib.IndexT(given["ids"], 0, 2, 1), p("weights"), p("gate_up"), given["gate_up_row"], 256,
        p("down"), given["down_row"], 128, p("residual"), given["ldr"], p("y"), given["ldy"], given["tokens"],
        given["top_k"], given["experts"], given["width"], given["ff"], given["activation"], p("scratch"),
        given["scratch_bytes"], None, None)


def test_refusals_of_the_feed_forward(lib):
    assert experts_call(lib) == 0  # no tokens
    for wrong in ({"x": None}, {"ids": None}, {"weights": None}, {"gate_up": None}, {"down": None}, {"y": None},
                  {"scratch": None}, {"ldx": 15}, {"gate_up_row": 15}, {"down_row": 7}, {"ldy": 15},
                  {"residual": 4096, "ldr": 15}, {"tokens": -1}, {"top_k": 0}, {"top_k": 33}, {"experts": 0},
                  {"experts": 1025}, {"width": 0}, {"ff": 0}, {"activation": 4}, {"tokens": 100, "scratch_bytes": 64},
                  {"tokens": 1 << 29}):
        assert experts_call(lib, **wrong) == -1, wrong
    assert lib.mie_expert_scratch_bytes(8, 2, 4, 16, 8) > 0
    assert lib.mie_expert_scratch_bytes(-1, 2, 4, 16, 8) == 0


def test_refusals_of_choices():
    """Before anything is allocated, and without tokens as well."""

    far = 1 << 32
    for tokens in (0, 2):
        logits = torch.zeros(tokens, 16)
        for options in ({"groups": far + 1}, {"top_groups": far + 1}, {"group_best": far + 1}, {"groups": 1 - far},
                        {"groups": 4, "top_groups": 2 - far}):
            with pytest.raises(ValueError, match="sizes"):
                route_experts(logits, 2, **options)
        for top_k, options in ((0, {}), (-1, {}), (17, {}), (5, {"groups": 4}), (1 << 30, {}), (33, {"logits": 64})):
            z = torch.zeros(tokens, options.pop("logits", 16))
            with pytest.raises(ValueError, match="cannot choose"):
                route_experts(z, top_k, **options)
        for options in ({"groups": 0}, {"groups": 3}, {"groups": 4, "top_groups": 5}, {"groups": 4, "top_groups": 0}):
            with pytest.raises(ValueError, match="groups"):
                route_experts(logits, 2, **options)
        for options in ({"group_best": 0}, {"group_best": 3}, {"groups": 16, "top_groups": 4, "group_best": 2}):
            with pytest.raises(ValueError, match="best"):
                route_experts(logits, 2, **options)
        with pytest.raises(ValueError, match="up to 1024 experts"):
            route_experts(torch.zeros(tokens, 1025), 2)
    with pytest.raises(ValueError, match="experts"):
        route_experts(torch.zeros(2, 0), 1)


def test_refusals_of_pools():
    """Pools and choices that no call takes, with and without tokens, before scratch is asked for."""

    status = torch.zeros(1, dtype=torch.int32)
    for tokens in (0, 2):
        for top_k, experts, width, ff in ((0, 4, 16, 8), (33, 64, 16, 8), (2, 0, 16, 8), (2, 1025, 16, 8), (2, 4, 0, 8),
                                          (2, 4, 16, 0)):
            given = (torch.zeros(tokens, width).bfloat16(), torch.zeros(tokens, top_k, dtype=torch.int32),
                     torch.zeros(tokens, top_k), torch.zeros(experts, 2 * ff, width).bfloat16(),
                     torch.zeros(experts, width, ff).bfloat16())
            with pytest.raises(ValueError, match="expert_mlp takes"):
                expert_mlp(*given, status=status)
    ids, weights = torch.zeros(1, 1, dtype=torch.int32).expand(1 << 26, 16), torch.zeros(1, 1).expand(1 << 26, 16)
    with pytest.raises(ValueError, match="pairs"):
        expert_mlp(torch.zeros(1, 16).bfloat16().expand(1 << 26, 16), ids, weights, torch.zeros(4, 16, 16).bfloat16(),
                   torch.zeros(4, 16, 8).bfloat16(), status=status)


def test_sizes_whose_tiles_pass_32_bits_are_refused(lib):
    """Tiles are counted in 32 bits, past the last row, column and block of k."""

    most = (1 << 31) - 4096
    for wrong in ({"width": most + 1, "ldx": 1 << 31, "gate_up_row": 1 << 31, "ldy": 1 << 31},
                  {"ff": (1 << 30) + 1, "down_row": 1 << 31}):
        assert experts_call(lib, tokens=1, scratch_bytes=1 << 60, **wrong) == -1, wrong
        assert lib.mie_expert_scratch_bytes(1, 2, 4, wrong.get("width", 16), wrong.get("ff", 8)) == 0
    assert experts_call(lib, width=most, ldx=most, gate_up_row=most, ldy=most) == 0


def test_tangents_are_refused():
    """Forward-mode derivatives would be lost."""

    from torch.autograd import forward_ad

    x, ids, weights = torch.zeros(2, 16).bfloat16(), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    gate_up, down, status = torch.zeros(4, 16, 16).bfloat16(), torch.zeros(4, 16, 8).bfloat16(), torch.zeros(1, dtype=torch.int32)
    given = {"x": x, "weights": weights, "gate_up": gate_up, "down": down, "residual": x.clone()}
    logits, bias = torch.zeros(2, 8), torch.zeros(8)
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            for name, value in given.items():
                dual = forward_ad.make_dual(value, torch.ones_like(value))
                with pytest.raises(ValueError, match="derivative"):
                    expert_mlp(ids=ids, status=status, **{**given, name: dual})
            with pytest.raises(ValueError, match="derivative"):
                route_experts(forward_ad.make_dual(logits, torch.ones_like(logits)), 2)
            with pytest.raises(ValueError, match="derivative"):
                route_experts(logits, 2, bias=forward_ad.make_dual(bias, torch.ones_like(bias)))
            with pytest.raises(ValueError, match="CUDA"):  # without a tangent nothing is in the way
                route_experts(logits, 2, bias=bias)
    with pytest.raises(ValueError, match="derivative"):
        torch.func.jvp(lambda z: route_experts(z, 2)[1], (logits,), (logits,))
