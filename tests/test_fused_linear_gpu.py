"""Fused projections against the product in 64 bits."""

from __future__ import annotations

import pytest
import torch

from mini_inference_engine_b200.engine.kernels.linear import fused_linear
from product_bounds import assert_within
from product_bounds import fused_linear as exact_fused_linear

pytestmark = pytest.mark.gpu


def operands(m, n, k, gated, bias, residual, device, pad=8):
    """Rows of wider buffers with nonsense behind them: the kernels must honour the strides."""

    def rows(r, c, scale=1.0):
        out = torch.full((r, c + pad), float("nan"), dtype=torch.bfloat16, device=device)[:, :c]
        return out.copy_(torch.randn(r, c, device=device) * scale)

    weight_rows = 2 * n if gated else n
    return (rows(m, k), rows(weight_rows, k, 2.0 * k ** -0.5),
            torch.randn(weight_rows, device=device).to(torch.bfloat16) if bias else None,
            rows(m, n) if residual else None)


def check(m, n, k, activation, gated, bias, residual, device, pad=8):
    torch.manual_seed(m * 131 + n * 17 + k)
    x, w, b, r = operands(m, n, k, gated, bias, residual, device, pad)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = fused_linear(x, w, b, activation=activation, gated=gated, residual=r, status=status)
    assert out.shape == (m, n) and out.dtype == torch.bfloat16
    assert_within(out, *exact_fused_linear(x, w, b, activation or "none", gated, r))
    assert int(status.item()) == 0


# Rows around every tile border of the kernels, columns and lengths around theirs.
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 256, 257, 385, 700])
@pytest.mark.parametrize("n,k", [(1, 8), (17, 72), (128, 64), (130, 520), (256, 1024), (1000, 256), (2112, 1096)])
@pytest.mark.parametrize("gated", [False, True])
def test_sizes(m, n, k, gated, device):
    check(m, n, k, "silu", gated, m % 2 == 0, m % 3 == 0, device)


@pytest.mark.parametrize("activation", [None, "none", "silu", "gelu", "relu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_epilogues(activation, gated, bias, residual, m, device):
    check(m, 320, 512, activation, gated, bias, residual, device)


@pytest.mark.parametrize("m", [1, 5, 33, 150, 300])
@pytest.mark.parametrize("n,k,pad", [(64, 63, 0), (33, 1, 0), (97, 257, 3), (40, 64, 1), (64, 100, 4), (128, 64, 7)])
@pytest.mark.parametrize("gated", [False, True])
def test_rows_without_alignment(m, n, k, pad, gated, device):
    check(m, n, k, "gelu", gated, True, True, device, pad)


@pytest.mark.parametrize("m,n,k,gated", [(1, 6144, 2048, True), (24, 2560, 9728, False), (3, 256, 12288, False),
                                         (2048, 1536, 2560, True), (1021, 5003, 2056, False), (128, 12288, 512, True),
                                         (256, 2560, 9728, False), (130, 1000, 4096, False), (400, 4096, 4096, False),
                                         (161, 2052, 2104, False), (300, 768, 3000, False), (512, 520, 8192, False)])
def test_long_and_wide(m, n, k, gated, device):
    check(m, n, k, "gelu", gated, True, True, device)


@pytest.mark.parametrize("m,n,k", [(8_500_000, 8, 8), (70_000, 520, 64), (3, 300_000, 64)])
def test_more_tiles_than_a_grid_has(m, n, k, device):
    torch.manual_seed(m)
    x, w, b, _ = operands(m, n, k, False, True, False, device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = fused_linear(x, w, b, activation="relu", status=status)
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300 if m > 300 else 0, m)):
        assert_within(out[rows], *exact_fused_linear(x[rows], w, b, "relu", False, None))
    assert int(status.item()) == 0


def test_operands_that_start_anywhere(device):
    """Views whose first entry is off a 16-byte border."""

    torch.manual_seed(0)
    for shift in (1, 2, 4):
        for m in (3, 200):
            x = torch.randn(m * 64 + shift, device=device).bfloat16()[shift:].view(m, 64)
            w = torch.randn(48 * 64 + shift, device=device).bfloat16()[shift:].view(48, 64)
            r = torch.randn(m * 48 + shift, device=device).bfloat16()[shift:].view(m, 48)
            status = torch.zeros(1, dtype=torch.int32, device=device)
            out = fused_linear(x, w, activation="relu", residual=r, status=status)
            assert_within(out, *exact_fused_linear(x, w, None, "relu", False, r))


@pytest.mark.parametrize("m", [2, 20, 300])
def test_infinities_and_nans_stay_where_they_belong(m, device):
    x = torch.ones(m, 128, dtype=torch.bfloat16, device=device)
    w = torch.ones(2 * 72, 128, dtype=torch.bfloat16, device=device)
    x[1, 3], w[7, 70] = float("inf"), float("nan")
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = fused_linear(x, w, activation="silu", gated=True, status=status).float()
    assert bool(out[:, 7].isnan().all())
    rest = torch.cat([out[:, :7], out[:, 8:]], dim=1)
    assert bool((rest[1] == float("inf")).all()) and bool((rest[0] == 128 * 128).all())


@pytest.mark.parametrize("activation", ["silu", "gelu", "relu"])
def test_activations_far_out(activation, device):
    """Every bf16 value through the activation by a product with one."""

    z = torch.arange(65536, device=device).to(torch.int32).to(torch.int16).view(torch.bfloat16)
    z = z[torch.isfinite(z)]
    x = torch.zeros(z.numel(), 8, dtype=torch.bfloat16, device=device)
    x[:, 0] = z
    w = torch.zeros(8, 8, dtype=torch.bfloat16, device=device)
    w[:, 0] = 1
    status = torch.zeros(1, dtype=torch.int32, device=device)
    for rows in (x, x[-40:], x[1000:1001]):
        out = fused_linear(rows, w, activation=activation, status=status)
        exact, bound = exact_fused_linear(rows, w, None, activation, False, None)
        assert bool(torch.isfinite(out).all())
        # Results that no normal fp32 number holds may be flushed to zero.
        assert_within(out, exact, torch.maximum(bound, torch.full_like(bound, 2.0 ** -126)))


def test_result_over_the_residual(device):
    """``y`` of the C entry may be the residual itself."""

    from mini_inference_engine_b200 import _lib

    for m in (2, 50, 400):
        torch.manual_seed(m)
        x, w, b, r = operands(m, 136, 128, False, True, True, device)
        exact, bound = exact_fused_linear(x, w, b, "none", False, r)
        status = torch.zeros(1, dtype=torch.int32, device=device)
        _lib.check(_lib.load().mie_fused_linear(
            _lib.ptr(x), x.stride(0), _lib.ptr(w), w.stride(0), _lib.ptr(b), _lib.ptr(r), r.stride(0), _lib.ptr(r),
            r.stride(0), m, 136, 128, 0, 0, _lib.ptr(status), _lib.stream_arg(device)))
        assert_within(r, exact, bound)


def test_other_stream_and_graph(device):
    """On a side stream, and captured and replayed over new inputs."""

    torch.manual_seed(3)
    for m in (1, 48, 260):
        x, w, b, r = operands(m, 264, 256, True, True, True, device)
        status = torch.zeros(1, dtype=torch.int32, device=device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = fused_linear(x, w, b, activation="silu", gated=True, residual=r, status=status)
        torch.cuda.current_stream().wait_stream(side)
        assert_within(first, *exact_fused_linear(x, w, b, "silu", True, r))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fused_linear(x, w, b, activation="silu", gated=True, residual=r, status=status)
        for _ in range(2):
            x.copy_(torch.randn(m, 256, device=device))
            graph.replay()
            assert_within(out, *exact_fused_linear(x, w, b, "silu", True, r))
        assert int(status.item()) == 0


def test_weights_written_by_a_queued_call(device):
    """The weight of a call is the result of the call before it."""

    torch.manual_seed(4)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    for m in (3, 40, 300):
        a = torch.randn(512, 256, device=device).bfloat16()
        eye = torch.eye(256, dtype=torch.bfloat16, device=device)
        x = torch.randn(m, 256, device=device).bfloat16()
        for _ in range(20):
            w = fused_linear(a, eye, status=status)
            out = fused_linear(x, w, status=status)
        assert_within(out, *exact_fused_linear(x, a, None, "none", False, None))


def whole_numbers(r, c, most, device):
    return torch.randint(-most, most + 1, (r, c), device=device).to(torch.bfloat16)


@pytest.mark.parametrize("m", [1, 16, 24, 64, 100, 256, 1021])
@pytest.mark.parametrize("n,k", [(256, 12288), (1000, 9728), (520, 4104), (96, 2055)])
@pytest.mark.parametrize("gated", [False, True])
def test_sums_of_whole_numbers_are_exact(m, n, k, gated, device):
    """No sum, in parts or whole, is held in less than fp32.

    Operands are whole numbers up to 16, so that every partial sum, whatever the order, is one below k 16^2 + 2 16 < 2^24 and
    exact in fp32; parts of it pass 2^11, where fp16 and bf16 would lose their last bits.  The residual takes the sum rounded
    to bf16 away: what is left, at most half a step of the sum (2^-9 of 2^22), is a multiple of a power of two with at most 14
    bits and is rounded once."""

    torch.manual_seed(m + n + k)
    x, w = whole_numbers(m, k, 16, device), whole_numbers(n, k, 16, device)
    bias = whole_numbers(1, n, 16, device)[0]
    exact = x.double() @ w.double().t() + bias.double()
    rounded = exact.to(torch.bfloat16)
    weight, b = w, bias
    if gated:  # ups of one: the bias alone
        weight, b = torch.cat([w, torch.zeros_like(w)]), torch.cat([bias, torch.ones_like(bias)])
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = fused_linear(x, weight, b, activation="none", gated=gated, residual=-rounded, status=status)
    assert torch.equal(out, (exact - rounded.double()).to(torch.bfloat16))
    assert int(status.item()) == 0
