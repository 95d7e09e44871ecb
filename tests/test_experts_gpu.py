"""Routing and the routed feed-forward against their definitions in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mini_inference_engine_b200.engine.kernels.experts import expert_mlp, route_experts
from mini_inference_engine_b200.engine.kernels.linear import fused_linear
from product_bounds import assert_within
from product_bounds import expert_mlp as exact_expert_mlp

pytestmark = pytest.mark.gpu
NEVER = float("-inf")


# -- routing ------------------------------------------------------------------------------------------------

def plain_route(logits, top_k, *, scores="softmax", bias=None, groups=1, top_groups=1, group_best=1, renormalize=True,
                scale=1.0):
    """The definition, row by row, in 64 bits (no NaN)."""

    z = logits.double().cpu().numpy()
    tokens, experts = z.shape
    if scores == "softmax":
        top = z.max(axis=1, keepdims=True)
        e = np.exp(z - np.where(np.isfinite(top), top, 0.0))
        total = e.sum(axis=1, keepdims=True)
        s = np.where(total > 0, e / np.where(total > 0, total, 1.0), 0.0)
    else:
        s = np.where(z >= 0, 1.0, np.exp(np.minimum(z, 0.0))) / (1.0 + np.exp(-np.abs(z)))
    # Without a bias the scores' order is the logits'; 64 bits do not tell large ones apart.
    by_logit = bias is None and (groups == 1 or group_best == 1)
    c = z.copy() if by_logit else s + (0.0 if bias is None else bias.double().cpu().numpy())
    c[z == -np.inf] = -np.inf
    size = experts // groups
    ids = np.zeros((tokens, top_k), dtype=np.int64)
    for t in range(tokens):
        allowed = list(range(experts))
        if groups > 1:
            sums = [sum(sorted(c[t, g * size:(g + 1) * size])[-group_best:]) for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-sums[g], g))[:top_groups]
            allowed = [e for e in range(experts) if e // size in kept]
        ids[t] = sorted(allowed, key=lambda e: (-c[t, e], e))[:top_k]
    w = np.take_along_axis(np.where(z == -np.inf, 0.0, s), ids, axis=1)
    if renormalize:
        # By logarithms (log sigmoid(z) = min(z, 0) - log(1 + exp(-|z|))): 64 bits, too, underflow at the lowest fp32 logit.
        log = np.take_along_axis(z if scores == "softmax" else np.minimum(z, 0.0) - np.log1p(np.exp(-np.abs(z))), ids, axis=1)
        most = log.max(axis=1, keepdims=True)
        w = np.exp(log - np.where(np.isfinite(most), most, 0.0))
        total = w.sum(axis=1, keepdims=True)
        w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
    return ids, w * scale


def check_route(logits, top_k, **options):
    ids, weights = route_experts(logits, top_k, **options)
    assert ids.dtype == torch.int32 and weights.dtype == torch.float32
    assert ids.shape == weights.shape == (logits.shape[0], top_k)
    exact_ids, exact_weights = plain_route(logits, top_k, **options)
    assert np.array_equal(ids.cpu().numpy(), exact_ids)
    # Exponentials within 2 ulp of arguments that are rounded once (up to 2^-24 |z - max| each), sums of up to 1024
    # terms in a tree of at most 37 roundings, two divisions and a product: below 2^-17 for |z| < 64.
    off = np.abs(weights.double().cpu().numpy() - exact_weights)
    assert (off <= 2.0 ** -17 * np.abs(exact_weights) + 1e-37).all(), off.max()


@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (8, 2), (31, 5), (32, 8), (33, 32), (60, 4), (64, 6), (100, 10),
                                           (128, 8), (160, 6), (256, 8), (300, 7), (512, 10), (513, 3), (1000, 32), (1024, 9)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_routing_sizes(experts, top_k, scores, with_bias, device):
    torch.manual_seed(experts * 7 + top_k)
    for tokens in (1, 7, 200):
        logits = 2.0 * torch.randn(tokens, experts + 3, device=device)[:, :experts]
        bias = 0.1 * torch.randn(experts, device=device) if with_bias else None
        check_route(logits, top_k, scores=scores, bias=bias, renormalize=tokens != 7, scale=2.5 if tokens == 200 else 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,groups,top_groups,group_best,top_k", [
    (64, 8, 3, 2, 6), (256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (32, 32, 4, 1, 4), (48, 3, 1, 2, 16), (96, 2, 2, 2, 8),
    (1024, 16, 2, 2, 32), (30, 5, 5, 2, 30)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_routing_by_groups(experts, groups, top_groups, group_best, top_k, scores, dtype, device):
    torch.manual_seed(experts + groups)
    logits = torch.randn(150, experts, device=device).to(dtype)
    bias = 0.05 * torch.randn(experts, device=device)
    for b in (None, bias):
        check_route(logits, top_k, scores=scores, bias=b, groups=groups, top_groups=top_groups, group_best=group_best)


def test_equal_choices_go_to_the_lowest_index(device):
    torch.manual_seed(1)
    logits = torch.randint(-2, 3, (300, 96), device=device).float()
    zero, shared = torch.zeros(96, device=device), torch.full((96,), 0.3, device=device)
    for scores in ("softmax", "sigmoid"):
        for bias in (None, zero, shared):
            check_route(logits, 12, scores=scores, bias=bias)
            check_route(logits, 12, scores=scores, bias=bias, groups=4, top_groups=2, group_best=1)
            check_route(logits, 12, scores=scores, bias=bias, groups=4, top_groups=2, group_best=2)
            check_route(logits.bfloat16(), 12, scores=scores, bias=bias)
    check_route(torch.zeros(5, 40, device=device), 32)  # as many as a token may choose
    check_route(torch.tensor([[0.0, -0.0, 0.0, -0.0]], device=device), 4)


def test_choices_that_32_bits_cannot_tell_apart(device):
    """Scores that differ by less than fp32 resolves are chosen as in 64 bits."""

    torch.manual_seed(2)
    base = torch.randn(400, 1, device=device).expand(400, 64)
    step = torch.randint(-3, 4, (400, 64), device=device).float()
    logits = (base * (1.0 + step * 2.0 ** -23)).contiguous()
    bias = torch.randint(-2, 3, (64,), device=device).float() * 2.0 ** -24
    for scores in ("softmax", "sigmoid"):
        check_route(logits, 9, scores=scores)
        check_route(logits, 9, scores=scores, bias=bias)
        check_route(logits, 9, scores=scores, bias=100.0 + bias * 2.0 ** 12)
        # Sums of two: those with steps 3 + 1 and 2 + 2 differ only in second order, by (2^-23 z)^2 |s''| < 2^-49 z^2, where
        # 64 bits have an error of three roundings of a score, 3 * 2^-53 each.  Rows in which the last group taken and the
        # first one left out are nearer than 2^-50 are not decided by the definition in 64 bits.
        options = {"scores": scores, "bias": bias, "groups": 8, "top_groups": 3, "group_best": 2}
        z = logits.double()
        c = (torch.softmax(z, dim=1) if scores == "softmax" else torch.sigmoid(z)) + bias.double()
        sums = c.view(400, 8, 8).topk(2, dim=2).values.sum(dim=2).sort(dim=1, descending=True).values
        decided = sums[:, 2] - sums[:, 3] >= 2.0 ** -50
        assert int(decided.sum()) > 0
        check_route(logits[decided], 9, **options)
    # Saturated sigmoids: without a bias the order is that of the logits.
    far = (40.0 + torch.rand(50, 64, device=device))
    check_route(far, 8, scores="sigmoid", renormalize=False)


def test_masked_experts(device):
    torch.manual_seed(3)
    logits = torch.randn(64, 48, device=device)
    logits[torch.rand(64, 48, device=device) < 0.8] = NEVER
    logits[:4] = NEVER          # nothing to choose from
    logits[4:8] = NEVER
    logits[4:8, 30] = 1.0       # one expert left
    logits[8, :] = torch.finfo(torch.float32).min
    bias = 0.5 * torch.randn(48, device=device)
    for scores in ("softmax", "sigmoid"):
        for b in (None, bias):
            for groups, top_groups, best in ((1, 1, 1), (4, 2, 1), (4, 2, 2)):
                check_route(logits, 10, scores=scores, bias=b, groups=groups, top_groups=top_groups, group_best=best)
                check_route(logits, 10, scores=scores, bias=b, groups=groups, top_groups=top_groups, group_best=best,
                            renormalize=False)


def test_scores_far_below_one(device):
    """Weights over the sum of the chosen depend on their ratios, however small the scores are."""

    torch.manual_seed(9)
    logits = torch.randn(40, 48, device=device)
    bias = torch.zeros(48, device=device)
    bias[:16] = 2.0                        # chosen for their bias
    for shift in (50.0, 70.0, 100.0, 300.0):
        low = logits.clone()
        low[:, :16] -= shift               # far below the row's maximum
        check_route(low, 6, scores="softmax", bias=bias)
        check_route(low, 6, scores="sigmoid", bias=bias)
        check_route(logits - shift, 6, scores="sigmoid")
        check_route(logits - shift, 6, scores="softmax")
        check_route(low, 6, scores="softmax", bias=bias, renormalize=False)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [3, 30, 64, 100, 256, 400, 1000])
def test_equals_at_the_border_of_the_choice(experts, scores, device):
    """The last expert taken and the first one left out have equal logits and biases, and a third one, behind them in 32 bits or
    by its index, is better in 64."""

    torch.manual_seed(experts)
    near = max(3, experts // 2)
    for top_k in sorted({1, 2, min(8, near - 1), min(32, near - 1)}):
        for base in (-3.0, 0.7, 2.0):
            # Logits of two values that are a rounding or two apart, at random places, with the others clearly below.
            step = (torch.rand(60, experts, device=device) < 0.1).float()
            logits = base * (1.0 + step * 2.0 ** -22)
            low = torch.argsort(torch.rand(60, experts, device=device), dim=1)[:, near:]
            logits.scatter_(1, low, base - 4.0)
            bias = torch.randint(0, 2, (experts,), device=device).float() * 2.0 ** -20
            for b in (torch.zeros(experts, device=device), torch.full((experts,), 0.3, device=device), bias):
                check_route(logits.contiguous(), top_k, scores=scores, bias=b)
                # (Mixed biases give groups whose sums are equal but for the roundings of 64 bits.)
                if experts % 4 == 0 and b is not bias:
                    check_route(logits.contiguous(), min(top_k, experts // 2), scores=scores, bias=b, groups=4, top_groups=2,
                                group_best=2)


def test_equal_saturated_scores_at_the_border(device):
    """Sigmoids that are all one in 32 bits and not in 64."""

    for experts in (3, 70, 300):
        zero = torch.zeros(experts, device=device)
        logits = torch.full((3, experts), 18.0, device=device)
        logits[0, -1] = 20.0
        logits[1, experts // 2] = 19.0
        logits[1, -1] = 19.5
        for top_k in (1, 2, min(32, experts - 1)):
            check_route(logits, top_k, scores="sigmoid", bias=zero)
            check_route(logits.bfloat16(), top_k, scores="sigmoid", bias=zero + 0.5)


def test_sigmoid_weights_of_any_ratio(device):
    """Weights over the chosen's sum whose sigmoids lie far apart, the smaller ones below what 32 bits hold.

    Arguments of the exponentials are differences up to 128, rounded once (2^-18); exponentials, sums and divisions add less
    than 2^-20: below 2^-17."""

    torch.manual_seed(20)
    for largest in (-59.9, -59.0, -40.0, -25.0, -10.0, 3.0):
        logits = largest - 80.0 * torch.rand(50, 24, device=device)
        logits[:, 5] = largest
        for top_k in (2, 10, 24):
            check_route(logits, top_k, scores="sigmoid")
            check_route(logits, top_k, scores="sigmoid", bias=0.1 * torch.randn(24, device=device))


def test_logits_that_are_no_numbers(device):
    torch.manual_seed(4)
    logits = torch.randn(6, 40, device=device)
    logits[1, 5] = float("nan")
    logits[2, :] = float("nan")
    logits[3, 7] = float("inf")
    bias = torch.randn(40, device=device)
    for scores in ("softmax", "sigmoid"):
        for b in (None, bias):
            ids, weights = route_experts(logits, 4, scores=scores, bias=b)
            assert bool(weights[1].isnan().all()) and bool(weights[2].isnan().all())
            assert bool(((ids >= 0) & (ids < 40)).all())
            assert all(len(set(row)) == 4 for row in ids.tolist())
            clean = torch.tensor([0, 4, 5], device=device)
            alone = route_experts(logits[clean].contiguous(), 4, scores=scores, bias=b)
            assert torch.equal(ids[clean], alone[0]) and torch.equal(weights[clean], alone[1])
    ids, weights = route_experts(logits, 4, scores="sigmoid")
    assert int(ids[3, 0]) == 7 and bool(torch.isfinite(weights[3]).all())


def test_routing_refuses(device):
    logits = torch.zeros(3, 16, device=device)
    with pytest.raises(ValueError, match="cannot choose"):
        route_experts(logits, 17)
    with pytest.raises(ValueError, match="groups"):
        route_experts(logits, 2, groups=3)
    with pytest.raises(ValueError, match="unknown scores"):
        route_experts(logits, 2, scores="max")
    with pytest.raises(ValueError, match="bias"):
        route_experts(logits, 2, bias=torch.zeros(15, device=device))
    with pytest.raises(ValueError, match="dense rows"):
        route_experts(torch.zeros(16, 3, device=device).t(), 2)
    with pytest.raises(ValueError, match="no gradient"):
        route_experts(logits.clone().requires_grad_(), 2)
    ids, weights = route_experts(logits[:0], 2)
    assert ids.shape == weights.shape == (0, 2)


# -- feed-forward ---------------------------------------------------------------------------------------------

def pool(experts, width, ff, device, pad=0):
    def stack(rows, cols):
        out = torch.full((experts, rows, cols + pad), float("nan"), dtype=torch.bfloat16, device=device)[:, :, :cols]
        return out.copy_(torch.randn(experts, rows, cols, device=device) * cols ** -0.5)

    return stack(2 * ff, width), stack(width, ff)


def check_experts(tokens, width, ff, experts, top_k, device, *, ids=None, activation="silu", residual=True, pad=0):
    torch.manual_seed(tokens * 31 + width + ff + experts)
    gate_up, down = pool(experts, width, ff, device, pad)
    x = torch.full((tokens, width + pad), float("nan"), dtype=torch.bfloat16, device=device)[:, :width]
    x.copy_(torch.randn(tokens, width, device=device))
    if ids is None:
        ids = torch.argsort(torch.randn(tokens, experts, device=device), dim=1)[:, :top_k].to(torch.int32)
    weights = torch.randn(tokens, top_k, device=device)
    r = torch.randn(tokens, width, device=device).bfloat16() if residual else None
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = expert_mlp(x, ids, weights, gate_up, down, activation=activation, residual=r, status=status)
    assert_within(out, *exact_expert_mlp(x, ids, weights, gate_up, down, activation, r))
    return int(status.item())


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16, 17, 40, 64, 100, 129, 300, 700])
@pytest.mark.parametrize("experts,top_k,width,ff", [(1, 1, 64, 64), (4, 2, 128, 72), (8, 8, 136, 264), (16, 3, 512, 128),
                                                    (128, 8, 256, 96), (60, 4, 1000, 40)])
def test_feed_forward_sizes(tokens, experts, top_k, width, ff, device):
    assert check_experts(tokens, width, ff, experts, top_k, device, residual=tokens % 2 == 0) == 0


@pytest.mark.parametrize("activation", ["none", "silu", "gelu", "relu"])
@pytest.mark.parametrize("tokens", [1, 30, 500])
def test_feed_forward_activations(activation, tokens, device):
    assert check_experts(tokens, 256, 128, 8, 2, device, activation=activation) == 0


@pytest.mark.parametrize("width,ff,pad", [(63, 33, 0), (64, 20, 0), (72, 48, 8), (128, 64, 3), (1, 1, 0)])
@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_feed_forward_without_alignment(width, ff, pad, tokens, device):
    assert check_experts(tokens, width, ff, 5, 2, device, pad=pad) == 0


@pytest.mark.parametrize("tokens", [1, 9, 33, 260, 900])
def test_every_token_to_one_expert(tokens, device):
    ids = torch.full((tokens, 1), 3, dtype=torch.int64, device=device)
    assert check_experts(tokens, 256, 136, 6, 1, device, ids=ids) == 0


@pytest.mark.parametrize("tokens", [1, 4, 40, 400])
def test_the_same_expert_twice(tokens, device):
    torch.manual_seed(tokens)
    ids = torch.randint(0, 3, (tokens, 6), device=device, dtype=torch.int32)
    assert check_experts(tokens, 192, 64, 3, 6, device, ids=ids) == 0


@pytest.mark.parametrize("tokens", [1, 6, 50, 300])
def test_no_expert_and_bad_experts(tokens, device):
    torch.manual_seed(tokens)
    ids = torch.randint(-1, 8, (tokens, 4), device=device, dtype=torch.int32)
    ids[0] = -1
    assert check_experts(tokens, 128, 64, 8, 4, device, ids=ids) == 0
    assert check_experts(tokens, 128, 64, 8, 4, device, ids=torch.full_like(ids, -1)) == 0
    ids[-1, 2] = 8
    assert check_experts(tokens, 128, 64, 8, 4, device, ids=ids) == 1024
    ids[-1, 2] = -7
    assert check_experts(tokens, 128, 64, 8, 4, device, ids=ids, residual=False) == 1024


def test_strided_ids(device):
    torch.manual_seed(5)
    wide = torch.randint(0, 8, (40, 9), device=device)
    assert check_experts(40, 128, 64, 8, 3, device, ids=wide[:, ::3]) == 0
    assert check_experts(40, 128, 64, 8, 3, device, ids=wide[:, :3].t().contiguous().t()) == 0


@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_what_is_no_number_stays_with_its_token(tokens, device):
    torch.manual_seed(6)
    gate_up, down = pool(6, 128, 64, device)
    x = torch.randn(tokens, 128, device=device).bfloat16()
    ids = torch.stack([torch.arange(tokens, device=device) % 3, 3 + torch.arange(tokens, device=device) % 3], dim=1)
    weights = torch.rand(tokens, 2, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    clean = expert_mlp(x, ids, weights, gate_up, down, status=status)
    x[1, 7] = float("nan")
    weights[2, 1] = float("inf")
    out = expert_mlp(x, ids, weights, gate_up, down, status=status)
    others = [t for t in range(tokens) if t not in (1, 2)]
    assert bool(out[1].isnan().all()) and not bool(torch.isfinite(out[2]).any())
    assert torch.equal(out[others], clean[others])


@pytest.mark.parametrize("magnitude", [2.0 ** 40, 2.0 ** -40])
def test_large_and_small_values(magnitude, device):
    """Rows whose sums no fp16 number holds."""

    torch.manual_seed(7)
    for tokens in (2, 30, 200):
        gate_up, down = pool(4, 128, 64, device)
        down = (down.float() * magnitude).bfloat16()
        x = torch.randn(tokens, 128, device=device).bfloat16()
        ids = torch.argsort(torch.rand(tokens, 4, device=device), dim=1)[:, :2]
        weights = torch.rand(tokens, 2, device=device)
        status = torch.zeros(1, dtype=torch.int32, device=device)
        out = expert_mlp(x, ids, weights, gate_up, down, status=status)
        assert_within(out, *exact_expert_mlp(x, ids, weights, gate_up, down, "silu", None))


@pytest.mark.parametrize("tokens", [1, 6, 20, 32, 33, 400])
def test_the_same_call_gives_the_same_bits(tokens, device):
    """Pairs are placed, and parts of sums arrive, in any order; the results do not depend on it."""

    torch.manual_seed(11)
    gate_up, down = pool(40, 512, 256, device)
    x, r = torch.randn(tokens, 512, device=device).bfloat16(), torch.randn(tokens, 512, device=device).bfloat16()
    ids = torch.argsort(torch.rand(tokens, 40, device=device), dim=1)[:, :6].to(torch.int32)
    weights = torch.rand(tokens, 6, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    first = expert_mlp(x, ids, weights, gate_up, down, residual=r, status=status)
    for _ in range(20):
        assert torch.equal(expert_mlp(x, ids, weights, gate_up, down, residual=r, status=status), first)


@pytest.mark.parametrize("tokens", [1, 8, 32, 40, 200])
def test_an_expert_that_is_no_number_stays_with_its_tokens(tokens, device):
    torch.manual_seed(12)
    gate_up, down = pool(12, 256, 128, device)
    x = torch.randn(tokens, 256, device=device).bfloat16()
    ids = torch.argsort(torch.rand(tokens, 12, device=device), dim=1)[:, :3].to(torch.int32)
    ids[0] = torch.tensor([5, 1, 2], device=device)
    weights = torch.rand(tokens, 3, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    clean = expert_mlp(x, ids, weights, gate_up, down, status=status)
    for broken in (float("nan"), float("inf")):
        gate, out = gate_up.clone(), down.clone()
        gate[5, 3, 7] = broken
        out[5, 9, 11] = broken
        touched = (ids == 5).any(dim=1)
        for g, d in ((gate, down), (gate_up, out)):
            got = expert_mlp(x, ids, weights, g, d, status=status)
            assert torch.equal(got[~touched], clean[~touched])
            assert not bool(torch.isfinite(got[0]).all())
        # Of the down weight only its own channel (the others' rows may be rounded by another exponent).
        others = torch.arange(256, device=device) != 9
        exact, bound = exact_expert_mlp(x, ids, weights, gate_up, down, "silu", None)
        assert_within(got[:, others], exact[:, others], bound[:, others])


def test_all_experts_in_use_of_a_large_pool(device):
    """1024 experts, 32 of them a token: the most a token may name."""

    for tokens in (1, 32, 70):
        torch.manual_seed(tokens)
        gate_up, down = pool(1024, 64, 32, device)
        x = torch.randn(tokens, 64, device=device).bfloat16()
        ids = torch.argsort(torch.rand(tokens, 1024, device=device), dim=1)[:, :32].to(torch.int32)
        weights = torch.rand(tokens, 32, device=device)
        status = torch.zeros(1, dtype=torch.int32, device=device)
        out = expert_mlp(x, ids, weights, gate_up, down, status=status)
        assert_within(out, *exact_expert_mlp(x, ids, weights, gate_up, down, "silu", None))
        assert int(status.item()) == 0


def test_weights_routed_by_the_call_before(device):
    """Ids and weights that a queued kernel writes, and a pool that the one before it wrote."""

    torch.manual_seed(13)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    for tokens in (1, 7, 20, 100):
        gate_up, down = pool(16, 256, 128, device)
        x = torch.randn(tokens, 256, device=device).bfloat16()
        router = torch.randn(16, 256, device=device).bfloat16()
        eye = torch.eye(128, dtype=torch.bfloat16, device=device)
        for _ in range(10):
            copy = torch.empty_like(down)
            for e in range(16):
                copy[e] = fused_linear(down[e], eye, status=status)
            ids, weights = route_experts(fused_linear(x, router, status=status), 4, status=status)
            out = expert_mlp(x, ids, weights, gate_up, copy, status=status)
            expected = expert_mlp(x, ids.clone(), weights.clone(), gate_up, down, status=status)
            assert torch.equal(out, expected)


@pytest.mark.parametrize("tokens", [1, 5, 16, 17, 32])
@pytest.mark.parametrize("experts,top_k,width,ff", [(4, 2, 512, 2048), (40, 8, 256, 1024), (8, 2, 4096, 512), (5, 2, 72, 4000)])
def test_few_rows_sums_of_whole_numbers_are_exact(tokens, experts, top_k, width, ff, device):
    """Up to 32 tokens no sum is held in less than fp32, within an expert or over them.

    Rows of x have one entry that is not zero, so that gates and ups are whole numbers up to 8 and hidden values (a rounding to
    bf16 of whole numbers up to 64) are exact; so is every partial sum, at most 2 top_k ff 64 16 <= 2^24.  The
    residual takes the sum rounded to bf16 away, and what is left is rounded once."""

    torch.manual_seed(tokens + width)
    whole = lambda most, *shape: torch.randint(-most, most + 1, shape, device=device).to(torch.bfloat16)  # noqa: E731
    gate_up, down = whole(8, experts, 2 * ff, width), whole(16, experts, width, ff)
    x = torch.zeros(tokens, width, dtype=torch.bfloat16, device=device)
    x[torch.arange(tokens, device=device), torch.randint(0, width, (tokens,), device=device)] = 1.0
    ids = torch.argsort(torch.rand(tokens, experts, device=device), dim=1)[:, :top_k].to(torch.int32)
    weights = torch.randint(1, 3, (tokens, top_k), device=device).float()
    exact = torch.zeros(tokens, width, dtype=torch.float64, device=device)
    for j in range(top_k):
        for t in range(tokens):
            e = int(ids[t, j])
            z = gate_up[e].double() @ x[t].double()
            exact[t] += weights[t, j].double() * (down[e].double() @ (z[:ff] * z[ff:]))
    rounded = exact.to(torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = expert_mlp(x, ids, weights, gate_up, down, activation="none", residual=-rounded, status=status)
    assert torch.equal(out, (exact - rounded.double()).to(torch.bfloat16))


@pytest.mark.parametrize("tokens", [33, 200, 700])
@pytest.mark.parametrize("width", [128, 1000])
def test_rows_of_pairs_have_an_exponent_per_run(tokens, width, device):
    """Channels in runs of 32 whose magnitudes lie up to 2^60 apart: a pair's row keeps fp16's precision in each of them.

    With one entry of x and one hidden value that are not zero a pair's row is exact before it becomes fp16 (a value is off by
    2^-11 of it, or by 2^-25 2^-14 of its run's largest where it is subnormal).  The residual takes the row rounded to bf16 away,
    so that the last rounding is one of what is left."""

    torch.manual_seed(tokens + width)
    experts, ff = 6, 64
    scale = 2.0 ** torch.randint(-30, 31, ((width + 31) // 32,), device=device).double().repeat_interleave(32)[:width]
    gate_up = torch.zeros(experts, 2 * ff, width, dtype=torch.bfloat16, device=device)
    gate_up[:, 3, 5] = 1.0
    gate_up[:, ff + 3, 5] = 1.0
    down = (torch.randn(experts, width, ff, device=device).double() * scale[:, None]).to(torch.bfloat16)
    x = torch.zeros(tokens, width, dtype=torch.bfloat16, device=device)
    x[:, 5] = 1.0
    ids = torch.randint(0, experts, (tokens, 1), device=device, dtype=torch.int32)
    # 1 + 2^-7: a hidden value of eight bits, so that a row has up to sixteen and is rounded as fp16.
    weights = torch.full((tokens, 1), 1.0 + 2.0 ** -7, device=device)
    row = down[ids[:, 0].long(), :, 3].double() * (1.0 + 2.0 ** -7)
    rounded = row.to(torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    out = expert_mlp(x, ids, weights, gate_up, down, activation="none", residual=-rounded, status=status).double()
    runs = torch.nn.functional.pad(row.abs(), (0, -width % 32)).view(tokens, -1, 32).amax(dim=2)
    bound = 2.0 ** -11 * row.abs() + 2.0 ** -39 * runs.repeat_interleave(32, dim=1)[:, :width]
    left = row - rounded.double()
    bound = bound + 2.0 ** -8 * (left.abs() + bound) + 2.0 ** -23 * row.abs()
    assert_within(out, left, bound)


def test_feed_forward_refuses(device):
    x, gate_up, down = torch.zeros(2, 16, device=device).bfloat16(), *pool(4, 16, 8, device)
    ids, weights = torch.zeros(2, 2, dtype=torch.int32, device=device), torch.zeros(2, 2, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    for change, message in (({"down": down[:, :, :7]}, "down"), ({"gate_up": gate_up[:3]}, "down"), ({"x": x[:, :8]}, "gate_up"),
                            ({"ids": ids.float()}, "ids"), ({"ids": ids[:1]}, "ids"), ({"weights": weights.double()}, "weights"),
                            ({"weights": weights[:, :1]}, "weights"), ({"weights": weights.t()}, "weights"),
                            ({"residual": x[:1]}, "residual"), ({"x": x.clone().requires_grad_()}, "gradient")):
        given = {"x": x, "ids": ids, "weights": weights, "gate_up": gate_up, "down": down, **change}
        with pytest.raises(ValueError, match=message):
            expert_mlp(**given, status=status)
    assert expert_mlp(x[:0], ids[:0], weights[:0], gate_up, down, status=status).shape == (0, 16)


# -- together ---------------------------------------------------------------------------------------------------

def routed_layer(x, stream, layer, status):
    """Router, routed experts and a shared expert onto the residual stream, as a decoder layer runs them."""

    logits = fused_linear(x, layer["router"], status=status)
    ids, weights = route_experts(logits, 4, scores="sigmoid", bias=layer["balance"], groups=4, top_groups=2, group_best=2,
                                 scale=2.5, status=status)
    routed = expert_mlp(x, ids, weights, layer["gate_up"], layer["down"], residual=stream, status=status)
    hidden = fused_linear(x, layer["shared_gate_up"], activation="silu", gated=True, status=status)
    return ids, weights, hidden, fused_linear(hidden, layer["shared_down"], residual=routed, status=status), routed


@pytest.mark.parametrize("tokens", [1, 24, 500])
def test_a_routed_layer(tokens, device):
    """The run of all operators, eagerly, captured and replayed over new inputs, each against its definition on what the
    one before it gave."""

    torch.manual_seed(tokens)
    gate_up, down = pool(16, 256, 128, device)
    layer = {"gate_up": gate_up, "down": down, "router": (torch.randn(16, 256, device=device) / 16).bfloat16(),
             "balance": 0.05 * torch.randn(16, device=device),
             "shared_gate_up": (torch.randn(512, 256, device=device) / 16).bfloat16(),
             "shared_down": (torch.randn(256, 256, device=device) / 16).bfloat16()}
    x, stream = torch.randn(tokens, 256, device=device).bfloat16(), torch.randn(tokens, 256, device=device).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=device)

    def verify(ids, weights, hidden, out, routed):
        from product_bounds import fused_linear as exact_fused_linear

        logits = fused_linear(x, layer["router"], status=status)
        exact_ids, _ = plain_route(logits, 4, scores="sigmoid", bias=layer["balance"], groups=4, top_groups=2, group_best=2)
        assert np.array_equal(ids.cpu().numpy(), exact_ids)
        assert_within(routed, *exact_expert_mlp(x, ids, weights, gate_up, down, "silu", stream))
        assert_within(hidden, *exact_fused_linear(x, layer["shared_gate_up"], None, "silu", True, None))
        assert_within(out, *exact_fused_linear(hidden, layer["shared_down"], None, "none", False, routed))

    verify(*routed_layer(x, stream, layer, status))
    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = routed_layer(x, stream, layer, status)
        graphs.append((graph, results))
    for step in range(4):
        x.copy_(torch.randn(tokens, 256, device=device))
        stream.copy_(torch.randn(tokens, 256, device=device))
        graph, results = graphs[step % 2]
        graph.replay()
        verify(*results)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = routed_layer(x, stream, layer, status)
    here = routed_layer(x, stream, layer, status)  # two at once
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(beside, here))
    assert int(status.item()) == 0


def test_a_status_that_the_device_cannot_write(device):
    x, gate_up, down = torch.zeros(2, 16, device=device).bfloat16(), *pool(4, 16, 8, device)
    ids, weights = torch.zeros(2, 2, dtype=torch.int32, device=device), torch.zeros(2, 2, device=device)
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=device),
                   torch.zeros(0, dtype=torch.int32, device=device)):
        with pytest.raises(ValueError, match="int32 word"):
            expert_mlp(x, ids, weights, gate_up, down, status=status)
        with pytest.raises(ValueError, match="int32 word"):
            fused_linear(x, x, status=status)
