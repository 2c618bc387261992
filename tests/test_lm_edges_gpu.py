"""Edges of the operators around the attention layers on the GPU: batches without a token, gradients of very different sizes and
infinite ones, a word with all the weight, 16-bit views, operands and rows of probabilities past 2^31 bytes, forward-mode derivatives.

U, half and the bounds are test_lm_gpu's."""

import math

import pytest
import torch

import selective_attention as sa
from test_lm_gpu import BF16, F16, F32, randn, xent_check, xent_inputs, xent_run

pytestmark = pytest.mark.gpu

THREE = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t)[6:])


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape", [(0,), (0, 5), (3, 0)], ids=str)
@THREE
def test_no_tokens(cuda, reduction, shape, dtype):
    """A batch without a token: the loss of no terms, gradients of zeros of either tensor or both, whatever weight holds."""
    for first in (1.0, math.inf, math.nan):
        w = torch.ones(7, 16, device="cuda", dtype=dtype)
        w[0] = first
        x, t = torch.empty(*shape, 16, device="cuda", dtype=dtype), torch.empty(shape, device="cuda", dtype=torch.int64)
        scored = sa.linear_cross_entropy(x, w, t, reduction=reduction)
        for need in ((True, True), (True, False), (False, True)):
            x, w = x.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
            loss = sa.linear_cross_entropy(x, w, t, reduction=reduction)
            for each in (loss, scored):
                assert each.dtype is F32 and each.shape == (shape if reduction == "none" else ())
                assert each.isnan() if reduction == "mean" else (each == 0).all()
            leaves = [a for a, n in zip((x, w), need) if n]
            for a, d in zip(leaves, torch.autograd.grad(loss, leaves, torch.full_like(loss, 2.0))):
                assert d.shape == a.shape and d.dtype is dtype and (d == 0).all()


@THREE
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=str)
def test_a_gradient_that_is_no_number(cuda, dtype, bad):
    """One token's incoming gradient is an infinity or a NaN: its own dx and all of dW are none either, the other tokens' dx keep their bits."""
    g = torch.Generator(device="cuda").manual_seed(31)
    x, w, t = xent_inputs(g, 70, 400, 64, dtype, dtype)
    dloss = randn(g, 70)
    dloss[3], dloss[4] = 4.0, 0.25   # (the largest is another's)
    clean = xent_run(x, w, t, "none", dloss)
    dloss = dloss.clone()
    dloss[4] = bad
    loss, _, dx, dw = xent_run(x, w, t, "none", dloss)
    sound = torch.arange(70, device="cuda") != 4
    assert torch.equal(loss, clean[0]) and torch.equal(dx[sound], clean[2][sound])
    assert not dx[4].isfinite().any() and not dw.isfinite().any()


@pytest.mark.parametrize("dtype,width", [(BF16, 96), (F32, 48)], ids=["bf16", "f32"])
def test_tokens_past_31_bits(cuda, dtype, width):
    """More than 2^31 bytes of rows, whose contraction is no multiple of the loop's four stages: the stages behind it read nothing, so that the NaN
    of a token 2^31 - 256 bytes behind the first reaches no other."""
    n, row = (1 << 31) // 192 + 1000, 192   # bytes
    g = torch.Generator(device="cuda").manual_seed(35)
    x = torch.empty(n, width, device="cuda", dtype=dtype).normal_(generator=g)
    ill = torch.tensor([0x7fffff00 // row, (0x7fffff00 + 63) // row], device="cuda").unique()
    x[ill] = math.nan
    w, t = randn(g, 40, width).to(dtype), torch.randint(40, (n,), device="cuda", generator=g)
    each = sa.linear_cross_entropy(x, w, t, reduction="none")
    sound = torch.ones(n, device="cuda", dtype=torch.bool)
    sound[ill] = False
    assert each[ill].isnan().all() and each[sound].isfinite().all()
    for part in (slice(0, 300), slice(n - 300, n)):
        xent_check(x[part], w, t[part], "none", dtype, each[part])
