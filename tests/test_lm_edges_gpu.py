"""Edges of the operators around the attention layers on the GPU: batches without a token, gradients of very different sizes and
infinite ones, a word with all the weight, 16-bit views, operands and rows of probabilities past 2^31 bytes, forward-mode derivatives.

U, half and the bounds are test_lm_gpu's."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import selective_attention as sa
from selective_attention import lm
from test_lm_gpu import BF16, F16, F32, F64, U, assert_within, half, randn, rounding, xent_check, xent_inputs, xent_run

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


@THREE
@pytest.mark.parametrize("n,vocab,width", [(50, 3001, 96), (300, 700, 200)])
def test_gradients_of_very_different_sizes(cuda, dtype, n, vocab, width):
    """Tokens' incoming gradients from 1 down to 1e-12, and 0: every row of dx is as exact as it is alone.

    As in xent_check, with each token's own f in the place of the largest: G_i = (p - onehot) f is held at 2^14 times its size beside the power of two
    at or below f_i, so its entries are off by half a step of fp16, or by 2^-39 of that power below fp16's normal numbers. In dW the rest of f_i is on
    the rows of x, the largest at 2^14: those are off by 2^-39 of the largest x f / (factor below 2) where they fall below fp16's normal numbers."""
    g = torch.Generator(device="cuda").manual_seed(32)
    x, w, t = xent_inputs(g, n, vocab, width, dtype, dtype)
    f = torch.pow(10.0, -12 * torch.rand(n, device="cuda", generator=g)) * torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    f[0], f[1], f[2], f[3] = 1.0, 1e-12, 0.0, -1e-9
    _, _, dx, dw = xent_run(x, w, t, "none", f)
    x64, w64, f64 = x.double(), w.double(), f.double()
    l = x64 @ w64.T
    dl = (width + 2) * U * (x64.abs() @ w64.abs().T).amax(1)
    lse = torch.logsumexp(l, 1)
    e_lse = dl + U * (160 + vocab / 1024) + 2.0 ** -22 * (4 + lse.abs())
    p = torch.exp(l - lse[:, None])
    G = p.clone()
    G[torch.arange(n, device="cuda"), t] -= 1.0
    fine, tiny = (0.0, 0.0) if dtype is F32 else (half(F16), 2.0 ** -38)
    e_G = (fine + U) * G.abs() + p * (2 * dl + e_lse)[:, None] * 1.01 + 3 * U * p + tiny
    size = f64.abs()[:, None]
    want = f64[:, None] * (G @ w64)
    bound = ((e_G + (vocab + 8) * U * G.abs()) * size) @ w64.abs()
    if dtype is BF16:
        bound += 2.0 ** -38 * w64.abs().max() * (size * G.abs()).sum(1, keepdim=True)
    assert (dx[2] == 0).all()
    assert_within(dx, want, bound * 1.01 + rounding(want, dtype), "dx")
    want = (f64[:, None] * G).T @ x64
    bound = ((e_G + (n + 8) * U * G.abs()) * size).T @ x64.abs() + tiny * x64.abs().max() * G.abs().sum(0)[:, None]
    assert_within(dw, want, bound * 1.01 + rounding(want, dtype), "dw")
    other = f.clone()
    other[::2] *= 1e7
    assert torch.equal(xent_run(x, w, t, "none", other)[2][1::2], dx[1::2])


@pytest.mark.parametrize("n", [20, 200, 600])
@pytest.mark.parametrize("dtype,far", [(BF16, 1.0), (F16, 1.0), (F32, 1.0), (BF16, 2.0 ** 116), (F32, 2.0 ** 116)], ids=str)
def test_a_word_with_all_the_weight(cuda, dtype, n, far):
    """The target's logit is 60 to 4000 (or near the end of fp32's range) and the others' are 25 or more below it: the loss is 0 but for 700 e^-25 <
    2^-26, and never below 0. The largest's own term of the sum is 1 and the others' do not change it; the gradient is at most that of
    the target's row, a step of 2^-23 in its probability, and of the others'."""
    g = torch.Generator(device="cuda").manual_seed(33)
    w = randn(g, 700, 256).sign() / 16   # (rows of norm 1; two have a product of at most 0.5)
    assert (w @ w.T - torch.eye(700, device="cuda")).max() < 0.5
    t = torch.randint(700, (n,), device="cuda", generator=g)
    x = (far * torch.randint(60, 4000, (n, 1), device="cuda", generator=g) * w[t]).to(dtype)   # (sums of 256 equal numbers: exact)
    x[0] = (far * 4000 * w[t[0]]).to(dtype)
    w = w.to(dtype)
    loss, _, dx, dw = xent_run(x, w, t, "none", torch.ones(n, device="cuda"))
    for each in (loss, sa.linear_cross_entropy(x, w, t, reduction="none")):
        assert (each >= 0).all() and each.max() <= 2.0 ** -23
    assert dx.abs().max() <= 2.0 ** -22 / 16
    assert 0 <= sa.linear_cross_entropy(x, w, t) <= 2.0 ** -23


VIEWS = {"columns": ((40, 200), lambda b: b[:, 64:128]), "offset": ((40, 65), lambda b: b[:, 1:]), "wide": ((40, 192), lambda b: b[:, 128:]),
         "every second": ((80, 64), lambda b: b[::2]), "one row": ((1, 64), lambda b: b.expand(40, 64)),
         "transposed": ((64, 40), lambda b: b.T)}


@pytest.mark.parametrize("dtype", [BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("xv", VIEWS)
@pytest.mark.parametrize("wv", VIEWS)
def test_sixteen_bit_views(cuda, dtype, xv, wv):
    """Views of 16-bit tensors: rows read in place a stride apart, rows of odd alignment, one row for all."""
    g = torch.Generator(device="cuda").manual_seed(34)
    x, w = (view(randn(g, *(s if i == 0 else tuple(2 * e if e in (40, 80) else e for e in s))).to(dtype))
            for i, (s, view) in enumerate((VIEWS[xv], VIEWS[wv])))
    assert not x.is_contiguous() and not w.is_contiguous() and x.shape[1] == w.shape[1] == 64
    t = torch.randint(w.shape[0], (40,), device="cuda", generator=g)
    t[::7] = -100
    loss, dloss, dx, dw = xent_run(x, w, t, "mean")
    xent_check(x, w, t, "mean", dtype, loss, dloss, dx, dw)
    xent_check(x, w, t, "none", dtype, sa.linear_cross_entropy(x, w, t, reduction="none"))


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


def test_words_past_26_bits(cuda):
    """Two tokens over more than 2^26 words, whose rows of G are longer than 2^27 bytes: in pieces, each of which lies within a tile's offsets."""
    n, vocab, width = 2, (1 << 26) + 70000, 32
    g = torch.Generator(device="cuda").manual_seed(36)
    w = torch.empty(vocab, width, device="cuda", dtype=F16).normal_(generator=g)
    t = torch.tensor([vocab - 5, 12345], device="cuda")
    x = randn(g, n, width).half()
    loss, _, dx, dw = xent_run(x, w, t, "sum")
    parts = [slice(a, min(a + (1 << 22), vocab)) for a in range(0, vocab, 1 << 22)]
    x64 = x.double()
    l = torch.cat([x64 @ w[p].double().T for p in parts], 1)
    dl = (width + 2) * U * torch.stack([(x64.abs() @ w[p].double().abs().T).amax(1) for p in parts]).amax(0)
    lse = torch.logsumexp(l, 1)
    e_lse = dl + U * (160 + vocab / 1024) + 2.0 ** -22 * (4 + lse.abs())
    at = torch.arange(n, device="cuda")
    each = lse - l[at, t]
    assert abs(loss.double() - each.sum()) <= (dl + e_lse + 5 * U * (lse.abs() + each)).sum()
    p_all = torch.exp(l - lse[:, None])
    del l
    want, bound = (torch.zeros(n, width, device="cuda", dtype=F64) for _ in range(2))
    for part in parts:
        p = p_all[:, part]
        G = p.clone()
        for i in range(n):
            if part.start <= int(t[i]) < part.stop:
                G[i, int(t[i]) - part.start] -= 1.0
        e_G = (half(F16) + U) * G.abs() + p * (2 * dl + e_lse)[:, None] * 1.01 + 3 * U * p + 2.0 ** -38
        w64 = w[part].double()
        dw_part = G.T @ x64
        assert_within(dw[part], dw_part, (e_G + (n + 8) * U * G.abs()).T @ x64.abs() * 1.01 + rounding(dw_part, F16), "dw")
        want += G @ w64
        # (a piece of the vocabulary has at most 2^21 words, and there are 33 of up to 64 parts)
        bound += (e_G + ((1 << 21) + 100) * U * G.abs()) @ w64.abs()
    assert_within(dx, want, bound * 1.01 + rounding(want, F16), "dx")


def test_forward_mode_derivatives_are_refused(cuda):
    """The operators have no forward-mode derivative and no batching rule, and say so: a tangent is not dropped."""
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(8, device="cuda")
    ids = torch.tensor([1, 0, 3, 2], device="cuda")
    calls = (lambda v: sa.layer_norm(v, w), lambda v: sa.add_layer_norm(x, v, w)[0], lambda v: sa.layer_norm(x, w, v[0]),
             lambda v: sa.embedding(ids, v), lambda v: sa.linear_cross_entropy(v, x, ids), lambda v: sa.linear_cross_entropy(x, v, ids))
    with forward_ad.dual_level():
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    call(forward_ad.make_dual(x, torch.ones_like(x)))
            call(x)   # (without a tangent there is nothing to refuse)
    for call in calls:
        for transformed in (lambda: torch.func.jvp(call, (x,), (torch.ones_like(x),)), lambda: torch.func.grad(lambda v: call(v).sum())(x),
                            lambda: torch.func.vmap(call)(x.expand(3, 4, 8))):
            with pytest.raises(RuntimeError):
                transformed()


@pytest.mark.parametrize("of", ["x", "weight", "both"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_rows_far_beyond_the_others(cuda, of, reduction):
    """A row of x, or of weight, 2^40 times as large as the others: the backward pass has the forward's probabilities all the same.

    Bounds as in xent_check with each logit's own dl (the largest's alone would cover everything): the sum of the exponentials is off by what
    those that have weight are. The gradients' products hold x and weight beside their largest number, off by 2^-38 of that times
    the G it meets: so dx is as exact as ever beside a row of x, dw beside one of weight."""
    n, vocab, width = 200, 900, 64
    g = torch.Generator(device="cuda").manual_seed(37)
    x, w, t = xent_inputs(g, n, vocab, width, BF16, BF16)
    if of != "weight":
        x[7] *= 2.0 ** 40
    if of != "x":
        w[9] *= 2.0 ** 40
    f = randn(g, n) if reduction == "none" else torch.full((n,), 1.0 / n, device="cuda")
    each, _, dx, dw = xent_run(x, w, t, reduction, f if reduction == "none" else None)
    x64, w64, f = x.double(), w.double(), f.double()[:, None]
    l = x64 @ w64.T
    p = torch.softmax(l, 1)
    dl = (width + 2) * U * (x64.abs() @ w64.abs().T)
    e_lse = ((p * dl).sum(1) + U * (160 + vocab / 1024) + 2.0 ** -22 * (4 + torch.logsumexp(l, 1).abs()))[:, None]
    G = p.clone()
    G[torch.arange(n, device="cuda"), t] -= 1.0
    e_G = (half(F16) + U) * G.abs() + p * (2 * dl + e_lse) * 1.01 + 3 * U * p + 2.0 ** -38
    want, size = f * (G @ w64), (f * G).abs()
    bound = ((e_G * f.abs() + (vocab + 8) * U * size) @ w64.abs() + 2.0 ** -38 * w64.abs().max() * size.sum(1, keepdim=True)) * 1.01
    assert_within(dx, want, bound + rounding(want, BF16), "dx")
    if of == "x":
        assert (bound[torch.arange(n, device="cuda") != 7] < 0.01 * f.abs().max()).all()
    want = (f * G).T @ x64
    bound = (e_G * f.abs() + (n + 8) * U * size).T @ x64.abs() + 2.0 ** -38 * x64.abs().max() * f.abs().max() * G.abs().sum(0)[:, None]
    assert_within(dw, want, bound * 1.01 + rounding(want, BF16), "dw")


@THREE
def test_reductions_of_the_two_passes(cuda, dtype):
    """What the forward pass leaves serves a backward pass of either reduction."""
    g = torch.Generator(device="cuda").manual_seed(38)
    x, w, t = xent_inputs(g, 90, 300, 64, dtype, dtype, ignored=0.2)
    code, none, total = lm._CODES[dtype], 0, 2
    dloss, one = randn(g, 90), torch.full((1,), 0.75, device="cuda")
    for forward in (none, 1, total):
        torch.full((4096,), 0x7f7f7f7f, device="cuda", dtype=torch.int32)   # (what is left in memory is no magnitude)
        _, lse, rows = lm._xent_impl(x, w, t, -100, forward, code, True)
        got = [lm._xent_backward_impl(x, w, t, lse, rows, d, r, code, True, True) for r, d in ((none, dloss), (total, one))]
        if forward == none:
            want = got
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q)), forward


@pytest.mark.parametrize("n,vocab,ignored", [(1, 700, 0.2), (2, 700, 0.2), (7, 700, 0.2), (32, 700, 0.2), (33, 700, 0.2), (64, 700, 0.2),
                                             (300, 700, 0.95), (2000, 700, 0.98), (5000, 20000, 0.992)])
@pytest.mark.parametrize("reduction", [0, 1])
def test_few_tokens_in_fp16(cuda, n, vocab, ignored, reduction):
    """Up to 64 tokens that are not ignored, with fp16 operands, have G in two numbers, to 22 bits: seen in fp32 gradients of fp32 tensors of fp16 numbers.

    Bounds as in xent_check, with 2^-22 of G in the place of 2^-11."""
    width = 16
    g = torch.Generator(device="cuda").manual_seed(39)
    x, w, t = xent_inputs(g, n, vocab, width, F16, F16, ignored=ignored)
    t[0] = 5
    kept = t != -100
    assert kept.sum() <= 64
    code = lm._CODES[F16]
    dloss = randn(g, n) if reduction == 0 else torch.ones((), device="cuda")
    _, lse, rows = lm._xent_impl(x.float(), w.float(), t, -100, reduction, code, True)
    dx, dw = lm._xent_backward_impl(x.float(), w.float(), t, lse, rows, dloss, reduction, code, True, True)
    x64, w64, at = x.double()[kept], w.double(), t[kept]
    f = (dloss.double()[kept] if reduction == 0 else torch.full((len(at),), 1.0 / len(at), device="cuda", dtype=F64))[:, None]
    l = x64 @ w64.T
    dl = (width + 2) * U * (x64.abs() @ w64.abs().T).amax(1)
    lse64 = torch.logsumexp(l, 1)
    e_lse = dl + U * (160 + vocab / 1024) + 2.0 ** -22 * (4 + lse64.abs())
    p = torch.exp(l - lse64[:, None])
    G = p.clone()
    G[torch.arange(len(at), device="cuda"), at] -= 1.0
    e_G = ((2.0 ** -22 + 3 * U) * G.abs() + p * (2 * dl + e_lse)[:, None] * 1.01 + 3 * U * p + 2.0 ** -38) * f.abs()
    G = G * f
    want = G @ w64
    assert (dx[~kept] == 0).all()
    assert_within(dx[kept], want, ((e_G + (2 * vocab + 8) * U * G.abs()) @ w64.abs()) * 1.01 + rounding(want, F32), "dx")
    want = G.T @ x64
    assert_within(dw, want, ((e_G + (2 * len(at) + 8) * U * G.abs()).T @ x64.abs() + 2.0 ** -38 * x64.abs().max() * f.abs().max() * p.sum(0)[:, None]) * 1.01
                  + rounding(want, F32), "dw")
