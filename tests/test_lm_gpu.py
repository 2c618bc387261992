"""The operators around the attention layers on the GPU against float64, within bounds taken from the arithmetic; their edges;
and a run of them together, as the decoder's fused loss.

u = 2^-24 is half a step of fp32, h(t) = finfo(t).eps / 2 half a step of an output's type (relative to the value, with the
type's smallest normal number below it)."""

import math

import pytest
import torch

import selective_attention as sa
from selective_attention import kernels, lm
from selective_attention.model import ModelConfig, SelectiveLM

pytestmark = pytest.mark.gpu

F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def rounding(value, dtype):
    """What rounding float64 `value` to dtype may change: half a step, half the smallest subnormal below the normal numbers."""
    return half(dtype) * value.abs() + torch.finfo(dtype).smallest_normal * half(dtype)


def assert_within(got, want, bound, name=""):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    worst = ((got - want).abs() / (bound + 1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times the bound"


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


# -- layer norm -------------------------------------------------------------------------------------------

def norm_check(x, branch, w, b, dtype, eps=1e-5, outs=None, grads=None, dy=None, ds=None):
    """Asserts a norm's results, and its gradients' where given.

    A lane adds up to 32 of a row's elements one after the other, then 6 exchanges and up to 16 wavefronts: sums of a row are off by at most
    60 u of the sum of the magnitudes. So mean by 60 u max|s|, the variance by 60 u + 3 u of itself (and the mean's error squared), rstd by 35
    u with its square root and division; h = (s - mean) rstd by dh = 62 u max|s| rstd + 37 u |h|."""
    s = x.double() if branch is None else (x.double() + branch.double()).to(x.dtype).double()
    if branch is not None:
        exact = x.double() + branch.double()
        # (the fp32 sum is rounded again to a 16-bit stream, which may move it by a step where it falls between two)
        assert_within(outs[1], exact, rounding(exact, x.dtype) + U * exact.abs(), "s")
        s = outs[1].double()
    mean = s.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((s - mean).square().mean(-1, keepdim=True) + eps)
    h = (s - mean) * r
    dh = 62 * U * s.abs().amax(-1, keepdim=True) * r + 37 * U * h.abs()
    w64, b64 = w.double(), 0.0 if b is None else b.double()
    y = h * w64 + b64
    assert outs[0].dtype is dtype
    assert_within(outs[0], y, (dh * w64.abs() + 3 * U * (h * w64).abs() + U * y.abs()) * (1 + half(dtype)) + rounding(y, dtype), "y")
    if grads is None:
        return
    dy64 = dy.double()
    v = dy64 * w64
    mv, mvh = v.mean(-1, keepdim=True), (v * h).mean(-1, keepdim=True)
    dx = r * (v - mv - h * mvh)
    e_mv = 62 * U * v.abs().mean(-1, keepdim=True)
    e_mvh = 62 * U * (v * h).abs().mean(-1, keepdim=True) + (v.abs() * dh).mean(-1, keepdim=True)
    e = r * (e_mv + h.abs() * e_mvh + dh * mvh.abs() + 4 * U * (v.abs() + mv.abs() + (h * mvh).abs())) + 37 * U * dx.abs()
    if ds is not None:
        dx = dx + ds.double()
        e = e + 2 * U * (dx.abs() + ds.double().abs())
    assert_within(grads["x"], dx, e * 1.01 + rounding(dx, x.dtype), "dx")
    if branch is not None:
        assert_within(grads["branch"], dx, e * 1.01 + rounding(dx, branch.dtype), "dbranch")
    rows = s.reshape(-1, s.shape[-1]).shape[0]
    depth = rows / 512 + 64   # a workgroup's rows in turn, then the workgroups' sums: 32 in turn, 16 and 4 more
    terms = lambda t: t.reshape(rows, -1).sum(0)
    dw = terms(dy64 * h)
    assert_within(grads["w"], dw, terms(dy64.abs() * dh) + depth * U * terms((dy64 * h).abs()) + rounding(dw, w.dtype), "dw")
    if b is not None:
        db = terms(dy64)
        assert_within(grads["b"], db, depth * U * terms(dy64.abs()) + rounding(db, b.dtype), "db")


NORMS = [(1, 1), (1, 64), (3, 7), (5, 256), (37, 513), (64, 768), (130, 1000), (33, 1001), (9, 1024), (17, 2048), (5, 2049), (3, 4096),
         (4, 5000), (2, 8192), (3, 8193), (2, 16384), (2, 16385), (2, 32768), (2100, 96)]
TYPES = [(F32, BF16, BF16, F32), (BF16, BF16, BF16, BF16), (F16, F32, F32, F16), (F32, None, F32, F32), (BF16, None, F16, F32),
         (F32, F32, F16, BF16)]


@pytest.mark.parametrize("rows,width", NORMS)
@pytest.mark.parametrize("xt,bt,yt,wt", TYPES, ids=lambda t: str(t)[6:])
def test_layer_norm(cuda, rows, width, xt, bt, yt, wt):
    g = torch.Generator(device="cuda").manual_seed(rows * 40000 + width)
    x = (2 * randn(g, rows, width) + 0.7).to(xt).requires_grad_()
    branch = None if bt is None else randn(g, rows, width).to(bt).requires_grad_()
    w = (1 + 0.2 * randn(g, width)).to(wt).requires_grad_()
    b = (0.3 * randn(g, width)).to(wt).requires_grad_() if (rows + width) % 2 else None
    dy, ds = randn(g, rows, width).to(yt), randn(g, rows, width).to(xt)
    outs = (sa.layer_norm(x, w, b, dtype=yt),) if bt is None else sa.add_layer_norm(x, branch, w, b, dtype=yt)
    leaves = {n: t for n, t in (("x", x), ("branch", branch), ("w", w), ("b", b)) if t is not None}
    grads = torch.autograd.grad(outs, tuple(leaves.values()), (dy, ds)[:len(outs)])
    for t, d in zip(leaves.values(), grads):
        assert d.shape == t.shape and d.dtype is t.dtype
    detached = [None if t is None else t.detach() for t in (x, branch, w, b)]
    norm_check(*detached, yt, outs=[o.detach() for o in outs], grads=dict(zip(leaves, grads)), dy=dy, ds=None if bt is None else ds)
    with torch.no_grad():   # the same bits without a gradient asked for
        again = (sa.layer_norm(x, w, b, dtype=yt),) if bt is None else sa.add_layer_norm(x, branch, w, b, dtype=yt)
    assert all(torch.equal(a, o) for a, o in zip(again, outs))


def test_layer_norm_views(cuda):
    """Strided rows, broadcast rows and weights, odd alignments, transposed and negated views, more dimensions."""
    g = torch.Generator(device="cuda").manual_seed(5)
    base = randn(g, 6, 10, 3 * 96 + 1)
    w, b = randn(g, 96), randn(g, 96)
    cases = [base[..., 96:192], base[..., 97:193], base[:, :, :96][1], base[:, ::2, 5:101], randn(g, 1, 96).expand(7, 96),
             randn(g, 96, 20).T, torch.complex(base[..., :96], base[..., 96:192]).conj().imag, randn(g, 2, 3, 4, 96)]
    for x in cases:
        branch = randn(g, *x.shape).flip(0)
        norm_check(x, None, w, b, F32, outs=[sa.layer_norm(x, w, b)])
        norm_check(x, branch, w, b, BF16, outs=sa.add_layer_norm(x, branch, w, b, dtype=BF16))
        norm_check(branch, x, w, b, BF16, outs=sa.add_layer_norm(branch, x, w, b, dtype=BF16))
    # gradients that arrive as views, and none for one of the results
    x, branch = randn(g, 6, 96).requires_grad_(), randn(g, 6, 96).bfloat16().requires_grad_()
    for dy, ds in ((torch.ones(1, 1, device="cuda").expand(6, 96), randn(g, 96, 6).T), (randn(g, 6, 200)[:, 50:146], None),
                   (None, randn(g, 6, 96))):
        y, s = sa.add_layer_norm(x, branch, w, b)
        outs, given = zip(*[(o, d) for o, d in ((y, dy), (s, ds)) if d is not None])
        dx, dbranch = torch.autograd.grad(outs, (x, branch), given)
        want_dy = torch.zeros(6, 96, device="cuda") if dy is None else dy
        s64 = s.detach().double()
        h = s64 - s64.mean(-1, keepdim=True)
        r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5)
        h = h * r
        v = want_dy.double() * w.double()
        want = r * (v - v.mean(-1, keepdim=True) - h * (v * h).mean(-1, keepdim=True)) + (0.0 if ds is None else ds.double())
        # (the bound of norm_check on numbers of this size: |s| < 12, |h| < 5, r < 3, |v| < 16)
        assert (dx.double() - want).abs().max() < 3 * (62 * 16 + 5 * 62 * 80 + 62 * 36 * 16 + 4 * 100) * U
        assert (dbranch.double() - want).abs().max() < 3 * (62 * 16 + 5 * 62 * 80 + 62 * 36 * 16 + 4 * 100) * U + half(BF16) * 64


def test_layer_norm_edges(cuda):
    x = torch.randn(4, 96, device="cuda", requires_grad=True)
    w = torch.ones(96, device="cuda", requires_grad=True)
    # constant rows: no variance, eps alone keeps the division; a row of NaN and one with an infinity stay in their rows
    with torch.no_grad():
        x[1] = 3.0
        x[2, 5] = math.nan
        x[3, 5] = math.inf
    y = sa.layer_norm(x, w)
    assert (y[1] == 0).all() and y[0].isfinite().all() and y[2].isnan().all() and y[3].isnan().all()
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx[:2].isfinite().all() and dx[2:].isnan().all()
    # large offsets: the squared deviations come from the deviations, not from a difference of sums
    big = torch.randn(3, 1000, device="cuda") + 4096.0
    norm_check(big, None, torch.ones(1000, device="cuda"), None, F32, outs=[sa.layer_norm(big, torch.ones(1000, device="cuda"))])
    # no rows
    e = torch.empty(0, 5, 96, device="cuda", requires_grad=True)
    y, s = sa.add_layer_norm(e, e, w, dtype=BF16)
    assert y.shape == s.shape == (0, 5, 96) and y.dtype == BF16
    de, dw = torch.autograd.grad((y, s), (e, w), (y.detach(), s.detach()))
    assert de.shape == e.shape and (dw == 0).all()
    # the same tensor twice, and gradients of some of the inputs only
    y, s = sa.add_layer_norm(x[:1], x[:1], w)
    dx, = torch.autograd.grad((y, s), x, (torch.zeros_like(y), torch.ones_like(s)))
    assert (dx[0] == 2).all() and (dx[1:] == 0).all()
    # two leaves that get the same gradient have it in memory of their own, also where it adds to what is there
    two = [torch.randn(5, 96, device="cuda", requires_grad=True) for _ in range(2)]
    for k in (1, 2):
        y, s = sa.add_layer_norm(*two, w.detach())
        (y.sum() + 2.0 * s.sum()).backward()
        assert two[0].grad.data_ptr() != two[1].grad.data_ptr() and torch.equal(two[0].grad, two[1].grad)
        assert (two[0].grad - 2.0 * k).abs().max() < 1e-4   # (y's rows sum to 0 whatever x is: |u| = 1, rstd < 2, 200 u of it)
    frozen = x[:2].detach()
    dw, = torch.autograd.grad(sa.layer_norm(frozen, w), w, torch.ones(2, 96, device="cuda"))
    assert dw.shape == w.shape


def test_layer_norm_difference(cuda):
    """The gradient against differences: of every input of a small call, along a random direction."""
    g = torch.Generator(device="cuda").manual_seed(7)
    args = [randn(g, 8, 40).requires_grad_(), randn(g, 8, 40).requires_grad_(), randn(g, 40).requires_grad_(), randn(g, 40).requires_grad_()]
    dy, ds = randn(g, 8, 40), randn(g, 8, 40)
    f = lambda a: sum((o.double() * d.double()).sum() for o, d in zip(sa.add_layer_norm(*a), (dy, ds)))
    grads = torch.autograd.grad(f(args), args)
    for k in range(4):
        d = randn(g, *args[k].shape)
        step = 1e-2
        with torch.no_grad():
            moved = [[a + (sign * step * d if i == k else 0) for i, a in enumerate(args)] for sign in (1, -1)]
            slope = (f(moved[0]) - f(moved[1])) / (2 * step)
        want = (grads[k].double() * d.double()).sum()
        # fp32 rounding of 640 outputs below 16 over the step (random signs: sqrt(640)); the third derivative's share, step^2
        assert abs(slope - want) < 640 ** 0.5 * 64 * 16 * U / step + 40 * step ** 2 * 320 ** 0.5, k


# -- embedding --------------------------------------------------------------------------------------------

def embed_check(ids, w, scale, y=None, dy=None, dw=None):
    """A table row is rounded once after one product; a gradient row adds up to 32 tokens in turn, then every eighth of its parts of 32 and
    8 sums: at most 32 + n / 256 + 9 roundings of the running sum, and one product."""
    if y is not None:
        want = scale * w.double()[ids.long()]
        assert_within(y, want, U * want.abs() + rounding(want, w.dtype) if scale != 1.0 else 0 * want, "y")
    if dw is not None:
        flat, d = ids.reshape(-1).long(), dy.double().reshape(-1, w.shape[1])
        total, size = torch.zeros(w.shape, dtype=F64, device="cuda"), torch.zeros(w.shape, dtype=F64, device="cuda")
        total.index_add_(0, flat, d)
        size.index_add_(0, flat, d.abs())
        depth = (42 + torch.bincount(flat, minlength=w.shape[0]) / 256)[:, None]
        want = scale * total
        assert_within(dw, want, U * depth * abs(scale) * size + rounding(want, w.dtype), "dw")
        assert (dw[torch.bincount(flat, minlength=w.shape[0]) == 0] == 0).all()


EMBEDS = [(1, 1, 1), (1, 300, 64), (31, 5, 7), (32, 1, 256), (33, 1, 256), (64, 2, 257), (1000, 257, 768), (4097, 50304, 96),
          (5000, 256, 1001), (8193, 1000, 33), (20000, 3, 64), (16384, 70001, 40), (3000, 600001, 8)]


@pytest.mark.parametrize("tokens,vocab,width", EMBEDS)
@pytest.mark.parametrize("dtype,scale", [(F32, 1.0), (BF16, 27.7), (F16, 1.0)], ids=lambda t: str(t))
def test_embedding(cuda, tokens, vocab, width, dtype, scale):
    g = torch.Generator(device="cuda").manual_seed(tokens + vocab)
    w = randn(g, vocab, width).to(dtype).requires_grad_()
    # (each id as likely as the one before it is not: few ids have most of the tokens)
    ids = (torch.exp(torch.rand(tokens, device="cuda", generator=g) * math.log(vocab + 1)) - 1).long().clamp_max(vocab - 1)
    ids = ids.int() if tokens % 2 else ids
    dy = randn(g, tokens, width).to(dtype)
    y = sa.embedding(ids, w, scale)
    dw, = torch.autograd.grad(y, w, dy)
    assert y.dtype is dtype and dw.dtype is dtype
    embed_check(ids, w.detach(), scale, y.detach(), dy, dw)
    assert torch.equal(sa.embedding(ids, w.detach(), scale), y)


@pytest.mark.parametrize("of", ["one", "last", "two in turn", "sorted", "runs of 32", "runs of 33"])
def test_embedding_gradient_of_uneven_ids(cuda, of):
    """One id has all the tokens, every other one; ids that begin and end with the pieces the tokens are summed in."""
    n, vocab = 3001, 300
    i = torch.arange(n, device="cuda")
    ids = {"one": 0 * i, "last": 0 * i + vocab - 1, "two in turn": 255 + i % 2, "sorted": i // 11, "runs of 32": i // 32,
           "runs of 33": i // 33}[of]
    g = torch.Generator(device="cuda").manual_seed(8)
    w, dy = randn(g, vocab, 300).requires_grad_(), randn(g, n, 300)
    dw, = torch.autograd.grad(sa.embedding(ids, w), w, dy)
    embed_check(ids, w.detach(), 1.0, None, dy, dw)
    order = torch.argsort(ids, stable=True)   # the sums go by the tokens' order, not by how the ids lie
    again, = torch.autograd.grad(sa.embedding(ids[order], w), w, dy[order])
    assert torch.equal(dw, again)


def test_embedding_views_and_edges(cuda):
    g = torch.Generator(device="cuda").manual_seed(9)
    table = randn(g, 50, 200)
    ids = torch.randint(50, (4, 6), device="cuda", generator=g)
    for w in (table[:, 60:124], table[::2, 3:67][:25], randn(g, 64, 50).T, randn(g, 1, 64).expand(50, 64)):
        at = ids % w.shape[0]
        for i in (at, at.T, at[:, ::2], at[0, 0], at[:0]):
            y = sa.embedding(i, w)
            assert torch.equal(y, w[i.long()])
    leaf = table.clone().requires_grad_()
    y = sa.embedding(ids, leaf[:, 60:124])
    dleaf, = torch.autograd.grad(y, leaf, randn(g, 6, 4, 64).transpose(0, 1))
    assert (dleaf[:, :60] == 0).all() and (dleaf[:, 124:] == 0).all()
    # ids that are none: rows of NaN, no gradient, and the others' as they were
    bad = ids.clone()
    bad[1, 2], bad[3, 0], bad[0, 0] = 50, -1, 1 << 40
    dy = randn(g, 4, 6, 200)
    y = sa.embedding(bad, leaf)
    real = (bad >= 0) & (bad < 50)
    assert y[~real].isnan().all() and torch.equal(y[real], table[bad[real]])
    dw, = torch.autograd.grad(y, leaf, dy)
    embed_check(bad[real], table, 1.0, None, dy[real], dw)
    # no ids at all
    dw, = torch.autograd.grad(sa.embedding(ids[:0], leaf), leaf, torch.empty(0, 6, 200, device="cuda"))
    assert (dw == 0).all()


# -- the vocabulary loss ------------------------------------------------------------------------------------

def xent_inputs(g, n, vocab, width, xt, wt, ignored=0.0):
    w = (randn(g, vocab, width) * (2.5 / math.sqrt(width))).to(wt)
    t = torch.randint(vocab, (n,), device="cuda", generator=g)
    x = (randn(g, n, width) + 1.8 * w.float()[t]).to(xt)
    t[torch.rand(n, device="cuda", generator=g) < ignored] = -100
    return x, w, t


def xent_check(x, w, t, reduction, operand, loss, dloss=None, dx=None, dw=None, ignore=-100):
    """In float64 from the operands as the products take them.

    Logits: a sum of C products in fp32, off by at most dl = (C + 2) u sum|x w|. lse: dl, and u times the additions (128 rows of a tile in turn, 9
    more, then every eighth of the tiles and 8) plus 2^-22 of rounding in the exponentials and logarithm for arguments below 2^6.
    G = (p - onehot) f is rounded to fp16 at 2^14 times its size (fp32 operands: not at all), off by half a step of it, 2^-11, or 2^-39 of the
    factors' unit below its normal numbers, and p (2 dl + dlse) before that; bf16 operands are held in fp16 with the largest at
    2^14, the smallest off by 2^-39 of that. A gradient adds V (tokens) products in fp32."""
    x64, w64 = x.to(operand).double(), w.to(operand).double()
    kept = t != ignore
    x64, at = x64[kept], t[kept]
    l = x64 @ w64.T
    size = x64.abs() @ w64.abs().T
    dl = (x.shape[1] + 2) * U * size.amax(1)
    lse = torch.logsumexp(l, 1)
    e_lse = dl + U * (160 + w.shape[0] / 1024) + 2.0 ** -22 * (4 + lse.abs())
    each = torch.zeros(t.shape[0], dtype=F64, device="cuda")
    each[kept] = lse - l[torch.arange(len(at), device="cuda"), at]
    e_each = torch.zeros_like(each)
    e_each[kept] = dl + e_lse + 4 * U * (lse.abs() + each[kept].abs())
    if reduction == "none":
        assert_within(loss, each, e_each, "loss")
    else:
        n = len(at) if reduction == "mean" else 1
        total = each.sum() / n
        assert_within(loss, total, (e_each.sum() + (each.shape[0] / 32 + 40) * U * each.abs().sum()) / n, "loss")
    if dx is None and dw is None:
        return
    p = torch.exp(l - lse[:, None])
    G = p.clone()
    G[torch.arange(len(at), device="cuda"), at] -= 1.0
    f = dloss.double().expand(t.shape[0])[kept] if reduction == "none" else dloss.double() / (len(at) if reduction == "mean" else 1) + 0 * at
    unit = f.abs().max() if len(at) else 0.0
    fine, unit = (0.0, 0.0) if operand is F32 else (half(F16), unit)
    e_G = (fine + U) * G.abs() + p * (2 * dl + e_lse)[:, None] * 1.01 + 3 * U * p
    e_G = e_G * f.abs()[:, None] + 2.0 ** -38 * unit
    low = 2.0 ** -38 if operand is BF16 else 0.0
    G = G * f[:, None]
    if dx is not None:
        want = torch.zeros(x.shape, dtype=F64, device="cuda")
        bound = torch.zeros_like(want)
        want[kept] = G @ w64
        bound[kept] = (e_G + (w.shape[0] + 8) * U * G.abs()) @ w64.abs() + low * w64.abs().max() * G.abs().sum(1, keepdim=True)
        assert (dx[~kept] == 0).all()
        assert_within(dx, want, bound * 1.01 + rounding(want, x.dtype), "dx")
    if dw is not None:
        want = G.T @ x64
        bound = (e_G + (len(at) + 8) * U * G.abs()).T @ x64.abs()
        if len(at):
            bound += low * x64.abs().max() * G.abs().sum(0)[:, None]
        assert_within(dw, want, bound * 1.01 + rounding(want, w.dtype), "dw")


def xent_run(x, w, t, reduction, dloss=None, need=(True, True), **kw):
    x, w = x.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
    loss = sa.linear_cross_entropy(x, w, t, reduction=reduction, **kw)
    if dloss is None:
        dloss = torch.ones_like(loss)
    leaves = [a for a, n in zip((x, w), need) if n]
    grads = iter(torch.autograd.grad(loss, leaves, dloss))
    return loss.detach(), dloss, *(next(grads) if n else None for n in need)


XENTS = [(1, 1, 1), (1, 300, 64), (2, 127, 17), (31, 129, 64), (33, 1000, 100), (128, 128, 128), (129, 257, 320), (300, 5003, 96),
         (1000, 2049, 64), (257, 8192, 768), (2111, 3001, 1024), (5003, 700, 40)]


@pytest.mark.parametrize("n,vocab,width", XENTS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("reduction", ["mean", "none", "sum"])
def test_linear_cross_entropy(cuda, n, vocab, width, dtype, reduction):
    g = torch.Generator(device="cuda").manual_seed(n + vocab)
    x, w, t = xent_inputs(g, n, vocab, width, dtype, dtype, ignored=0.3 if n % 2 else 0.0)
    t[0] = vocab - 1
    dloss = randn(g, n) if reduction == "none" else torch.tensor(1.0 if reduction == "mean" else -0.5, device="cuda")
    loss, _, dx, dw = xent_run(x, w, t, reduction, dloss)
    assert loss.dtype is F32 and dx.dtype is dtype and dw.dtype is dtype
    xent_check(x, w, t, reduction, dtype, loss, dloss, dx, dw)
    scored = sa.linear_cross_entropy(x, w, t, reduction=reduction)   # no gradient: smaller kernels, rows in place
    xent_check(x, w, t, reduction, dtype, scored)


@pytest.mark.parametrize("n,vocab,width,train", [(4100, 16400, 128, True), (2300, 50257, 64, True), (16384, 9000, 64, True),
                                                 (5000, 33000, 320, False), (1, 50304, 768, False), (200, 50304, 768, False)])
def test_linear_cross_entropy_large(cuda, n, vocab, width, train):
    """The larger tiles, several pieces of the vocabulary, split contractions, one token over a whole vocabulary."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x, w, t = xent_inputs(g, n, vocab, width, BF16, BF16, ignored=0.2 if n > 1 else 0.0)
    if not train:
        xent_check(x, w, t, "none", BF16, sa.linear_cross_entropy(x, w, t, reduction="none"))
        return
    loss, dloss, dx, dw = xent_run(x, w, t, "mean")
    xent_check(x, w, t, "mean", BF16, loss, dloss, dx, dw)
    again = xent_run(x, w, t, "mean")
    assert torch.equal(loss, again[0]) and torch.equal(dx, again[2]) and torch.equal(dw, again[3])


@pytest.mark.parametrize("xt,wt,precision,operand", [(BF16, F32, None, BF16), (F32, F32, "bf16", BF16), (F16, F32, None, F16),
                                                     (BF16, BF16, "ieee", F32), (F32, BF16, None, F32), (F16, F16, "tf32", F32)])
def test_linear_cross_entropy_types(cuda, xt, wt, precision, operand):
    g = torch.Generator(device="cuda").manual_seed(11)
    x, w, t = xent_inputs(g, 70, 333, 72, xt, wt, ignored=0.2)
    loss, dloss, dx, dw = xent_run(x, w, t, "mean", dot_precision=precision)
    assert dx.dtype is xt and dw.dtype is wt
    xent_check(x, w, t, "mean", operand, loss, dloss, dx, dw)


def test_linear_cross_entropy_views(cuda):
    """Slices read in place or copied, transposed weights, more dimensions, one gradient only, gradients that arrive as views."""
    g = torch.Generator(device="cuda").manual_seed(12)
    for xv, wv in ((randn(g, 40, 200)[:, 64:128], randn(g, 90, 192)[:, 128:]), (randn(g, 40, 65)[:, 1:], randn(g, 64, 90).T),
                   (randn(g, 80, 64)[::2], randn(g, 180, 64)[::2]), (randn(g, 64, 40).T, randn(g, 1, 64).expand(90, 64))):
        for dt in (F32, BF16):
            x, w = xv.to(dt) if dt is F32 else xv.bfloat16().as_strided(xv.shape, xv.bfloat16().stride()), wv.to(dt)
            t = torch.randint(90, (40,), device="cuda", generator=g)
            loss, dloss, dx, dw = xent_run(x, w, t, "mean")
            xent_check(x, w, t, "mean", dt, loss, dloss, dx, dw)
            xent_check(x, w, t, "none", dt, sa.linear_cross_entropy(x, w, t, reduction="none"))
    x, w, t = xent_inputs(g, 24, 90, 64, BF16, BF16)
    whole = xent_run(x, w, t, "none", randn(g, 48)[::2])
    xent_check(x, w, t, "none", BF16, whole[0], whole[1], whole[2], whole[3])
    for need in ((True, False), (False, True)):
        part = xent_run(x, w, t, "none", whole[1], need)
        assert torch.equal(part[0], whole[0])
        assert all(torch.equal(a, b) for a, b, n in zip(part[2:], whole[2:], need) if n)
    shaped = sa.linear_cross_entropy(x.reshape(2, 3, 4, 64), w, t.reshape(2, 3, 4), reduction="none")
    assert shaped.shape == (2, 3, 4) and torch.equal(shaped.flatten(), sa.linear_cross_entropy(x, w, t, reduction="none"))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=lambda t: str(t)[6:])
def test_linear_cross_entropy_ignored_rows(cuda, dtype):
    """What ignored tokens hold reaches nothing; every token ignored; other values to ignore."""
    g = torch.Generator(device="cuda").manual_seed(13)
    x, w, t = xent_inputs(g, 300, 500, 64, dtype, dtype, ignored=0.4)
    t[0] = -100
    clean = xent_run(x, w, t, "mean")
    xent_check(x, w, t, "mean", dtype, *clean)
    dirty = x.clone()
    dirty[t == -100] = math.nan
    dirty[0, :5] = math.inf
    for a, b in zip(xent_run(dirty, w, t, "mean"), clean):
        assert torch.equal(a, b)
    for n in (20, 300):   # rows in place, rows listed
        each = sa.linear_cross_entropy(dirty[:n], w, t[:n], reduction="none")
        xent_check(x[:n], w, t[:n], "none", dtype, each)
        assert (each[t[:n] == -100] == 0).all()
    other = torch.where(t == -100, 7, torch.where(t == 7, 8, t))
    loss, dloss, dx, dw = xent_run(x, w, other, "sum", ignore_index=7)
    xent_check(x, w, other, "sum", dtype, loss, dloss, dx, dw, ignore=7)
    none_kept = torch.full_like(t, -100)
    for reduction in ("mean", "sum", "none"):
        loss, _, dx, dw = xent_run(dirty, w, none_kept, reduction)
        assert loss.isnan().all() if reduction == "mean" else (loss == 0).all()
        assert (dx == 0).all() and (dw == 0).all()
    no_x, no_t = x[:0].clone().requires_grad_(), t[:0]
    for reduction in ("mean", "sum", "none"):
        loss = sa.linear_cross_entropy(no_x, w, no_t, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        assert loss.isnan() if reduction == "mean" else (loss == 0).all()


def test_linear_cross_entropy_edges(cuda):
    g = torch.Generator(device="cuda").manual_seed(14)
    x, w, t = xent_inputs(g, 40, 200, 64, BF16, BF16)
    # targets that are no word: NaN, loud, for their token or the mean
    bad = t.clone()
    bad[3], bad[5] = 200, -1
    each = sa.linear_cross_entropy(x, w, bad, reduction="none")
    real = (bad >= 0) & (bad < 200)
    assert each[~real].isnan().all() and torch.equal(each[real], sa.linear_cross_entropy(x, w, t, reduction="none")[real])
    assert sa.linear_cross_entropy(x, w, bad).isnan()
    _, _, dx, dw = xent_run(x, w, bad, "mean")
    assert dx[~real].isnan().all() and dw.isnan().all()
    # logits far apart: one word has all the weight, far above and far below the others
    far = (40.0 * randn(g, 200, 64)).bfloat16()
    loss, dloss, dx, dw = xent_run(x, far, t, "mean")
    assert loss.isfinite() and dx.isfinite().all() and dw.isfinite().all()
    want = torch.nn.functional.cross_entropy(x.double() @ far.double().T, t)
    assert abs(loss.double() - want) < 66 * U * (x.double().abs() @ far.double().abs().T).max() * 4
    # an infinity or a NaN in a kept row reaches its token and the whole of dW, as the formula has it
    ill = x.clone()
    ill[4, 0] = math.nan
    each, _, dx, dw = xent_run(ill, w, t, "none")
    sound = torch.arange(40, device="cuda") != 4
    assert each[4].isnan() and each[sound].isfinite().all() and dx[4].isnan().all() and dx[sound].isfinite().all() and dw.isnan().all()
    clean = xent_run(x, w, t, "none")
    ill[4, 0] = math.inf   # (the others' gradients are what they are without it)
    each, _, dx, dw = xent_run(ill, w, t, "none")
    assert not each[4].isfinite() and not dx[4].isfinite().any() and torch.equal(each[sound], clean[0][sound])
    assert torch.equal(dx[sound], clean[2][sound])
    # operands far from 1, of any size that bf16 has: the products' units come back out
    for xs, wscale in ((2.0 ** 60, 2.0 ** -60), (2.0 ** -100, 2.0 ** 95), (2.0 ** -20, 2.0 ** -110), (2.0 ** 30, 0.0)):
        xb, wb = x * xs, w * wscale
        loss, dloss, dx, dw = xent_run(xb, wb, t, "mean")
        xent_check(xb, wb, t, "mean", BF16, loss, dloss, dx, dw)
    # factors of very different sizes, zero among them
    dloss = torch.tensor([1e4, 1.0, 1e-3, 0.0], device="cuda").repeat(10)
    for dt in (BF16, F16, F32):
        loss, _, dx, dw = xent_run(x.to(dt), w.to(dt), t, "none", dloss)
        xent_check(x.to(dt), w.to(dt), t, "none", dt, loss, dloss, dx, dw)
        assert (dx[3::4] == 0).all()
    _, _, dx, dw = xent_run(x, w, t, "none", torch.zeros(40, device="cuda"))
    assert (dx == 0).all() and (dw == 0).all()


def test_linear_cross_entropy_difference(cuda):
    g = torch.Generator(device="cuda").manual_seed(15)
    x, w, t = xent_inputs(g, 48, 300, 40, F32, F32, ignored=0.2)
    loss, _, dx, dw = xent_run(x, w, t, "sum")
    step = 1e-2
    for a, d_a in ((0, dx), (1, dw)):
        d = randn(g, *d_a.shape)
        moved = [sa.linear_cross_entropy(*((x + s * step * d, w) if a == 0 else (x, w + s * step * d)), t, reduction="none").double().sum()
                 for s in (1, -1)]
        slope, want = (moved[0] - moved[1]) / (2 * step), (d_a.double() * d.double()).sum()
        # fp32 losses below 32 of 48 tokens over the step; the third derivative: logits move by up to |d| |w| ~ 20 step a token
        assert abs(slope - want) < 48 * 64 * 32 * U / step + 48 * (20 * step) ** 3 / step, a


# -- together -----------------------------------------------------------------------------------------------

def small_model(dtype=F32, **kw):
    torch.manual_seed(16)
    cfg = ModelConfig(**{**dict(vocab_size=1003, n_layers=2, d_model=128, n_heads=4, context_length=300), **kw})
    return SelectiveLM(cfg).cuda().to(dtype)


@pytest.mark.parametrize("kw", [{}, dict(bias=True), dict(attention="softmax")], ids=str)
def test_the_decoders_loss_is_forwards(cuda, kw):
    """SelectiveLM.loss against forward, fp32 throughout: both are within their own rounding of the same numbers. The two differ by sums of up to
    1003 products and of 600 tokens, 2 layers deep: 1e-4 of the largest gradient is 2^11 u, an order over what those give."""
    model = small_model(**kw)
    idx, targets = torch.randint(1003, (2, 300), device="cuda"), torch.randint(1003, (2, 300), device="cuda")
    targets[0, :50] = -100
    want = model(idx, targets)[1]
    grads = torch.autograd.grad(want, tuple(model.parameters()))
    got = model.loss(idx, targets)
    assert abs(got - want) < 1e-5 * want.abs()
    for (name, _), a, b in zip(model.named_parameters(), torch.autograd.grad(got, tuple(model.parameters())), grads):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max(), name
    each = model.loss(idx, targets, reduction="none")
    assert (each[0, :50] == 0).all() and abs(each.sum() / (targets != -100).sum() - want) < 1e-5 * want.abs()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=lambda t: str(t)[6:])
def test_the_decoders_loss_under_autocast(cuda, dtype):
    """Against the same model in float64 arithmetic of the plain forms (fp32 weights): the loss and every gradient as near as forward's own are,
    up to a factor of two: both round the same operands to the same type, at places of their own."""
    model = small_model()
    idx, targets = torch.randint(1003, (2, 300), device="cuda"), torch.randint(1003, (2, 300), device="cuda")
    exact = model(idx, targets)[1]   # fp32
    names = [n for n, _ in model.named_parameters()]
    true = torch.autograd.grad(exact, tuple(model.parameters()))
    with torch.autocast("cuda", dtype=dtype):
        runs = [f() for f in (lambda: model(idx, targets)[1], lambda: model.loss(idx, targets))]
    far = []
    for loss in runs:
        assert loss.dtype is F32 and abs(loss - exact) < 32 * half(dtype) * exact.abs()
        grads = torch.autograd.grad(loss, tuple(model.parameters()))
        assert all(d.dtype is F32 for d in grads)
        far.append([((a - b).norm() / b.norm()).item() for a, b in zip(grads, true)])
    for name, theirs, ours in zip(names, *far):
        assert ours <= 2 * theirs + 2 * half(dtype), (name, theirs, ours)


def test_a_step_captured_and_replayed(cuda):
    """A whole forward and backward pass of the operators as one graph, replayed on new inputs with eager work between; each replay
    equals the eager result."""
    g = torch.Generator(device="cuda").manual_seed(17)
    vocab, width, n = 1500, 128, 200
    table, w, gain = randn(g, vocab, width), randn(g, width), 0.1 * randn(g, n, width)
    ids, targets = (torch.randint(vocab, (n,), device="cuda", generator=g) for _ in range(2))

    def step(table, w, gain, ids, targets):
        table, w, gain = (t.detach().requires_grad_() for t in (table, w, gain))   # leaves of this step's own
        x = sa.embedding(ids, table, 2.0)
        y, s = sa.add_layer_norm(x, gain, w, dtype=BF16)
        y2, _ = sa.add_layer_norm(s, y, w, dtype=BF16)
        loss = sa.linear_cross_entropy(y2, table, targets)
        return (loss.detach(), *torch.autograd.grad(loss, (table, w, gain)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, w, gain, ids, targets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(table, w, gain, ids, targets)
    for k in range(3):
        ids.copy_(torch.randint(vocab, (n,), device="cuda", generator=g))
        targets.copy_(torch.randint(vocab, (n,), device="cuda", generator=g))
        targets[: 20 * k] = -100
        table.normal_(generator=g)
        want = step(table, w, gain, ids, targets)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_two_streams_at_once(cuda):
    """The same calls on two streams: nothing of one reaches the other."""
    g = torch.Generator(device="cuda").manual_seed(18)
    inputs = [xent_inputs(g, 700, 2000, 128, BF16, BF16, ignored=0.2) for _ in range(2)]
    ws = randn(g, 128)
    alone = [(xent_run(*i, "mean"), sa.layer_norm(i[0], ws)) for i in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append((xent_run(*i, "mean"), sa.layer_norm(i[0], ws)))
    torch.cuda.synchronize()
    for k, (run, y) in enumerate(got):
        want, wy = alone[k % 2]
        assert torch.equal(y, wy) and all(torch.equal(a, b) for a, b in zip(run, want))


def test_compiled_and_checked_as_custom_ops(cuda):
    """torch.compile traces the operators without a graph break, and the custom ops' schemas and fake kernels hold."""
    g = torch.Generator(device="cuda").manual_seed(19)
    table, w, b = randn(g, 90, 64).requires_grad_(), randn(g, 64).requires_grad_(), randn(g, 64).requires_grad_()
    ids, t = torch.randint(90, (2, 20), device="cuda"), torch.randint(90, (2, 20), device="cuda")

    def f(ids, t):
        x = sa.embedding(ids, table)
        y, s = sa.add_layer_norm(x, 0.5 * x, w, b)
        return sa.linear_cross_entropy(sa.layer_norm(y + s, w), table, t)

    want = f(ids, t)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(ids, t)
    torch.testing.assert_close(got, want, rtol=1e-6, atol=0)
    for a, c in zip(torch.autograd.grad(got, (table, w, b)), torch.autograd.grad(want, (table, w, b))):
        torch.testing.assert_close(a, c, rtol=1e-5, atol=1e-6)
    x, dx = randn(g, 6, 64), randn(g, 6, 64)
    stats = torch.ones(2, 6, device="cuda")
    check = lambda op, args: torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
    w, b, table = w.detach(), b.detach(), table.detach()
    check(lm._norm_op, (x, dx, w, b, 1e-5, 0, True))
    check(lm._norm_op, (x, None, w, None, 1e-5, 1, False))
    check(lm._norm_backward_op, (x, dx, None, w, stats, 0, True, True, False))
    check(lm._embedding_op, (ids, table, 1.0))
    check(lm._embedding_backward_op, (ids, randn(g, 2, 20, 64), 90, 1.0))
    check(lm._xent_op, (x, table, ids[0, :6], -100, 1, 1, True))
    _, lse, rows = lm._xent_impl(x, table, ids[0, :6], -100, 1, 1, True)
    check(lm._xent_backward_op, (x, table, ids[0, :6], lse, rows, torch.ones((), device="cuda"), 1, 1, True, False))


def test_refusals(cuda):
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(8, device="cuda")
    ids, t = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (
        lambda: sa.layer_norm(x, w[:7]), lambda: sa.layer_norm(x, w, w.bfloat16()), lambda: sa.layer_norm(x, w, w[:7]),
        lambda: sa.layer_norm(x, w.cpu()), lambda: sa.layer_norm(x.int(), w), lambda: sa.layer_norm(x, w, eps=-1.0),
        lambda: sa.layer_norm(x, w, eps=math.nan), lambda: sa.layer_norm(x, w, dtype=F64), lambda: sa.layer_norm(x[0, 0], w),
        lambda: sa.layer_norm(torch.empty(1, 32769, device="cuda"), torch.empty(32769, device="cuda")),
        lambda: sa.layer_norm(x[:, :0], w[:0]), lambda: sa.add_layer_norm(x, x[:2], w), lambda: sa.add_layer_norm(x, x.double(), w),
        lambda: sa.embedding(ids.float(), x), lambda: sa.embedding(ids.cpu(), x), lambda: sa.embedding(ids, w),
        lambda: sa.embedding(ids, x[:0]), lambda: sa.embedding(ids, x.double()),
        lambda: sa.embedding(ids[:1].expand(1 << 30), x),
        lambda: sa.linear_cross_entropy(x, x[:, :7], t), lambda: sa.linear_cross_entropy(x, x, t[:3]),
        lambda: sa.linear_cross_entropy(x, x, t.int()), lambda: sa.linear_cross_entropy(x, x, t, reduction="batch"),
        lambda: sa.linear_cross_entropy(x, x, t, dot_precision="fp8"), lambda: sa.linear_cross_entropy(x, x.cpu(), t),
        lambda: sa.linear_cross_entropy(x, x, t, ignore_index=0.5), lambda: sa.linear_cross_entropy(x[:, :0], x[:, :0], t),
        lambda: sa.linear_cross_entropy(x[0, 0], x, t),
    ):
        with pytest.raises(ValueError):
            call()
    # a second derivative, of gradients that depend on the leaf through what arrives or through what was saved
    leaf = x.clone().requires_grad_()
    for f in (lambda: sa.layer_norm(leaf, w).square().sum(), lambda: sa.layer_norm(leaf, w).sum(), lambda: sa.linear_cross_entropy(leaf, x, t),
              lambda: sa.embedding(t, leaf).square().sum()):
        d, = torch.autograd.grad(f(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum() + leaf.sum(), leaf)


# -- sizes past 32 bits ---------------------------------------------------------------------------------------

def test_layer_norm_past_32_bits(cuda):
    """Rows behind element 2^31 give what they give alone."""
    rows, width = (1 << 31) // 1024 + 70, 1024
    g = torch.Generator(device="cuda").manual_seed(21)
    x = torch.empty(rows, width, device="cuda", dtype=BF16).normal_(generator=g)
    branch, w = x.flip(0), (1 + 0.1 * randn(g, width)).bfloat16()
    leaves = [t.requires_grad_() for t in (x, branch, w)]
    y, s = sa.add_layer_norm(*leaves)
    dx, _, dw = torch.autograd.grad((y, s), leaves, (y.detach(), s.detach()))
    for part in (slice(rows - 90, rows), slice(0, 64)):
        few = [x.detach()[part].clone().requires_grad_(), branch.detach()[part].clone().requires_grad_(), w]
        y2, s2 = sa.add_layer_norm(*few)
        dx2, = torch.autograd.grad((y2, s2), few[0], (y2.detach(), s2.detach()))
        assert torch.equal(y[part], y2) and torch.equal(s[part], s2) and torch.equal(dx[part], dx2)
    # dw is a sum over 2^21 rows of about 1: within bf16's own rounding of fp32 sums of 4100 rows' sums each
    h = torch.zeros(width, dtype=F64, device="cuda")
    for a in range(0, rows, 1 << 18):
        part = s.detach()[a:a + (1 << 18)].double()
        c = part - part.mean(-1, keepdim=True)
        h += (y.detach()[a:a + (1 << 18)].double() * c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5)).sum(0)
    assert ((dw.double() - h).abs() <= 2 * half(BF16) * h.abs()).all()


def test_embedding_past_32_bits(cuda):
    vocab, width, tokens = (1 << 31) // 1024 + 3000, 1024, 5000
    g = torch.Generator(device="cuda").manual_seed(22)
    w = torch.empty(vocab, width, device="cuda", dtype=BF16).normal_(generator=g).requires_grad_()
    ids = vocab - 1 - torch.randint(4000, (tokens,), device="cuda", generator=g)
    dy = randn(g, tokens, width).bfloat16()
    y = sa.embedding(ids, w)
    assert torch.equal(y, w.detach()[ids])
    dw, = torch.autograd.grad(y, w, dy)
    first = vocab - 4000
    embed_check(ids - first, w.detach()[first:], 1.0, None, dy, dw[first:])
    assert (dw[:first] == 0).all()


@pytest.mark.parametrize("pull", [20.0, 3.0])
def test_linear_cross_entropy_past_32_bits(cuda, pull):
    """A weight of more than 2^31 elements; the words behind that are found, and get their gradient. Targets of weight 1 (pull 20) and of
    about a hundredth.

    Bounds as in xent_check: G = (p - onehot) / n is off by half a step of it, and by p (2 dl + dlse) / n whatever remains of p - 1."""
    n, width = 40, 8192
    vocab = (1 << 31) // width + 900
    g = torch.Generator(device="cuda").manual_seed(23)
    w = torch.empty(vocab, width, device="cuda", dtype=BF16).normal_(std=0.02, generator=g)
    t = vocab - 1 - torch.randint(800, (n,), device="cuda", generator=g)
    t[:8] = torch.arange(8, device="cuda")
    x = (randn(g, n, width) + pull * w[t].float()).bfloat16()
    loss, dloss, dx, dw = xent_run(x, w, t, "mean")
    parts = [slice(a, a + 16384) for a in range(0, vocab, 16384)]
    x64 = x.double()
    l = torch.cat([x64 @ w[p].double().T for p in parts], 1)
    dl = (width + 2) * U * torch.stack([(x64.abs() @ w[p].double().abs().T).amax(1) for p in parts]).amax(0)
    lse = torch.logsumexp(l, 1)
    e_lse = dl + U * (160 + vocab / 1024) + 2.0 ** -22 * (4 + lse.abs())
    at = torch.arange(n, device="cuda")
    each = lse - l[at, t]
    assert abs(loss.double() - each.mean()) <= (dl + e_lse + 5 * U * (lse.abs() + each)).mean()
    e_G = torch.exp(l - lse[:, None])   # p
    G = e_G.clone()
    G[at, t] -= 1.0
    e_G *= (2 * dl + e_lse)[:, None] * 1.01 + 3 * U
    e_G += (half(F16) + (vocab + 8) * U) * G.abs() + 2.0 ** -38
    e_G /= n
    G /= n
    for p in (slice(vocab - 900, vocab), slice(0, 300)):
        want = G[:, p].T @ x64
        bound = e_G[:, p].T @ x64.abs() + 2.0 ** -38 * x64.abs().max() * G[:, p].abs().sum(0)[:, None]
        assert_within(dw[p], want, bound * 1.01 + rounding(want, BF16), "dw")
    want, bound = (torch.zeros(n, width, device="cuda", dtype=F64) for _ in range(2))
    for p in parts:
        want += G[:, p] @ w[p].double()
        bound += e_G[:, p] @ w[p].double().abs()
    assert_within(dx, want, bound * 1.01 + 2.0 ** -38 * G.abs().sum(1, keepdim=True) + rounding(want, BF16), "dx")
