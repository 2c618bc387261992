"""The operators around the attention layers without a GPU: their plain forms against torch's own functions, the decoder's
fused loss against its forward pass, the refusals, and the C ABI's argument checks."""

import math

import pytest
import torch
import torch.nn.functional as F

import selective_attention as sa
from selective_attention import _lib
from selective_attention.model import ModelConfig, SelectiveLM

F64 = torch.float64


def test_layer_norm_reference_is_the_layer_norm():
    g = torch.Generator().manual_seed(0)
    x, b, w, c = (torch.randn(*s, dtype=F64, generator=g) for s in ((3, 5, 33), (3, 5, 33), (33,), (33,)))
    torch.testing.assert_close(sa.layer_norm_reference(x, w, c), F.layer_norm(x, (33,), w, c), rtol=1e-12, atol=1e-12)
    y, s = sa.add_layer_norm_reference(x, b, w, c, 1e-3)
    assert torch.equal(s, x + b)
    torch.testing.assert_close(y, F.layer_norm(x + b, (33,), w, c, 1e-3), rtol=1e-12, atol=1e-12)


def test_embedding_reference_is_the_embedding():
    g = torch.Generator().manual_seed(1)
    w, ids = torch.randn(11, 7, dtype=F64, generator=g), torch.tensor([[0, 10, 3], [3, -1, 11]])
    y = sa.embedding_reference(ids, w, 2.0)
    assert torch.equal(y[0], 2.0 * F.embedding(ids[0], w)) and torch.equal(y[1, 0], 2.0 * w[3])
    assert y[1, 1:].isnan().all()


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_linear_cross_entropy_reference_is_the_cross_entropy(reduction):
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(4, 9, 17, dtype=F64, generator=g), torch.randn(23, 17, dtype=F64, generator=g)
    t = torch.randint(23, (4, 9), generator=g)
    t[:, 2] = -100
    want = F.cross_entropy((x @ w.T).flatten(0, 1), t.flatten(), reduction=reduction)
    got = sa.linear_cross_entropy_reference(x, w, t, reduction=reduction)
    torch.testing.assert_close(got.flatten() if reduction == "none" else got, want, rtol=1e-12, atol=1e-12)


def test_linear_cross_entropy_reference_edges():
    x, w = torch.randn(3, 4, requires_grad=True), torch.randn(5, 4, requires_grad=True)
    with torch.no_grad():
        x[1] = math.nan
    t = torch.tensor([1, -100, 5])
    each = sa.linear_cross_entropy_reference(x, w, t, reduction="none")
    assert each[0].isfinite() and each[1] == 0 and each[2].isnan()
    loss = sa.linear_cross_entropy_reference(x, w, torch.tensor([1, -100, 0]))
    loss.backward()
    assert loss.isfinite() and x.grad.isfinite().all() and (x.grad[1] == 0).all() and w.grad.isfinite().all()
    assert sa.linear_cross_entropy_reference(x, w, torch.full((3,), -100)).isnan()


@pytest.mark.parametrize("kw", [{}, dict(bias=True), dict(n_layers=0), dict(attention="softmax")], ids=str)
def test_loss_is_forwards_loss(kw):
    torch.manual_seed(3)
    cfg = ModelConfig(**{**dict(vocab_size=61, n_layers=2, d_model=32, n_heads=2, context_length=40), **kw})
    model = SelectiveLM(cfg)
    idx, targets = torch.randint(61, (2, 24)), torch.randint(61, (2, 24))
    targets[0, :5] = -100
    want = model(idx, targets)[1]
    grads = torch.autograd.grad(want, tuple(model.parameters()))
    got = model.loss(idx, targets)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    for n, a, b in zip(dict(model.named_parameters()), torch.autograd.grad(got, tuple(model.parameters())), grads):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6, msg=n)
    each = model.loss(idx, targets, reduction="none")
    assert each.shape == idx.shape and (each[0, :5] == 0).all()
    torch.testing.assert_close(each.sum() / (targets != -100).sum(), want, rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError, match="context_length"):
        model.loss(torch.zeros(1, 41, dtype=torch.int64), torch.zeros(1, 41, dtype=torch.int64))


def test_tensors_off_the_gpu_are_refused():
    x, w, t = torch.randn(2, 4), torch.randn(4), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: sa.layer_norm(x, w), lambda: sa.add_layer_norm(x, x, w), lambda: sa.embedding(t, x),
                 lambda: sa.linear_cross_entropy(x, x, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="float"):
        sa.layer_norm(x.double(), w)


# -- the C ABI: every refusal comes before a pointer is read ---------------------------------------------

A = 1 << 20   # an aligned address that nothing reads


def _refused(fn, args, changes, status):
    for i, value in changes:
        bad = list(args)
        bad[i] = value
        assert fn(*bad) == status, (i, value)


def test_layer_norm_abi_refuses():
    lib = _lib.load()
    args = [A, 64, A, 64, A, A, A, A, A, A, 10, 64, 1e-5, 0, 1, 2, 0, None]
    _refused(lib.sa_layer_norm, args, [(13, 9), (14, -1), (15, 3), (16, 7)], -3)
    _refused(lib.sa_layer_norm, args, [(0, None), (4, None), (6, None), (7, None), (8, None), (9, None), (1, -1), (3, -1), (10, -1),
                                       (11, 0), (11, 32769), (12, -1.0), (12, math.nan), (12, math.inf), (0, A + 1), (2, A + 2),
                                       (4, A + 1)], -1)
    assert lib.sa_layer_norm(None, 0, None, 0, None, None, None, None, None, None, 0, 64, 1e-5, 0, 0, 0, 0, None) == 0   # no rows
    assert lib.sa_layer_norm_backward_workspace_bytes(10, 0) == -1
    size = lib.sa_layer_norm_backward_workspace_bytes(10, 64)
    assert size > 0
    args = [A, 64, A, 64, A, 64, A, A, A, A, A, A, A, A, size, 10, 64, 0, 1, 2, 0, None]
    _refused(lib.sa_layer_norm_backward, args, [(17, 9), (18, 9), (19, 9), (20, 9)], -3)
    _refused(lib.sa_layer_norm_backward, args, [(0, None), (2, None), (6, None), (7, None), (8, None), (9, A + 1), (10, A + 2), (16, 0)], -1)
    _refused(lib.sa_layer_norm_backward, args, [(13, None), (13, A + 8), (14, size - 1)], -4)


def test_embedding_abi_refuses():
    lib = _lib.load()
    args = [A, 8, A, 64, A, 10, 100, 64, 1.0, 0, None]
    _refused(lib.sa_embedding, args, [(9, 5)], -3)
    _refused(lib.sa_embedding, args, [(0, None), (1, 2), (0, A + 4), (2, None), (2, A + 1), (3, -1), (4, None), (5, -1), (5, 1 << 30),
                                      (6, 0), (6, 1 << 28), (7, 0), (7, 1 << 24)], -1)
    assert lib.sa_embedding_backward_workspace_bytes(1, 0, 1) == -1
    size = lib.sa_embedding_backward_workspace_bytes(10, 100, 64)
    args = [A, 8, A, 64, A, A, size, 10, 100, 64, 1.0, 0, None]
    _refused(lib.sa_embedding_backward, args, [(11, 5)], -3)
    _refused(lib.sa_embedding_backward, args, [(0, None), (1, 2), (2, None), (4, None), (3, -1), (7, 1 << 30), (8, 0)], -1)
    _refused(lib.sa_embedding_backward, args, [(5, None), (5, A + 8), (6, size - 1)], -4)
    # more pieces of work than a launch holds threads for
    big = lib.sa_embedding_backward_workspace_bytes(1 << 29, 100, 256)
    assert lib.sa_embedding_backward(A, 8, A, 256, A, A, big, 1 << 29, 100, 256, 1.0, 0, None) == -1


def test_linear_xent_abi_refuses():
    lib = _lib.load()
    size = lib.sa_linear_xent_workspace_bytes(A, 64, A, 64, 10, 100, 64, 1, 1, 0, 0, 0)
    assert size > 0
    assert lib.sa_linear_xent_workspace_bytes(A, 64, A, 64, 0, 100, 64, 1, 1, 0, 0, 0) == -1
    assert lib.sa_linear_xent_workspace_bytes(A, 64, A, 64, 10, 100, 64, 1, 1, 0, 0, 4) == -1
    args = [A, 64, A, 64, A, A, A, A, A, size, 10, 100, 64, -100, 1, 0, 0, 0, None]
    _refused(lib.sa_linear_xent, args, [(15, 4), (16, 4), (17, 4)], -3)
    _refused(lib.sa_linear_xent, args, [(0, None), (2, None), (4, None), (5, None), (7, None), (0, A + 1), (4, A + 4), (1, -1), (10, 0),
                                        (10, 1 << 28), (11, 0), (11, 1 << 28), (12, 0), (12, 65537), (14, 3), (14, -1)], -1)
    _refused(lib.sa_linear_xent, args, [(8, None), (8, A + 8), (9, size - 1)], -4)
    size = lib.sa_linear_xent_backward_workspace_bytes(A, 64, 10, 100, 64, 1, 1, 0, 0)
    args = [A, 64, A, 64, A, A, A, A, A, A, A, size, 10, 100, 64, 1, 0, 0, 0, None]
    _refused(lib.sa_linear_xent_backward, args, [(16, 4), (17, 4), (18, 4)], -3)
    _refused(lib.sa_linear_xent_backward, args, [(0, None), (2, None), (4, None), (5, None), (6, None), (7, None), (8, A + 8), (9, A + 4),
                                                 (12, 0), (13, 0), (14, 0), (15, 5)], -1)
    _refused(lib.sa_linear_xent_backward, args, [(10, None), (11, size - 1)], -4)
    bad = list(args)
    bad[8] = bad[9] = None
    assert lib.sa_linear_xent_backward(*bad) == 0   # nothing asked for
    # tiles past what one launch holds
    assert lib.sa_linear_xent_workspace_bytes(A, 64, A, 64, 1 << 21, 1 << 20, 64, 1, 1, 0, 0, 0) == -1
