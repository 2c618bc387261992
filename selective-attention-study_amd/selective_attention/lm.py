"""The operators of a decoder around its attention layers, with their gradients: the token embedding, the layer norms with
the residual addition before them, and the softmax cross entropy of the output head (no reference counterpart: the reference
runs them through torch, model.py:342-418).

    y = embedding(ids, weight)                               # (..., C) rows of the table
    y, x = add_layer_norm(x, branch, weight, dtype=...)      # x + branch, and its norm in the next product's type
    loss = linear_cross_entropy(y, weight, targets)          # the logits y @ weight.T are never in memory

SelectiveLM.loss runs a training step's forward pass through them. Tensors are float16, bfloat16 or float32, each of a type of
its own where the docstring does not tie them together; arithmetic, statistics and sums are fp32 and every result is rounded once. Equal calls give
equal bits. The calls allocate from torch's caching allocator and launch on the current stream of their tensors' device, so
they can be captured into a graph, backward passes too. (As with any operator, capture a backward pass on leaves that no
eager graph still holds: torch accumulates into a leaf on the stream that first used it, and a capture cannot wait for another stream.)
Each has a gradient; second derivatives, forward-mode ones and torch.func's transforms raise.

The `_reference` functions are the same in plain torch, on any device.
"""

import math
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad
from torch import Tensor

from . import _lib
from .kernels import DTYPES, _custom_op, _plain, _resolve_precision
from .paged import _call

_CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}
_TYPES = {code: dtype for dtype, code in _CODES.items()}
MAX_WIDTH = 32768   # of a normed row
MAX_HEAD_WIDTH = 1 << 16   # of the head's rows


# -- checks ---------------------------------------------------------------------------------------------

def _check_float(name: str, t: Tensor, device: torch.device | None = None) -> None:
    if t.dtype not in DTYPES:
        raise ValueError(f"{name}'s dtype must be float16, bfloat16 or float32; got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (ROCm) tensor; the _reference functions run anywhere")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}; got {t.device}")


def _rows(x: Tensor, width: int) -> tuple[Tensor, int]:
    """(x, elements from a row to the next) of a tensor of (..., width) rows that the kernels can read: contiguous rows a fixed
    stride apart are read in place, anything else (a view that is negated when read, too) becomes contiguous first."""
    if x.is_neg():
        x = x.resolve_neg()
    if x.is_contiguous():
        return x, width
    flat = x.reshape(-1, width)
    row, unit = flat.stride()
    if (unit == 1 or width == 1) and 0 <= row < 1 << 31:
        return flat, row
    return flat.contiguous(), width


def _vector(x: Tensor) -> Tensor:
    return x.contiguous().resolve_neg()


def _wants_grad(*tensors: Tensor | None) -> bool:
    """Whether the call goes through its autograd function: one of the tensors wants a gradient, or may have a forward-mode tangent, which
    the function refuses and the op would drop."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or forward_ad._current_level >= 0


def _ptr(t: Tensor | None):
    return None if t is None else t.data_ptr()


# (A short step's host work is of the size of its kernels', half of it on autograd's own thread: the implementations below allocate
# what they return and nothing else, None in the place of what is not asked for, and read each attribute once. The custom ops, which
# can return tensors only, put empty ones there.)

def _empty(like: Tensor, dtype: torch.dtype) -> Tensor:
    """A contiguous tensor of like's shape and device."""
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _filled(*results: Tensor | None, like: Tensor) -> tuple[Tensor, ...]:
    return tuple(like.new_empty(0) if r is None else r for r in results)


def _mode_plain(plain: bool, *tensors: Tensor | None) -> bool:
    """_plain in a backward pass, of the gradients that arrive: what was saved was looked at in the forward pass. Where a second
    derivative may follow (create_graph) it is the op that runs, which raises then."""
    return plain and not torch.is_grad_enabled() and _plain(*[t for t in tensors if t is not None])


def _sized(device: torch.device, query, *args) -> int:
    """A workspace size that depends on the device's compute units."""
    if device.index == torch._C._cuda_getDevice():
        return query(*args)
    with torch.cuda.device(device):
        return query(*args)


# -- layer norm -------------------------------------------------------------------------------------------

def _norm_impl(x: Tensor, branch: Optional[Tensor], weight: Tensor, bias: Optional[Tensor], eps: float, dtype: int, stats: bool):
    """sa_layer_norm: y, the sum (None without a branch), and the rows' mean and rstd (2, rows), None without `stats`."""
    width, device, code = weight.shape[0], x.device, _CODES[x.dtype]
    rows = x.numel() // width
    y = _empty(x, _TYPES[dtype])
    total = None if branch is None else _empty(x, x.dtype)
    held = torch.empty(2, rows, device=device, dtype=torch.float32) if stats else None
    if rows == 0:
        return y, total, held
    x, x_ld = _rows(x, width)
    branch_ld = branch_code = 0
    if branch is not None:
        branch, branch_ld = _rows(branch, width)
        branch_code = _CODES[branch.dtype]
    weight = _vector(weight)
    if bias is not None:
        bias = _vector(bias)
    mean = None if held is None else held.data_ptr()
    _call(device, _lib.load().sa_layer_norm, x.data_ptr(), x_ld, _ptr(branch), branch_ld, weight.data_ptr(), _ptr(bias),
          y.data_ptr(), _ptr(total), mean, None if mean is None else mean + 4 * rows, rows, width, eps, code, branch_code, dtype,
          _CODES[weight.dtype])
    return y, total, held


def _norm_dense(x: Tensor, branch: Optional[Tensor], weight: Tensor, bias: Optional[Tensor], eps: float, dtype: int,
                stats: bool) -> tuple[Tensor, Tensor, Tensor]:
    y, total, held = _norm_impl(x, branch, weight, bias, eps, dtype, stats)
    return (y, *_filled(total, like=x), *_filled(held, like=x.new_empty(0, dtype=torch.float32)))


_norm_op = _custom_op("layer_norm_forward", _norm_dense)


@_norm_op.register_fake
def _norm_fake(x, branch, weight, bias, eps, dtype, stats):
    return (x.new_empty(x.shape, dtype=_TYPES[dtype]), x.new_empty(x.shape if branch is not None else (0,)),
            x.new_empty((2, x.numel() // weight.shape[0]) if stats else (0,), dtype=torch.float32))


def _norm_backward_impl(s: Tensor, dy: Tensor, ds: Optional[Tensor], weight: Tensor, stats: Tensor, branch_dtype: int,
                        need_x: bool, need_weight: bool, need_bias: bool):
    """sa_layer_norm_backward: dx, the branch's gradient (None where it is of dx's type, whose values it has: branch_dtype is then -1),
    dweight and dbias (None where not needed)."""
    width, device, code = weight.shape[0], s.device, _CODES[s.dtype]
    rows = s.numel() // width
    lib = _lib.load()
    dx = _empty(s, s.dtype) if need_x else None
    dbranch = _empty(s, _TYPES[branch_dtype]) if branch_dtype >= 0 else None
    weight = _vector(weight)
    dweight = torch.empty_like(weight) if need_weight else None
    dbias = torch.empty_like(weight) if need_bias else None
    s, s_ld = _rows(s, width)
    dy, dy_ld = _rows(dy, width)
    ds_ld = size = 0
    if ds is not None:
        ds, ds_ld = _rows(ds, width)
    ws = None
    if need_weight or need_bias:
        size = lib.sa_layer_norm_backward_workspace_bytes(rows, width)
        ws = torch.empty(size, device=device, dtype=torch.uint8)
    mean = stats.data_ptr()
    _call(device, lib.sa_layer_norm_backward, s.data_ptr(), s_ld, dy.data_ptr(), dy_ld, _ptr(ds), ds_ld, weight.data_ptr(), mean,
          mean + 4 * rows, _ptr(dx), _ptr(dbranch), _ptr(dweight), _ptr(dbias), _ptr(ws), size, rows, width, code, max(branch_dtype, 0),
          _CODES[dy.dtype], _CODES[weight.dtype])
    return dx, dbranch, dweight, dbias


def _norm_backward_dense(s: Tensor, dy: Tensor, ds: Optional[Tensor], weight: Tensor, stats: Tensor, branch_dtype: int,
                         need_x: bool, need_weight: bool, need_bias: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dx, dbranch, dweight, dbias = _norm_backward_impl(s, dy, ds, weight, stats, branch_dtype, need_x, need_weight, need_bias)
    other = s if branch_dtype < 0 else s.new_empty(0, dtype=_TYPES[branch_dtype])
    return (*_filled(dx, like=s), *_filled(dbranch, like=other), *_filled(dweight, dbias, like=weight))


_norm_backward_op = _custom_op("layer_norm_backward", _norm_backward_dense)


@_norm_backward_op.register_fake
def _norm_backward_fake(s, dy, ds, weight, stats, branch_dtype, need_x, need_weight, need_bias):
    other = branch_dtype >= 0
    return (s.new_empty(s.shape if need_x else (0,)),
            s.new_empty(s.shape if other else (0,), dtype=_TYPES[branch_dtype] if other else s.dtype),
            weight.new_empty((weight.shape[0] if need_weight else 0,)), weight.new_empty((weight.shape[0] if need_bias else 0,)))


class _LayerNormFn(torch.autograd.Function):
    """y, and with a branch the sum. The backward pass takes the sum (or x) and the rows' statistics."""

    @staticmethod
    def forward(ctx, x, branch, weight, bias, eps, dtype):
        ctx.plain = plain = _plain(*[t for t in (x, branch, weight, bias) if t is not None])
        y, total, stats = (_norm_impl if plain else _norm_op)(x, branch, weight, bias, eps, _CODES[dtype], True)
        ctx.set_materialize_grads(False)
        if branch is None:
            ctx.save_for_backward(x, weight, stats)
            ctx.branch_dtype = None
            return y
        ctx.save_for_backward(total, weight, stats)
        ctx.branch_dtype = branch.dtype
        return y, total

    @staticmethod
    def backward(ctx, dy, ds=None):
        s, weight, stats = ctx.saved_tensors
        need_x, need_branch, need_weight, need_bias, _, _ = ctx.needs_input_grad
        if dy is None:   # (only the sum was used)
            if ds is None:
                return (None,) * 6
            dy = torch.zeros_like(s)
        other = need_branch and ctx.branch_dtype != s.dtype
        plain = _mode_plain(ctx.plain, dy, ds)
        dx, dbranch, dweight, dbias = (_norm_backward_impl if plain else _norm_backward_op)(
            s, dy, ds, weight, stats, _CODES[ctx.branch_dtype] if other else -1, need_x or (need_branch and not other), need_weight,
            need_bias)
        return (dx if need_x else None, (dbranch if other else dx) if need_branch else None, dweight if need_weight else None,
                dbias if need_bias else None, None, None)


def _check_norm(x: Tensor, branch: Tensor | None, weight: Tensor, bias: Tensor | None, eps: float,
                dtype: torch.dtype | None) -> tuple[float, torch.dtype]:
    _check_float("x", x)
    width = x.shape[-1] if x.dim() else 0
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"x must be (..., C) with C from 1 to {MAX_WIDTH}; got {tuple(x.shape)}")
    if branch is not None:
        _check_float("branch", branch, x.device)
        if branch.shape != x.shape:
            raise ValueError(f"branch must have x's shape {tuple(x.shape)}; got {tuple(branch.shape)}")
    _check_float("weight", weight, x.device)
    if weight.shape != (width,):
        raise ValueError(f"weight must be ({width},); got {tuple(weight.shape)}")
    if bias is not None and (bias.shape != (width,) or bias.dtype is not weight.dtype or bias.device != x.device):
        raise ValueError(f"bias must be ({width},) of weight's dtype {weight.dtype} on {x.device}; got {bias.dtype} "
                         f"{tuple(bias.shape)} on {bias.device}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be a finite number >= 0; got {eps}")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be float16, bfloat16 or float32; got {dtype}")
    return float(eps), dtype


def _norm(x, branch, weight, bias, eps, dtype):
    eps, dtype = _check_norm(x, branch, weight, bias, eps, dtype)
    if _wants_grad(x, branch, weight, bias):
        return _LayerNormFn.apply(x, branch, weight, bias, eps, dtype)
    plain = _plain(*[t for t in (x, branch, weight, bias) if t is not None])
    y, total, _ = (_norm_impl if plain else _norm_op)(x, branch, weight, bias, eps, _CODES[dtype], False)
    return y if branch is None else (y, total)


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5, dtype: torch.dtype | None = None) -> Tensor:
    """weight (x - mean) / sqrt(var + eps) + bias over the last dimension of x (..., C), C up to 32768, in `dtype` (x's by default). weight
    and bias: (C,), of one type. Statistics are fp32, taken in two passes over the row."""

    return _norm(x, None, weight, bias, eps, dtype)


def add_layer_norm(x: Tensor, branch: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5,
                   dtype: torch.dtype | None = None) -> tuple[Tensor, Tensor]:
    """A pre-norm block's residual addition and the norm after it, in one pass: (layer_norm(s), s) for s = x + branch in x's type. The
    norm is that of s as it is returned (rounded, where x is a 16-bit stream), as with the two written one after the other.

    x and branch: (..., C), each of its own type (a fp32 stream and a bf16 branch, under autocast); otherwise as layer_norm."""

    return _norm(x, branch, weight, bias, eps, dtype)


# -- embedding --------------------------------------------------------------------------------------------

def _embedding_impl(ids: Tensor, weight: Tensor, scale: float) -> Tensor:
    """sa_embedding: (*ids.shape, C)."""
    vocab, width = weight.shape
    out = weight.new_empty((*ids.shape, width))
    tokens = ids.numel()
    if tokens == 0:
        return out
    ids = ids.contiguous()
    weight, ld = _rows(weight, width)
    _call(weight.device, _lib.load().sa_embedding, ids.data_ptr(), ids.element_size(), weight.data_ptr(), ld, out.data_ptr(), tokens,
          vocab, width, scale, _CODES[weight.dtype])
    return out


_embedding_op = _custom_op("embedding_forward", _embedding_impl)


@_embedding_op.register_fake
def _embedding_fake(ids, weight, scale):
    return weight.new_empty((*ids.shape, weight.shape[1]))


def _embedding_backward_impl(ids: Tensor, dout: Tensor, vocab: int, scale: float) -> Tensor:
    """sa_embedding_backward: (vocab, C) in dout's dtype."""
    width, tokens = dout.shape[-1], ids.numel()
    lib = _lib.load()
    dweight = dout.new_empty((vocab, width))
    ids = ids.contiguous()
    dout, ld = _rows(dout, width)
    size = lib.sa_embedding_backward_workspace_bytes(tokens, vocab, width)
    ws = torch.empty(size, device=dout.device, dtype=torch.uint8)
    _call(dout.device, lib.sa_embedding_backward, ids.data_ptr(), ids.element_size(), dout.data_ptr(), ld, dweight.data_ptr(), ws.data_ptr(),
          size, tokens, vocab, width, scale, _CODES[dout.dtype])
    return dweight


_embedding_backward_op = _custom_op("embedding_backward", _embedding_backward_impl)


@_embedding_backward_op.register_fake
def _embedding_backward_fake(ids, dout, vocab, scale):
    return dout.new_empty((vocab, dout.shape[-1]))


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = weight.shape[0], scale
        ctx.plain = plain = _plain(ids, weight)
        return (_embedding_impl if plain else _embedding_op)(ids, weight, scale)

    @staticmethod
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        backward = _embedding_backward_impl if _mode_plain(ctx.plain, dout) else _embedding_backward_op
        return None, backward(ids, dout, ctx.vocab, ctx.scale), None


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """scale * weight[ids]: ids of any shape (int32 or int64), weight (V, C); (*ids.shape, C) in weight's dtype.

    Nothing on the host looks at the ids: one outside [0, V) gives a row of NaN and no gradient. The gradient, (V, C) in weight's dtype, sums
    each id's tokens in their order (fp32), whatever else the batch holds."""

    _check_float("weight", weight)
    if ids.dtype not in (torch.int32, torch.int64) or ids.device != weight.device:
        raise ValueError(f"ids must be int32 or int64 on {weight.device}; got {ids.dtype} on {ids.device}")
    if weight.dim() != 2 or not 1 <= weight.shape[0] < 1 << 28 or not 1 <= weight.shape[1] < 1 << 24:
        raise ValueError(f"weight must be (V, C) with V from 1 to 2^28 - 1 and C from 1 to 2^24 - 1; got {tuple(weight.shape)}")
    if ids.numel() >= 1 << 30 or -(-ids.numel() // 32) * -(-weight.shape[1] // 256) >= 1 << 23:
        raise ValueError(f"{ids.numel()} tokens of {weight.shape[1]} columns are too many for one call")
    scale = float(scale)
    if _wants_grad(weight):
        return _EmbeddingFn.apply(ids, weight, scale)
    return (_embedding_impl if _plain(ids, weight) else _embedding_op)(ids, weight, scale)


# -- the vocabulary loss ------------------------------------------------------------------------------------

def _xent_impl(x: Tensor, weight: Tensor, targets: Tensor, ignore: int, reduction: int, code: int, train: bool):
    """sa_linear_xent on x (N, C): the loss, and for the backward pass (`train`; else None) the kept tokens'
    largest logits and reciprocal sums (2, N), and which those are."""
    tokens, width = x.shape
    vocab, device = weight.shape[0], x.device
    lib = _lib.load()
    x, x_ld = _rows(x, width)
    weight, w_ld = _rows(weight, width)
    targets = targets.contiguous()
    none = reduction == _lib.REDUCTIONS["none"]
    loss = torch.empty((tokens,) if none else (), device=device, dtype=torch.float32)
    lse = torch.empty(2, tokens, device=device, dtype=torch.float32) if train else None
    rows = torch.empty(_lib.XENT_ROWS + 2 * tokens, device=device, dtype=torch.int32)
    if tokens == 0:   # (a mean, or a sum, of nothing; no gradient reads the rest)
        return loss.fill_(math.nan if reduction == _lib.REDUCTIONS["mean"] else 0.0), lse, rows if train else None
    x_code, w_code, x_ptr, w_ptr = _CODES[x.dtype], _CODES[weight.dtype], x.data_ptr(), weight.data_ptr()
    size = _sized(device, lib.sa_linear_xent_workspace_bytes, x_ptr, x_ld, w_ptr, w_ld, tokens, vocab, width, reduction, train, x_code,
                  w_code, code)
    ws = torch.empty(size, device=device, dtype=torch.uint8)
    _call(device, lib.sa_linear_xent, x_ptr, x_ld, w_ptr, w_ld, targets.data_ptr(), loss.data_ptr(), _ptr(lse), rows.data_ptr(),
          ws.data_ptr(), size, tokens, vocab, width, ignore, reduction, x_code, w_code, code)
    return loss, lse, rows if train else None


def _xent_dense(x: Tensor, weight: Tensor, targets: Tensor, ignore: int, reduction: int, code: int,
                train: bool) -> tuple[Tensor, Tensor, Tensor]:
    loss, lse, rows = _xent_impl(x, weight, targets, ignore, reduction, code, train)
    return (loss, *_filled(lse, like=loss), *_filled(rows, like=x.new_empty(0, dtype=torch.int32)))


_xent_op = _custom_op("linear_cross_entropy_forward", _xent_dense)


@_xent_op.register_fake
def _xent_fake(x, weight, targets, ignore, reduction, code, train):
    f32 = dict(dtype=torch.float32)
    tokens = x.shape[0]
    return (x.new_empty((tokens,) if reduction == 0 else (), **f32), x.new_empty((2, tokens) if train else (0,), **f32),
            x.new_empty((_lib.XENT_ROWS + 2 * tokens if train else 0,), dtype=torch.int32))


def _xent_backward_impl(x: Tensor, weight: Tensor, targets: Tensor, lse: Tensor, rows: Tensor, dloss: Tensor, reduction: int, code: int,
                        need_x: bool, need_weight: bool):
    """sa_linear_xent_backward: dx and dweight in their tensors' types (None where not needed)."""
    tokens, width = x.shape
    vocab, device = weight.shape[0], x.device
    lib = _lib.load()
    dx = _empty(x, x.dtype) if need_x else None
    dweight = _empty(weight, weight.dtype) if need_weight else None
    if tokens == 0:
        return dx, dweight.zero_() if need_weight else None
    x, x_ld = _rows(x, width)
    weight, w_ld = _rows(weight, width)
    targets, dloss = targets.contiguous(), _vector(dloss)
    w_code, w_ptr = _CODES[weight.dtype], weight.data_ptr()
    size = _sized(device, lib.sa_linear_xent_backward_workspace_bytes, w_ptr, w_ld, tokens, vocab, width, need_x, need_weight, w_code, code)
    ws = torch.empty(size, device=device, dtype=torch.uint8)
    _call(device, lib.sa_linear_xent_backward, x.data_ptr(), x_ld, w_ptr, w_ld, targets.data_ptr(), lse.data_ptr(), rows.data_ptr(),
          dloss.data_ptr(), _ptr(dx), _ptr(dweight), ws.data_ptr(), size, tokens, vocab, width, reduction, _CODES[x.dtype], w_code, code)
    return dx, dweight


def _xent_backward_dense(x: Tensor, weight: Tensor, targets: Tensor, lse: Tensor, rows: Tensor, dloss: Tensor, reduction: int, code: int,
                         need_x: bool, need_weight: bool) -> tuple[Tensor, Tensor]:
    dx, dweight = _xent_backward_impl(x, weight, targets, lse, rows, dloss, reduction, code, need_x, need_weight)
    return (*_filled(dx, like=x), *_filled(dweight, like=weight))


_xent_backward_op = _custom_op("linear_cross_entropy_backward", _xent_backward_dense)


@_xent_backward_op.register_fake
def _xent_backward_fake(x, weight, targets, lse, rows, dloss, reduction, code, need_x, need_weight):
    return (x.new_empty(x.shape if need_x else (0,)), weight.new_empty(weight.shape if need_weight else (0,)))


class _LinearCrossEntropyFn(torch.autograd.Function):
    """Keeps x, weight, two numbers per token and the kept tokens' places; the backward pass computes the logits again."""

    @staticmethod
    def forward(ctx, x, weight, targets, ignore, reduction, code):
        ctx.plain = plain = _plain(x, weight, targets)
        loss, lse, rows = (_xent_impl if plain else _xent_op)(x, weight, targets, ignore, reduction, code, True)
        ctx.save_for_backward(x, weight, targets, lse, rows)
        ctx.reduction, ctx.code = reduction, code
        return loss

    @staticmethod
    def backward(ctx, dloss):
        x, weight, targets, lse, rows = ctx.saved_tensors
        need_x, need_weight = ctx.needs_input_grad[:2]
        backward = _xent_backward_impl if _mode_plain(ctx.plain, dloss) else _xent_backward_op
        dx, dweight = backward(x, weight, targets, lse, rows, dloss, ctx.reduction, ctx.code, need_x, need_weight)
        return dx if need_x else None, dweight if need_weight else None, None, None, None, None


def _check_reduction(reduction: str) -> int:
    if reduction not in _lib.REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', not {reduction!r}")
    return _lib.REDUCTIONS[reduction]


def _check_targets(x: Tensor, weight: Tensor, targets: Tensor, ignore_index: int) -> int:
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or x.shape[-1] < 1 or weight.shape[0] < 1:
        raise ValueError(f"x must be (..., C) and weight (V, C); got {tuple(x.shape)}, {tuple(weight.shape)}")
    if targets.dtype is not torch.int64 or targets.shape != x.shape[:-1] or targets.device != x.device:
        raise ValueError(f"targets must be int64 {tuple(x.shape[:-1])} on {x.device}; got {targets.dtype} {tuple(targets.shape)} on "
                         f"{targets.device}")
    if int(ignore_index) != ignore_index or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be a 64-bit integer; got {ignore_index}")
    return int(ignore_index)


def linear_cross_entropy(x: Tensor, weight: Tensor, targets: Tensor, ignore_index: int = -100, reduction: str = "mean",
                         dot_precision: str | None = None) -> Tensor:
    """Softmax cross entropy of the logits x @ weight.T, which are never in memory: for x (..., C), weight (V, C) and targets (...) the
    fp32 loss of every token ("none"), their sum, or their mean over the tokens whose target is not ignore_index (NaN where
    there is none, with gradients of zeros). Ignored tokens cost nothing, and whatever their rows of x hold reaches no result.
    A target outside [0, V) makes the loss and the gradients NaN.

    dot_precision: None takes the products' operands in x's dtype, "bf16" in bf16, "tf32" and "ieee" in fp32 (no TF32 on this
    hardware); x and weight are rounded to it where they are of another type (the fp32 weight of a bf16 autocast step), products
    are summed in fp32. Gradients have x's and weight's own types. The probabilities that enter the gradients' products are
    rounded to 11 bits for bf16 and fp16 operands (to 22 in fp16 where no more than 64 tokens are kept of 64 or of twice as many), not at all for fp32. (bf16 operands enter these in fp16 times a power of two: exactly, but
    for numbers 2^31 times smaller than the largest of x or weight, which are off by 2^-39 of that; "ieee" has no such limit.) With "none" each token's
    row of probabilities has a unit of its own, by the gradient that arrives for it, so that small ones beside large ones keep their bits in x's
    gradient; in weight's, where they are added, what is 2^28 times smaller than the largest (of x times the gradient that arrives) loses bits.

    The backward pass computes the logits again, a piece of the vocabulary at a time: its scratch memory is two pieces of up to 256 MB, fp32
    sums of x's size, two copies of x, a copy of weight where the operands are bf16, and one where its rows do not lie as the kernels read them or are
    of another type. C up to 65536, up to 2^28 - 1 tokens and vocabulary rows, 2^37 logits."""

    _check_float("x", x)
    _check_float("weight", weight, x.device)
    ignore = _check_targets(x, weight, targets, ignore_index)
    code = _check_reduction(reduction)
    operands = _CODES[x.dtype] if dot_precision is None else _resolve_precision(dot_precision, x.dtype)
    vocab, width = weight.shape
    tokens = targets.numel()
    if width > MAX_HEAD_WIDTH or tokens >= 1 << 28 or vocab >= 1 << 28 or -(-tokens // 128) * -(-vocab // 128) >= 1 << 23:
        raise ValueError(f"{tokens} tokens of {width} columns over {vocab} words are too many for one call")
    flat, targets = x.reshape(tokens, width), targets.reshape(tokens)
    if _wants_grad(x, weight):
        loss = _LinearCrossEntropyFn.apply(flat, weight, targets, ignore, code, operands)
    else:
        loss = (_xent_impl if _plain(flat, weight, targets) else _xent_op)(flat, weight, targets, ignore, code, operands, False)[0]
    return loss.reshape(x.shape[:-1]) if reduction == "none" else loss


# -- the same, written plainly ------------------------------------------------------------------------------

def _wide(x: Tensor) -> Tensor:
    return x if x.dtype == torch.float64 else x.float()


def layer_norm_reference(x: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5,
                         dtype: torch.dtype | None = None) -> Tensor:
    """layer_norm, written plainly in fp32 (float64 for float64 inputs); differentiable."""
    centred = _wide(x) - _wide(x).mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps) * _wide(weight)
    y = y if bias is None else y + _wide(bias)
    return y.to(x.dtype if dtype is None else dtype)


def add_layer_norm_reference(x: Tensor, branch: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5,
                             dtype: torch.dtype | None = None) -> tuple[Tensor, Tensor]:
    """add_layer_norm, written plainly."""
    s = (_wide(x) + _wide(branch)).to(x.dtype)
    return layer_norm_reference(s, weight, bias, eps, dtype), s


def embedding_reference(ids: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """embedding, written plainly."""
    held = (ids >= 0) & (ids < weight.shape[0])
    rows = _wide(weight)[torch.where(held, ids, 0).long()] * scale
    return torch.where(held[..., None], rows, float("nan")).to(weight.dtype)


def linear_cross_entropy_reference(x: Tensor, weight: Tensor, targets: Tensor, ignore_index: int = -100, reduction: str = "mean",
                                   dot_precision: str | None = None) -> Tensor:
    """linear_cross_entropy, written plainly with the logits in memory, in fp32 whatever dot_precision."""
    ignore = _check_targets(x, weight, targets, ignore_index)
    _check_reduction(reduction)
    if dot_precision is not None:
        _resolve_precision(dot_precision, x.dtype)
    kept = targets != ignore
    real = (targets >= 0) & (targets < weight.shape[0])
    logits = torch.where(kept[..., None], _wide(x), 0.0) @ _wide(weight).T
    each = torch.logsumexp(logits, -1) - logits.gather(-1, torch.where(real, targets, 0)[..., None])[..., 0]
    each = torch.where(kept, torch.where(real, each, float("nan")), 0.0)
    return each if reduction == "none" else each.sum() if reduction == "sum" else each.sum() / kept.sum()
