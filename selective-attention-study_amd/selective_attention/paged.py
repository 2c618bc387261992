"""Selective Attention over a paged cache: batches of requests of different lengths, whose keys and values sit in
pages of one pool (no reference counterpart: the reference's caches hold one batch of equal lengths, model.py:76-93).

    k_pages, v_pages   (pages, H, P, D): P positions of one request per page, P a power of two from 8 on
    table              (R, W) int32: position j of request r is in page table[r, j // P], row j % P
    selected           (R, G, L) fp32: the selection every cached position has received, from the request's own queries

A page belongs to one request: page_plan gives it out for one and takes it back when that one has ended, whoever else's
table names it, and counts no holders. (The attention reads pages only, by tables of any making.)

One step of a batch, lengths and tables on the GPU throughout:

    plan = page_plan(cached, new, table, free, taken, P, tokens)           # once (and any max_new, max_len of the attention)
    paged_append(k, v, k_pages, v_pages, plan.slots)                       # per layer
    y = selective_attention_paged(q, k_pages, v_pages, table, plan.lengths, plan.starts, selected)

A step may hold chunks of prompts, single generated tokens and anything between; q, k, v are the new tokens' rows (N, H,
D), request after request. The calls allocate from torch's caching allocator and launch on the current stream of their
tensors' device, so they can be captured into a graph.

The `_reference` functions are the same in plain torch (any device), as `kernels.selective_attention_reference` is.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from .kernels import DTYPES, HEAD_DIMS, _check_exempt, _resolve_precision, _stream

_CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}


class PagePlan(NamedTuple):
    """A step's tables (page_plan)."""

    starts: Tensor    # (R + 1) int32: request r's new tokens are rows starts[r] .. starts[r + 1] - 1
    lengths: Tensor   # (R,) int32: positions after the step; 0 for a request left out of it
    cached: Tensor    # (R,) int32: positions in the cache after the step: the next step's `cached`
    slots: Tensor     # (tokens,) int64: page * P + row of every token; -1: none
    taken: Tensor     # (1,) int32: pages taken from the stack: the next step's `taken`


# -- checks ---------------------------------------------------------------------------------------------

# (A step's host work is of the size of its kernels' for small batches, so the checks read each attribute once. A
# negation can be pending on q, k and v only: what torch makes such views of, the imaginary parts of complex tensors, is no int
# and not contiguous, and the other checks refuse it.)

def _check_page_size(page_size: int) -> int:
    if int(page_size) != page_size or not 8 <= page_size <= 1 << 20 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 8 to 2^20; got {page_size}")
    return int(page_size)


def _check_ints(name: str, t: Tensor, size: int | None, device: torch.device, dtype=torch.int32) -> None:
    """A contiguous vector of `size` (None: any) integers."""
    shape = t.shape
    if (t.dtype is not dtype or t.device != device or len(shape) != 1 or (size is not None and shape[0] != size)
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {'any number of' if size is None else size} elements on "
                         f"{device}; got {t.dtype} {tuple(shape)} on {t.device}")


def _check_table(table: Tensor, requests: int, device: torch.device) -> tuple[int, int]:
    """(row stride, width) of a block table."""
    shape = table.shape
    if table.dtype is torch.int32 and table.device == device and len(shape) == 2 and shape[0] == requests and shape[1] >= 1:
        ld, unit = table.stride()
        if unit == 1 and ld >= shape[1]:
            return ld, shape[1]
    raise ValueError(f"table must be a ({requests}, W) int32 tensor with unit column stride on {device}; got "
                     f"{table.dtype} {tuple(shape)} on {table.device}")


def _check_bounds(max_new: int | None, max_len: int | None, tokens: int, holds: int) -> tuple[int, int]:
    """(max_new, max_len) of a step of `tokens` tokens whose requests have room for `holds` positions."""
    if max_len is None:
        max_len = holds
    elif int(max_len) != max_len or not 1 <= max_len <= holds:
        raise ValueError(f"max_len must be an integer from 1 to the {holds} positions that there is room for; got {max_len}")
    if max_new is None:
        max_new = tokens
    elif int(max_new) != max_new or max_new < 1:
        raise ValueError(f"max_new must be an integer >= 1; got {max_new}")
    return min(int(max_new), tokens), int(max_len)


@functools.lru_cache(maxsize=None)
def _attention_code(dot_precision: str | None, dtype: torch.dtype) -> int:
    """sa_paged_attention's dtype argument."""
    wide = _resolve_precision(dot_precision, dtype) == _lib.DTYPE_F32
    return _CODES[dtype] | (_lib.WIDE_WEIGHTS if wide else 0)


def _check_pages(k_pages: Tensor, v_pages: Tensor) -> tuple[int, int, int, int, torch.dtype, torch.device]:
    """(pages, heads, page size, head dim, dtype, device) of a cache; ValueError unless the kernels can use it."""
    shape, dtype, device = k_pages.shape, k_pages.dtype, k_pages.device
    if len(shape) != 4 or shape != v_pages.shape or shape[0] < 1 or shape[1] < 1:
        raise ValueError(f"k_pages and v_pages must both be (pages, H, P, D); got {tuple(shape)}, {tuple(v_pages.shape)}")
    if dtype not in DTYPES or v_pages.dtype is not dtype:
        raise ValueError(f"the cache's dtype must be float16, bfloat16 or float32, one for both; got {dtype}, {v_pages.dtype}")
    if shape[3] not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}; got {shape[3]}")
    if v_pages.device != device or not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous, on one device")
    return shape[0], shape[1], _check_page_size(shape[2]), shape[3], dtype, device


def _check_cuda(t: Tensor) -> None:
    if not t.is_cuda:
        raise ValueError("the paged operators take CUDA (ROCm) tensors; the _reference functions run anywhere")


def _rows(x: Tensor) -> Tensor:
    """(N, H, D) rows as the kernels read them: 16-byte pieces of contiguous elements, tokens and heads any 16-byte
    multiple apart (a slice of a packed projection is read in place), tokens less than 2^24 bytes; else a contiguous copy (of
    a view that is negated when read, too)."""
    size = x.element_size()
    token, head, unit = x.stride()
    if (unit == 1 and x.shape[2] <= token < (1 << 24) // size and head >= 0 and token * size % 16 == 0 and head * size % 16 == 0
            and x.data_ptr() % 16 == 0 and not x.is_neg()):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _call(device: torch.device, fn, *args) -> None:
    if device.index == torch._C._cuda_getDevice():
        _lib.check(fn(*args, _stream(device)))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _stream(device)))


# -- the operators ----------------------------------------------------------------------------------------

def page_plan(cached: Tensor, new: Tensor, table: Tensor, free: Tensor, taken: Tensor, page_size: int, tokens: int,
              finished: Tensor | None = None, max_new: int | None = None, max_len: int | None = None) -> PagePlan:
    """The tables of one step, made on the GPU from the requests' lengths, without a look at them on the host.

    cached, new: (R,) int32, the positions each request has in the cache and the tokens it gets in this step (0: none).
    table: (R, W) int32, extended in place. free: (F,) int32, the pool's page ids, a stack of which the first
    `taken` (a (1,) int32 tensor) are in use. tokens: rows of the step's batch, at least the sum of `new` (rows behind
    the last request are padding). finished: (R,) bool, optional: requests that have ended; their pages go back on the
    stack first (in place), and their rows start anew, with `new` tokens of another request or with none. (All the pages of their
    `cached` positions: a row that was edited to name another's pages must not be finished here, nor that other one.)

    max_new, max_len: the bounds that the step's selective_attention_paged is given, which leaves requests past them out; they
    are left out of the plan too (where `selected` holds fewer positions than the table, that is such a bound).

    Pages are handed out in request order, all that a request needs or none: a request whose pages are not there, whose
    positions the table cannot hold, whose rows are not among `tokens` or which is past a bound is left out of the step (its
    length 0, its slots -1; `cached` of the plan stays what it was). `cached`, `new` and `taken` are not changed: the plan holds what follows.
    """

    _check_cuda(cached)
    device = cached.device
    if cached.dim() != 1 or not 1 <= cached.shape[0] < 65536:
        raise ValueError(f"cached must be one length per request, 1 to 65535 of them; got {tuple(cached.shape)}")
    requests = cached.shape[0]
    _check_ints("cached", cached, requests, device)
    _check_ints("new", new, requests, device)
    ld, width = _check_table(table, requests, device)
    _check_ints("free", free, None, device)
    _check_ints("taken", taken, 1, device)
    page_size = _check_page_size(page_size)
    if int(tokens) != tokens or not 0 <= tokens < 1 << 24:
        raise ValueError(f"tokens must be an integer from 0 to 2^24 - 1; got {tokens}")
    if width * page_size > 1 << 30:
        raise ValueError("a table row may hold up to 2^30 positions")
    if finished is not None:
        _check_ints("finished", finished, requests, device, torch.bool)
    tokens = int(tokens)
    max_new, max_len = _check_bounds(max_new, max_len, tokens, width * page_size)
    lib = _lib.load()
    starts, lengths, after, now_taken = torch.empty(3 * requests + 2, device=device, dtype=torch.int32).split(
        (requests + 1, requests, requests, 1))
    slots = torch.empty(tokens, device=device, dtype=torch.int64)
    _call(device, lib.sa_page_plan_within, cached.data_ptr(), new.data_ptr(), None if finished is None else finished.data_ptr(),
          table.data_ptr(), ld, free.data_ptr(), taken.data_ptr(), starts.data_ptr(), lengths.data_ptr(),
          after.data_ptr(), slots.data_ptr(), now_taken.data_ptr(), requests, width, free.shape[0], tokens, page_size,
          max(max_new, 1), max_len)
    return PagePlan(starts, lengths, after, slots, now_taken)


def paged_append(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, slots: Tensor) -> None:
    """Writes the new tokens' keys and values (N, H, D) into the cache, row i at slots[i] (N int64 values of
    page * P + row, as page_plan's; distinct; a slot outside the cache, -1 too, leaves its row out). k and v may be any
    views with contiguous head rows (slices of a packed projection), of any of the cache's dtypes; they are rounded
    to the cache's own."""

    _check_cuda(k_pages)
    pages, heads, page_size, head_dim, dtype, device = _check_pages(k_pages, v_pages)
    shape, source = k.shape, k.dtype
    if len(shape) != 3 or shape != v.shape or shape[1] != heads or shape[2] != head_dim:
        raise ValueError(f"k and v must both be (N, {heads}, {head_dim}); got {tuple(shape)}, {tuple(v.shape)}")
    if source not in DTYPES or v.dtype is not source:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, one for both; got {source}, {v.dtype}")
    if k.device != device or v.device != device:
        raise ValueError("k, v and the cache must be on one device")
    tokens = shape[0]
    _check_ints("slots", slots, tokens, device, torch.int64)
    if tokens >= 1 << 24:
        raise ValueError(f"a step holds up to 2^24 - 1 tokens; got {tokens}")
    if tokens * heads * head_dim * k_pages.element_size() >= 1 << 36:   # (a thread per 16 bytes)
        raise ValueError(f"{tokens} tokens of {heads} heads are too many for one launch")
    if tokens == 0:
        return
    lib = _lib.load()
    k, v = _rows(k), _rows(v)
    _call(device, lib.sa_paged_append, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
          k_pages.data_ptr(), v_pages.data_ptr(), slots.data_ptr(), tokens, heads, head_dim, pages, page_size,
          _CODES[source], _CODES[dtype])


def _check_step(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, starts: Tensor, selected: Tensor,
                exempt: int, max_new: int | None, max_len: int | None) -> tuple:
    """The sizes of a step over a paged cache, as selective_attention_paged passes them on."""
    pages, heads, page_size, head_dim, dtype, device = _check_pages(k_pages, v_pages)
    shape = q.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim or q.dtype is not dtype or q.device != device:
        raise ValueError(f"q must be (N, {heads}, {head_dim}) in the cache's dtype {dtype}, on its device; got "
                         f"{tuple(shape)} {q.dtype} on {q.device}")
    tokens = shape[0]
    if tokens >= 1 << 24 or tokens * heads >= 1 << 30:
        raise ValueError(f"a step holds up to 2^24 - 1 tokens and 2^30 - 1 head rows; got {tuple(shape)}")
    if lengths.dim() != 1 or not 1 <= lengths.shape[0] < 65536:
        raise ValueError(f"lengths must be one per request, 1 to 65535 of them; got {tuple(lengths.shape)}")
    requests = lengths.shape[0]
    _check_ints("lengths", lengths, requests, device)
    _check_ints("starts", starts, requests + 1, device)
    ld, width = _check_table(table, requests, device)
    state, strides = selected.shape, selected.stride()
    if (len(state) != 3 or state[0] != requests or state[1] < 1 or heads % state[1] != 0 or selected.dtype is not torch.float32
            or selected.device != device or strides[2] != 1 or strides[0] != state[1] * strides[1] or strides[1] < state[2]):
        raise ValueError(f"selected must be a ({requests}, G, L) fp32 tensor with G dividing H, rows a fixed stride apart, "
                         f"on q's device; got {selected.dtype} {tuple(state)} on {selected.device}")
    holds = min(width * page_size, state[2], (1 << 30) - 1)
    if holds < 1:
        raise ValueError("selected holds no position")
    max_new, max_len = _check_bounds(max_new, max_len, tokens, holds)
    if requests * (heads + state[1] * -(-max_len // 1024)) >= (1 << 24) - 1:   # (workgroups that join parts and write the state)
        raise ValueError(f"a step of {requests} requests of {heads} heads and up to {max_len} positions is too large for one launch")
    return (requests, tokens, heads, state[1], head_dim, pages, page_size, width, max_new, max_len, ld,
            strides[1], dtype, device, _check_exempt(exempt))


def selective_attention_paged(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, starts: Tensor,
                              selected: Tensor, exempt: int = 1, max_new: int | None = None,
                              max_len: int | None = None, dot_precision: str | None = None) -> Tensor:
    """Selective Attention of a step's new tokens over a paged cache that already holds their keys and values.

    q: (N, H, D) in the cache's dtype (any view with contiguous head rows); request r's queries are rows starts[r] ..
    starts[r + 1] - 1, at its positions lengths[r] - n .. lengths[r] - 1. selected: (R, G, L) fp32, G dividing H: for
    every cached position the selection it has received (group g's heads are g*H/G ... and its selector is the
    first of them: G = 1 head 0 for all, G = H every head for itself); updated in place, the new positions' entries
    overwritten. Returns (N, H, D) in q's dtype: for every request what selective_attention_prefill (or, with one
    token, selective_attention_decode) gives on its own contiguous cache. Rows of no request are 0.

    max_new, max_len: upper bounds, known to the caller, of a request's new tokens and of its positions (default: N, and
    what table and selected hold); they size the launch and its workspace, and max_new=1 runs the single-token
    kernels. A request that exceeds a bound, or has fewer positions than new tokens (0 where page_plan left it out), is
    left out: its rows are 0, its state stays (page_plan takes the same bounds, so that such a request's keys are not cached
    either). Positions whose table entry is not a page of the cache read as zeros.

    The state then holds the selection of all the step's queries. To keep only some of its tokens (a draft that is rejected
    from somewhere on), put `selected` and page_plan's `cached` and `taken` back as they were before the step, in which no
    request may have been `finished`, and run the tokens that are kept as a step of their own. (Lowering `cached` alone would
    lose the pages past it.)

    dot_precision, as the package's other entry points have it: None is "bf16" for a bf16 cache and fp32 arithmetic for the others.
    On a bf16 or fp16 cache steps of several tokens run that type's matrix instructions. With "bf16" the softmax weights are
    rounded to the cache's type for the product with the values; with "tf32" or "ieee" they are the sum of two such numbers
    (bf16 to 2^-16, fp16 to 2^-22), which leaves fp32's accuracy, as products of 16-bit numbers are exact in it. Logits, F, softmax
    statistics and sums are fp32 either way, as everything is for an fp32 cache and for single tokens. The output is
    rounded to the cache's type.

    No autograd.
    """

    _check_cuda(k_pages)
    (requests, tokens, heads, groups, head_dim, pages, page_size, width, max_new, max_len, table_ld, state_ld, dtype, device,
     exempt) = _check_step(q, k_pages, v_pages, table, lengths, starts, selected, exempt, max_new, max_len)
    code = _attention_code(dot_precision, dtype)
    out = torch.empty(tokens, heads, head_dim, device=device, dtype=dtype)
    if tokens == 0:
        return out
    lib = _lib.load()
    q = _rows(q)
    size = lib.sa_paged_attention_workspace_bytes(requests, tokens, heads, groups, head_dim, max_new, max_len, code)
    ws = torch.empty(size, device=device, dtype=torch.uint8)
    _call(device, lib.sa_paged_attention, q.data_ptr(), q.stride(0), q.stride(1), k_pages.data_ptr(), v_pages.data_ptr(),
          out.data_ptr(), table.data_ptr(), table_ld, lengths.data_ptr(), starts.data_ptr(), selected.data_ptr(), state_ld,
          ws.data_ptr(), size, requests, tokens, heads, groups, head_dim, pages, page_size, width, max_new, max_len,
          1.0 / math.sqrt(head_dim), code, exempt)
    return out


# -- the same, written plainly ------------------------------------------------------------------------------

def page_plan_reference(cached: Tensor, new: Tensor, table: Tensor, free: Tensor, taken: Tensor, page_size: int, tokens: int,
                        finished: Tensor | None = None, max_new: int | None = None, max_len: int | None = None) -> PagePlan:
    """page_plan, request after request, on the host."""

    max_new, max_len = _check_bounds(max_new, max_len, tokens, table.shape[1] * page_size)
    pages = lambda n: -(-n // page_size)
    stack, top = free.tolist(), int(taken)
    rows, ended = table.tolist(), [False] * len(table) if finished is None else finished.tolist()
    have = [max(n, 0) for n in cached.tolist()]
    back = [page for r, e in enumerate(ended) if e for page in rows[r][:pages(have[r])]]
    top -= len(back)
    stack[top:top + len(back)] = back
    have = [0 if e else c for c, e in zip(have, ended)]
    starts, lengths, after, slots = [0], [], [], []
    asked = given = 0   # pages, by the requests so far and to the last one served
    for row, c, n in zip(rows, have, (max(n, 0) for n in new.tolist())):
        fits = pages(c + n) <= table.shape[1] and (n == 0 or (n <= max_new and c + n <= max_len))
        need = pages(c + n) - pages(c) if fits else 0
        asked += need
        served = fits and starts[-1] + n <= tokens and (need == 0 or asked <= len(stack) - top)
        if served and need:
            row[pages(c):pages(c + n)] = stack[top + asked - need:top + asked]
            given = asked
        slots += [row[j // page_size] * page_size + j % page_size if served else -1 for j in range(c, c + n)]
        starts.append(starts[-1] + n)
        lengths.append(c + n if served else 0)
        after.append(c + n if served else c)

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=cached.device)

    table.copy_(ints(rows))
    free.copy_(ints(stack))
    return PagePlan(ints([min(s, tokens) for s in starts]), ints(lengths), ints(after),
                    ints((slots + [-1] * tokens)[:tokens], torch.int64), ints([top + given]))


def paged_append_reference(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, slots: Tensor) -> None:
    """paged_append, written plainly."""

    page_size = k_pages.shape[2]
    kept = (slots >= 0) & (slots < k_pages.shape[0] * page_size)
    page, row = slots[kept] // page_size, slots[kept] % page_size
    k_pages[page, :, row] = k[kept].to(k_pages.dtype)
    v_pages[page, :, row] = v[kept].to(v_pages.dtype)


def selective_attention_paged_reference(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
                                        starts: Tensor, selected: Tensor, exempt: int = 1, max_new: int | None = None,
                                        max_len: int | None = None, dot_precision: str | None = None) -> Tensor:
    """selective_attention_paged, request after request, in fp32 whatever dot_precision (float64 for float64 inputs); any
    head dim."""

    exempt = _check_exempt(exempt)
    _resolve_precision(dot_precision, q.dtype)
    pages, heads, page_size, head_dim = k_pages.shape
    groups = selected.shape[1]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    holds = min(table.shape[1] * page_size, selected.shape[2])
    max_len = holds if max_len is None else max_len
    max_new = q.shape[0] if max_new is None else max_new
    bounds = starts.tolist()
    for r, t in enumerate(lengths.tolist()):
        a, b = bounds[r], bounds[r + 1]
        n, c = b - a, t - (b - a)
        if n < 1 or c < 0 or t > max_len or n > max_new:
            continue
        pos = torch.arange(t, device=q.device)
        page = table[r, pos // page_size]
        held = (page >= 0) & (page < pages)

        def positions(x):   # (H, t, D)
            rows = x[torch.where(held, page, 0), :, pos % page_size].to(wide)
            return torch.where(held[:, None, None], rows, 0.0).transpose(0, 1)

        keys, vals = positions(k_pages), positions(v_pages)
        logits = (q[a:b].to(wide).transpose(0, 1) @ keys.transpose(1, 2)) / math.sqrt(head_dim)     # (H, n, t)
        grouped = logits.reshape(groups, heads // groups, n, t)
        at = pos[c:, None]
        chosen = torch.where((pos >= exempt) & (pos < at), grouped[:, 0].clamp_min(0.0), 0.0)       # (G, n, t)
        before = torch.where(pos < c, selected[r, :, :t].to(wide), 0.0)
        history = before[:, None] + torch.cumsum(chosen, 1) - chosen
        z = (grouped - history[:, None]).masked_fill(pos > at, float("-inf"))
        out[a:b] = (torch.softmax(z, -1).reshape(heads, n, t) @ vals).transpose(0, 1).to(q.dtype)
        selected[r, :, :t] = (before + chosen.sum(1)).to(selected.dtype)
    return out
