"""Edges of the paged operators on an MI355X: weights far below a row's largest, bounds, rows of no request, values that are not
finite. Bounds of the comparisons as in tests/paged_cases.py."""

import random

import pytest
import torch

import selective_attention as sa
from paged_cases import Server, Step, check
from selective_attention.model import ModelConfig, SelectiveLM
from test_paged_edges_cpu import continued, one_holder, retired, small_model, taken_back

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]
ROUNDED = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: None}


def put(step, r, k=None, v=None):
    """Other keys and values (H, t, D) of request r, in its pages too."""
    pos = torch.arange(step.lengths[r])
    at = step.table[r, pos // step.page_size].long(), slice(None), pos % step.page_size
    for x, pages, mine in ((k, step.k_pages, step.k), (v, step.v_pages, step.v)):
        if x is not None:
            mine[r] = x.to(step.dtype)
            pages[at] = mine[r].transpose(0, 1)


def attend(step, device, **kw):
    args = step.args(device)
    out = sa.selective_attention_paged(*args, exempt=step.exempt, **kw)
    torch.cuda.synchronize()
    return out, args[-1]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("head_dim,heads,groups,new", [(64, 2, 1, 2), (64, 2, 1, 40), (64, 4, 1, 40), (128, 2, 2, 40), (16, 2, 1, 3)])
def test_one_key_above_a_long_tail(cuda, dtype, head_dim, heads, groups, new):
    """Every row's weight is on position 0, the others' 2^-25.5 of it each, below what fp16 can hold beside 1; their values are
    what the output is made of."""
    c = 3000
    step = Step([c], [new], heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, exempt=c + new)   # (nothing selects)
    step.selected[:, :, :c] = 0.0
    g = torch.Generator().manual_seed(1)
    step.q = torch.zeros(new, heads, head_dim)
    step.q[..., 0] = head_dim**0.5                   # logits: a key's first element, times 1 and what rounding the root leaves
    step.q = step.q.to(dtype)
    k, v = torch.zeros(heads, c + new, head_dim), 4.0 + 4.0 * torch.rand(heads, c + new, head_dim, generator=g)
    k[:, 0, 0] = 17.675 / float(step.q[0, 0, 0]) * head_dim**0.5   # 25.5 log 2
    v[:, 0] = 0.0
    put(step, 0, k, v)
    out, _ = attend(step, cuda)
    want, off, _, _ = step.exact(ROUNDED[dtype])
    # fp16 weights are taken at 2^10 times their size beside the row's largest: rounded to 2^-25 where they are not normal
    # numbers, 2^-35 of the largest (which is all but 2^-13 of the sum)
    if dtype == torch.float16:
        off = off + 2.0**-35 * step.v[0].double().sum(1)[None]
    far = (out.double().cpu() - want).abs()
    assert (far <= off).all(), f"off by {far.max():.3g} of {want.max():.3g}"


# what a weight may be off by as the sum of two numbers of its type
WIDE = {torch.bfloat16: 2.0**-16, torch.float16: 2.0**-22}


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("head_dim,heads,groups,page_size,exempt", [
    (64, 4, 1, 16, 1), (64, 8, 2, 8, 3), (64, 2, 1, 32, 1), (64, 3, 3, 16, 1), (64, 3, 1, 16, 1), (128, 2, 1, 16, 16), (128, 2, 2, 64, 1),
    (32, 4, 1, 16, 1), (16, 2, 1, 16, 1), (16, 2, 2, 32, 1)])
@pytest.mark.parametrize("cached,new", [([0, 31, 64, 0], [33, 33, 60, 2]), ([9, 300], [7, 2]), ([700], [50])])
def test_fp32_arithmetic_on_16_bit_caches(cuda, dtype, head_dim, heads, groups, page_size, exempt, cached, new):
    """dot_precision "ieee" or "tf32": nothing is rounded to the cache's type but the output. The package's default for fp16."""
    step = Step(cached, new, heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, page_size=page_size, exempt=exempt)
    out, state = attend(step, cuda, dot_precision="ieee")
    # (fp16: 2^-35 of a row's largest weight besides, for each of at most 800 keys: less than 2^-25 of values of a size
    # of 4, under half a step of the smallest output that is no zero)
    check(out, state, step, WIDE[dtype])
    assert torch.equal(out, attend(step, cuda, dot_precision="tf32")[0])
    rounded, _ = attend(step, cuda, dot_precision="bf16")
    assert not torch.equal(out, rounded)
    assert torch.equal(attend(step, cuda)[0], out if dtype == torch.float16 else rounded)


def test_precisions_that_change_nothing(cuda):
    step = Step([9, 300], [7, 2], dtype=torch.float32)   # an fp32 cache
    out, _ = attend(step, cuda)
    assert all(torch.equal(out, attend(step, cuda, dot_precision=p)[0]) for p in ("ieee", "tf32", "bf16"))
    step = Step([9, 300], [1, 1], dtype=torch.bfloat16)   # single tokens
    out, _ = attend(step, cuda, max_new=1)
    assert all(torch.equal(out, attend(step, cuda, max_new=1, dot_precision=p)[0]) for p in ("ieee", "tf32", "bf16"))
    with pytest.raises(ValueError, match="dot_precision"):
        attend(step, cuda, dot_precision="fp8")


def test_the_slots_precision_reaches_the_kernels(cuda):
    """A bf16 slot set to "ieee": its paged step is the operator's with fp32 arithmetic, and not the default's."""
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, n_layers=1, d_model=256, n_heads=4, context_length=64)
    slot = SelectiveLM(cfg).to(cuda, torch.bfloat16).eval().transformer.h[0].attn
    x = torch.randn(1, 50, 256, device=cuda).bfloat16()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    got = {}
    with torch.no_grad():
        q, k, v = (y[0].transpose(0, 1) for y in slot.project(x))
        for precision in (None, "ieee"):
            cache, table = slot.new_pages(1, 4, 16, 64, cuda, torch.bfloat16), ints(2, 0, 1, 3).view(1, 4)
            plan = sa.page_plan(ints(0), ints(50), table, ints(2, 0, 1, 3), ints(0), 16, 50)
            slot.dot_precision = precision
            got[precision] = slot.step_paged(x, cache, table, plan)
            y = sa.selective_attention_paged(q, cache["k"], cache["v"], table, plan.lengths, plan.starts,
                                             torch.zeros_like(cache["selected"]), dot_precision=precision)
            assert torch.equal(got[precision], slot.emit(y.transpose(0, 1)[None]))
    assert not torch.equal(got[None], got["ieee"])


@pytest.mark.parametrize("max_new", [1, 2, 40])
def test_rows_before_the_first_request(cuda, max_new):
    """starts[0] is not 0: a call on some of a step's requests. The rows of no request are zeros, whatever memory held."""
    step = Step([70, 5, 40], [max_new, 1, max_new], dtype=torch.bfloat16)
    args = step.args(cuda)
    want, lead = sa.selective_attention_paged(*args, max_new=max_new), 300
    args = step.args(cuda)
    args[0] = torch.cat([args[0].new_zeros(lead, *args[0].shape[1:]), args[0], args[0].new_zeros(7, *args[0].shape[1:])])
    args[5] = args[5] + lead
    for _ in range(2):
        junk = torch.full(args[0].shape, float("nan"), dtype=args[0].dtype, device=cuda)   # the block that the output takes
        del junk
        out = sa.selective_attention_paged(*args[:6], args[6].clone(), max_new=max_new)
        assert (out[:lead] == 0).all() and (out[lead + step.tokens:] == 0).all()
    assert not out.isnan().any() and torch.allclose(out[lead:lead + step.tokens].float(), want.float(), atol=2.0**-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("new", [1, 2, 40])
@pytest.mark.parametrize("head_dim,first", [(64, 64), (64, 0), (128, 320), (16, 1024)])
def test_a_page_of_nan_is_not_lost(cuda, dtype, new, head_dim, first):
    """Keys that are NaN a whole page long: every row that sees them is NaN, as for a single one."""
    step = Step([1300], [new], heads=2, head_dim=head_dim, dtype=dtype, page_size=128)
    at = first // 128 * 128
    step.k_pages[int(step.table[0, at // 128]), 1] = float("nan")
    out, _ = attend(step, cuda, max_new=new)
    assert out[:, 1].isnan().all() and not out[:, 0].isnan().any()


@pytest.mark.parametrize("requests,width,pool,page_size,most", [(7, 6, 30, 16, 40), (70, 40, 2500, 16, 300), (1300, 5, 6000, 8, 12)])
def test_plan_with_bounds_matches_the_plain_form(cuda, requests, width, pool, page_size, most):
    rng = random.Random(requests)
    a, b = Server(requests, width, pool, page_size), Server(requests, width, pool, page_size, cuda)
    left_out = 0
    for turn in range(8):
        new = [rng.choice([0, 1, 1, 1, rng.randrange(most)]) for _ in range(requests)]
        ended = [rng.random() < 0.1 for _ in range(requests)]
        kw = dict(max_new=rng.choice([1, most // 2, most, 10**12]), max_len=rng.choice([page_size, width * page_size // 2 + 3, width * page_size]))
        want, got = (s.step(lambda *args: plan(*args, **kw), new, None, ended)
                     for s, plan in ((a, sa.page_plan_reference), (b, sa.page_plan)))
        for name, x, y in zip(want._fields, want, got):
            assert torch.equal(x, y.cpu()), (turn, name, kw)
        assert torch.equal(a.table, b.table.cpu()) and torch.equal(a.free, b.free.cpu()), turn
        left_out += sum(n > kw["max_new"] for n in new)
    assert left_out > 0


@pytest.mark.parametrize("bounds", [dict(max_new=4), dict(max_len=8)])
def test_a_request_past_a_bound_is_left_out_of_the_plan(cuda, bounds):
    continued(small_model().to(cuda), cuda, bounds, 0)


def test_a_step_without_tokens(cuda):
    retired(small_model().to(cuda), cuda)


def test_a_pending_negation(cuda):
    """Views that are negated when read: as the same values laid out."""
    step = Step([30, 3], [20, 1], dtype=torch.bfloat16)
    args = step.args(cuda)
    want = sa.selective_attention_paged(*args)
    args = step.args(cuda)
    q = torch._neg_view(-args[0])
    assert q.is_neg() and torch.equal(sa.selective_attention_paged(q, *args[1:]), want)
    pages = [torch.zeros(4, 4, 16, 64, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    slots = torch.arange(21, device=cuda)
    k = torch.randn(21, 4, 64, device=cuda).bfloat16()
    sa.paged_append(torch._neg_view(-k), k, *pages, slots)
    assert torch.equal(*pages) and pages[0].count_nonzero() > 0


@pytest.mark.parametrize("seed", range(4))
def test_a_page_has_one_holder(cuda, seed):
    one_holder(sa.page_plan, cuda, seed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_is_taken_back(cuda, dtype):
    # (fp32: sums of some twenty terms in another order; bf16: outputs and weights rounded, 2^-8 each, of values up to 4)
    rtol, atol = (1e-5, 1e-5) if dtype == torch.float32 else (2.0**-7, 2.0**-5)
    taken_back((sa.page_plan, sa.paged_append, sa.selective_attention_paged), cuda, dtype, rtol, atol)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("precision", ["bf16", "ieee"])
@pytest.mark.parametrize("heads,groups", [(4, 1), (8, 2), (2, 1)])
@pytest.mark.parametrize("cached,new", [([300, 200], [70, 40]), ([1200], [40])])
def test_large_logits_in_groups(cuda, dtype, precision, heads, groups, cached, new):
    """Logits of up to some hundreds: rows whose softmax is one key, newer tiles outgrown by older ones."""
    step = Step(cached, new, heads=heads, groups=groups, dtype=dtype, spread=4.0)
    out, state = attend(step, cuda, dot_precision=precision)
    check(out, state, step, ROUNDED[dtype] if precision == "bf16" else WIDE[dtype])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("precision", ["bf16", "ieee"])
@pytest.mark.parametrize("heads,groups", [(4, 1), (8, 2), (2, 1)])
@pytest.mark.parametrize("c", [200, 1500])
def test_older_tiles_outgrow_newer_ones(cuda, dtype, precision, heads, groups, c):
    """Steps up of a row's logits from tile to tile, newest first: by slightly less than what the four-head kernel lets pass before
    it looks for another maximum (2^14 of bf16 weights, 2^5 of fp16's over their 2^10), by slightly more, by far more, for all
    rows and for every third row only. c = 1500: the tiles are shared out over workgroups."""
    n = 40
    step = Step([c], [n], heads=heads, groups=groups, dtype=dtype, exempt=c + n, page_size=8)   # (nothing selects)
    step.selected[:, :, :c] = 0.0
    g = torch.Generator().manual_seed(2)
    log2 = 0.6931
    k = 0.02 * torch.randn(heads, c + n, 64, generator=g)
    steps = torch.zeros(c + n)
    for at, up in ((c - 40, 4.9), (c - 80, 9.7), (c - 110, 9.7 + 13.9), (c - 140, 9.7 + 28.2), (c - 170, 24.0)):
        steps[at:at + 5] = up * log2     # of every row
    k[:, :, 0] = steps
    k[:, c - 190:c - 185, 1] = 60.0 * log2   # of every third row: far more
    k[:, c - 60, 1] = 14.1 * log2
    put(step, 0, k, torch.randn(heads, c + n, 64, generator=g) + 0.5)
    q = 0.02 * torch.randn(n, heads, 64, generator=g)
    q[..., 0] = 8.0
    q[..., 1] = 0.0
    q[::3, :, 1] = 8.0
    step.q = q.to(dtype)
    out, state = attend(step, cuda, dot_precision=precision)
    check(out, state, step, ROUNDED[dtype] if precision == "bf16" else WIDE[dtype])


def test_a_decoders_step_is_captured(cuda):
    """paged_step in a graph, replayed as the requests grow, with a request that ends and starts again: the logits and the counts
    of eager steps, bounds and all."""
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, n_layers=2, d_model=256, n_heads=4, context_length=64)
    model = SelectiveLM(cfg).to(cuda, torch.bfloat16).eval()
    caches = [model.new_paged_cache(3, 12, 16, capacity=64) for _ in range(2)]
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
    tensors = lambda cache: [cache[k] for k in ("table", "free", "taken", "cached")] + [x for layer in cache["layers"] for x in layer.values()]
    g = torch.Generator().manual_seed(1)
    ids, new, ended = (torch.zeros(8, dtype=torch.int64, device=cuda), ints(0, 0, 0), torch.zeros(3, dtype=torch.bool, device=cuda))
    with torch.no_grad():
        prompt = torch.randint(0, 97, (20,), generator=g).to(cuda)
        for cache in caches:
            model.paged_step(prompt, ints(9, 11, 0), cache)
        step = lambda cache: model.paged_step(ids, new, cache, ended, max_new=6, max_len=64)
        kept = [x.clone() for x in tensors(caches[1])]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(caches[1])   # warm-up, undone below
        torch.cuda.current_stream().wait_stream(side)
        for x, y in zip(tensors(caches[1]), kept):
            x.copy_(y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits, plan = step(caches[1])
        for counts, ends in (((1, 1, 6), None), ((2, 1, 1), None), ((7, 1, 0), None), ((3, 0, 5), (1, 0, 0)), ((1, 1, 1), None)):
            ids.copy_(torch.randint(0, 97, (8,), generator=g))
            new.copy_(ints(*counts))
            ended.copy_(torch.tensor(ends or (0, 0, 0), device=cuda).bool())
            graph.replay()
            want, made = step(caches[0])
            torch.cuda.synchronize()
            rows = [r for r in range(3) if counts[r] and int(made.lengths[r])]
            assert all(torch.equal(x, y) for x, y in zip(made, plan)) and torch.equal(want[rows], logits[rows]), counts
            assert all(torch.equal(x, y) for x, y in zip(tensors(caches[0]), tensors(caches[1]))), counts
