"""The paged cache's kernels on an MI355X, against the operator written out in 64 bits (tests/paged_cases.py) with bounds that
follow from the arithmetic, and against the plain forms."""

import random

import pytest
import torch

import selective_attention as sa
from paged_cases import Server, Step, check, serve
from selective_attention.model import ModelConfig, SelectiveLM

pytestmark = pytest.mark.gpu

# half a step of the type that softmax weights are rounded to for the value product (several tokens)
ROUNDED = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: None}
TYPES = [torch.bfloat16, torch.float16, torch.float32]

# cached and new positions of a batch: nothing cached, tiles and pages that end anywhere, no new token, one, many
MIXED = ([0, 5, 31, 0, 33, 64, 100, 0], [1, 7, 33, 130, 0, 32, 60, 20])
SINGLE = ([0, 1, 31, 32, 63, 64, 100, 300, 7], [1, 1, 1, 1, 1, 1, 1, 1, 0])


def attend(step, device, **kw):
    args = step.args(device)
    out = sa.selective_attention_paged(*args, exempt=step.exempt, **kw)
    torch.cuda.synchronize()
    return out, args[-1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim,heads,groups,page_size,exempt", [
    (64, 4, 1, 16, 1), (64, 3, 1, 8, 1), (64, 4, 4, 64, 3), (64, 4, 2, 32, 16), (128, 2, 1, 16, 1), (128, 2, 2, 128, 1),
    (32, 4, 1, 16, 3), (32, 2, 2, 8, 1), (16, 2, 1, 16, 1), (16, 3, 3, 32, 40)])
def test_several_tokens(cuda, dtype, head_dim, heads, groups, page_size, exempt):
    step = Step(*MIXED, heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, page_size=page_size, exempt=exempt, pad=3)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[dtype])
    assert (out[-3:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim,heads,groups,page_size,exempt", [
    (64, 4, 1, 16, 1), (64, 3, 3, 8, 3), (128, 4, 2, 64, 1), (32, 2, 1, 16, 16), (16, 2, 1, 32, 1)])
def test_one_token(cuda, dtype, head_dim, heads, groups, page_size, exempt):
    step = Step(*SINGLE, heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, page_size=page_size, exempt=exempt, pad=2)
    out, state = attend(step, cuda, max_new=1)
    check(out, state, step)
    assert (out[-2:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 2, 32, 33])
def test_a_long_context_is_split(cuda, dtype, new):
    """Key spans of several workgroups joined, and one token's chunks."""
    step = Step([2500, 40, 1023], [new, 1, new], dtype=dtype, heads=2, spread=0.5)
    out, state = attend(step, cuda, max_new=new)
    check(out, state, step, ROUNDED[dtype] if new > 1 else None)


@pytest.mark.parametrize("new", [1, 5, 70])
def test_large_logits(cuda, new):
    """Rows whose softmax is one key; histories that leave nothing of most keys."""
    step = Step([300, 200], [new, new], dtype=torch.bfloat16, heads=2, spread=4.0)
    out, state = attend(step, cuda, max_new=new)
    check(out, state, step, ROUNDED[torch.bfloat16] if new > 1 else None)


@pytest.mark.parametrize("requests", [1, 65, 300])
def test_many_requests(cuda, requests):
    rng = random.Random(requests)
    step = Step([rng.randrange(40) for _ in range(requests)], [rng.choice([0, 1, 1, 2, 9]) for _ in range(requests - 1)] + [3],
                heads=2, head_dim=32)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[torch.bfloat16])


@pytest.mark.parametrize("max_new", [1, 4])
def test_left_out_requests_and_missing_pages(cuda, max_new):
    new = [max_new] * 4
    step = Step([10, 20, 15, 40], new, dtype=torch.float32, pad=1)
    args = step.args(cuda)
    args[4][1] = max_new - 1     # fewer positions than new tokens
    args[4][3] = 10**6           # more than the bounds hold
    args[3][2, 0] = 10**6        # no such page: its 16 positions are zero rows
    before = args[-1].clone()
    out = sa.selective_attention_paged(*args, max_new=max_new)
    for r in (1, 3):
        assert (out[r * max_new:(r + 1) * max_new] == 0).all()
        assert torch.equal(args[-1][r].nan_to_num(-1.0), before[r].nan_to_num(-1.0))
    step.k[2][:, :16] = 0.0
    step.v[2][:, :16] = 0.0
    want, off, _, _ = step.exact()
    rows = [i for r in (0, 2) for i in range(r * max_new, (r + 1) * max_new)]
    assert ((out.cpu().double() - want).abs() <= off)[rows].all()
    out = sa.selective_attention_paged(*step.args(cuda), max_new=max_new, max_len=24)   # requests 0, 1 and 2 stay within
    assert (out[3 * max_new:] == 0).all() and out[:3 * max_new].abs().sum(-1).gt(0).all()


def test_garbage_starts_and_lengths_stay_in_bounds(cuda):
    step = Step(*MIXED)
    for starts, lengths in (([5, 3, 900, -7, 0, 20, 283, 283, 10**9], [10**9, -5, 0, 7, 2**31 - 1, 64, 3, 1]),
                            ([0] * 9, [50] * 8), ([283] * 9, [0] * 8)):
        args = step.args(cuda)
        args[4], args[5] = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (lengths, starts))
        for max_new in (1, None):
            sa.selective_attention_paged(*args, max_new=max_new)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_bounds_do_not_change_the_bits(cuda, dtype):
    """max_len and a wider table size the launch; the same splits give the same bits, and repeated calls do."""
    step = Step([100, 0], [40, 9], dtype=dtype)
    a, sa_ = attend(step, cuda)
    b, sb = attend(step, cuda, max_len=140, max_new=40)
    c, sc = attend(step, cuda)
    assert torch.equal(a, c) and torch.equal(sa_.nan_to_num(-1), sc.nan_to_num(-1))
    assert torch.equal(a, b) and torch.equal(sa_.nan_to_num(-1), sb.nan_to_num(-1))


def test_queries_from_a_packed_projection(cuda):
    step = Step(*MIXED, heads=4)
    args = step.args(cuda)
    want = sa.selective_attention_paged(*args)
    packed = torch.full((step.tokens, 3, 4, 64), float("nan"), dtype=torch.bfloat16, device=cuda)
    packed[:, 0] = step.q.to(cuda)
    args = step.args(cuda)
    assert torch.equal(sa.selective_attention_paged(packed[:, 0], *args[1:]), want)
    odd = torch.zeros(step.tokens, 4, 67, dtype=torch.bfloat16, device=cuda)   # rows that are not 16-byte aligned
    odd[..., 3:] = step.q.to(cuda)
    args = step.args(cuda)
    assert torch.equal(sa.selective_attention_paged(odd[..., 3:], *args[1:]), want)


def test_it_is_the_prefill_and_the_decode_step(cuda):
    """A request alone on its contiguous cache through the package's other entry points, then in pages among others."""
    step = Step([64, 0, 37], [33, 50, 9], heads=4)
    out, state = attend(step, cuda)
    for r, (c, n) in enumerate(zip(step.cached, step.new)):
        q = step.q[int(step.starts[r]):][:n].transpose(0, 1)[None].to(cuda)
        k, v = (x[r][None].to(cuda) for x in (step.k, step.v))
        mine = step.selected[r, :, :c + n].nan_to_num(0.0).to(cuda).clone()
        y = sa.selective_attention_prefill(q, k, v, mine, c)
        got = out[int(step.starts[r]):][:n].transpose(0, 1)[None].float()
        assert (got - y).abs().max() < 2e-2   # the two kernels' bf16 weights, each within the package's bf16 tolerance of exact
        assert torch.allclose(state[r, :, :c + n], mine, rtol=1e-5, atol=1e-5)
    step = Step([200], [1], heads=4)
    out, state = attend(step, cuda, max_new=1)
    mine = step.selected.nan_to_num(0.0)[:, :, :201].to(cuda).contiguous()
    y = sa.selective_attention_decode(step.q.to(cuda), step.k[0][None].to(cuda), step.v[0][None].to(cuda), mine)
    assert (out.float() - y).abs().max() <= y.abs().max() * 2.0**-7 and torch.allclose(state[:, :, :201], mine, rtol=1e-5, atol=1e-5)


# -- the tables and the cache write -------------------------------------------------------------------------

@pytest.mark.parametrize("requests,width,pool,page_size,most", [
    (1, 4, 4, 8, 20), (7, 6, 20, 16, 40), (64, 10, 300, 8, 30), (70, 40, 1500, 16, 300), (1300, 5, 4000, 8, 12)])
def test_plan_matches_the_plain_form(cuda, requests, width, pool, page_size, most):
    """A server's steps: growing requests, ends and restarts, pools that run out, padded and cut batches."""
    rng = random.Random(requests)
    a, b = Server(requests, width, pool, page_size), Server(requests, width, pool, page_size, cuda)
    for turn in range(6):
        new = [rng.choice([0, 1, 1, 1, rng.randrange(most), -1]) for _ in range(requests)]
        ended = None if turn % 3 == 1 else [rng.random() < 0.2 for _ in range(requests)]
        tokens = max(0, sum(max(n, 0) for n in new) + rng.choice([0, 0, 5, -3]))
        want, got = a.step(sa.page_plan_reference, new, tokens, ended), b.step(sa.page_plan, new, tokens, ended)
        for name, x, y in zip(want._fields, want, got):
            assert torch.equal(x, y.cpu()), (turn, name)
        assert torch.equal(a.table, b.table.cpu()) and torch.equal(a.free, b.free.cpu()), turn


def test_plan_of_a_long_batch(cuda):
    """More tokens than one workgroup maps itself."""
    a, b = Server(40, 400, 9000, 16), Server(40, 400, 9000, 16, cuda)
    for new, extra in (([rng * 37 % 500 for rng in range(40)], 9), ([3000] + [1] * 38 + [1900], 0), ([0] * 39 + [4097], 1)):
        want, got = (s.step(f, new, sum(new) + extra) for s, f in ((a, sa.page_plan_reference), (b, sa.page_plan)))
        for x, y in zip(want, got):
            assert torch.equal(x, y.cpu())
        assert torch.equal(a.table, b.table.cpu())


def test_plan_stays_in_bounds_on_inconsistent_counts(cuda):
    """Counts that no sequence of steps gives: more taken than the pool, finished requests with more pages than taken."""
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
    for taken in (-5, 0, 3, 10**6):
        table, free = ints(*range(12)).view(3, 4), ints(*range(6))
        plan = sa.page_plan(ints(10**6, 2**31 - 1, 9), ints(2**31 - 1, 3, 2**31 - 1), table, free, ints(taken), 8, 16,
                            torch.tensor([True, False, True], device=cuda))
        assert plan.lengths.tolist()[0] == 0 and 0 <= int(plan.taken) <= 6
    torch.cuda.synchronize()


@pytest.mark.parametrize("source", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128])
def test_append_matches_the_plain_form(cuda, source, dtype, head_dim):
    g = torch.Generator(device=cuda).manual_seed(1)
    N, H, P, pages = 77, 3, 8, 30
    packed = torch.randn(N, 3, H, head_dim, device=cuda, generator=g).mul(100).to(source)
    slots = torch.randperm(pages * P, device=cuda, generator=g)[:N]
    slots[5], slots[9], slots[11] = -1, pages * P, 1 << 40
    odd = torch.nn.functional.pad(packed[:, 0], (1, 0))[..., 1:]   # rows that are not 16-byte aligned
    for k, v in ((packed[:, 1], packed[:, 2]), (packed[:, 1].contiguous(), packed[:, 2].contiguous()), (odd, packed[:, 0])):
        want = [torch.full((pages, H, P, head_dim), 7.0, dtype=dtype, device=cuda) for _ in range(2)]
        got = [x.clone() for x in want]
        sa.paged_append_reference(k, v, *want, slots)
        sa.paged_append(k, v, *got, slots)
        assert all(torch.equal(x, y) for x, y in zip(want, got))
    sa.paged_append(packed[:0, 1], packed[:0, 2], *got, slots[:0])   # no token


def test_a_cache_past_32_bit_offsets(cuda):
    """Pages whose elements and bytes lie past 2^31 and 2^32."""
    H, P, D = 16, 64, 128
    pages = (1 << 32) // (H * P * D) + 4          # 2^32 elements and more
    kp, vp = (torch.empty(pages, H, P, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    g = torch.Generator(device=cuda).manual_seed(3)
    for n, c in ((40, 30), (1, 69)):
        table = torch.tensor([[pages - 1, pages // 2 + 1]], dtype=torch.int32, device=cuda)
        k, v, q = (torch.randn(70, H, D, device=cuda, generator=g).bfloat16() for _ in range(3))
        pos = torch.arange(70, device=cuda)
        slots = table[0, pos // P].long() * P + pos % P
        sa.paged_append(k, v, kp, vp, slots)
        ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
        states = [torch.zeros(1, 1, 128, device=cuda) for _ in range(2)]
        out = sa.selective_attention_paged(q[c:], kp, vp, table, ints(70), ints(0, n), states[0], max_new=n)
        small = [x.view(1, 70, H, D).transpose(1, 2) for x in (k, v)]
        small = [torch.nn.functional.pad(x, (0, 0, 0, 58)).view(H, 2, P, D).transpose(0, 1).contiguous() for x in small]
        want = sa.selective_attention_paged(q[c:], *small, ints(0, 1).view(1, 2), ints(70), ints(0, n), states[1], max_new=n)
        assert torch.equal(out, want) and torch.equal(*states)
    del kp, vp
    torch.cuda.empty_cache()


# -- together, as they are used -----------------------------------------------------------------------------

class Layer:
    """One layer's cache with the step's tables: plan, append, attend."""

    def __init__(self, cuda, requests=3, width=8, page_size=16, heads=4, dtype=torch.bfloat16):
        self.s = Server(requests, width, requests * width, page_size, cuda)
        self.k, self.v = (torch.zeros(requests * width, heads, page_size, 64, dtype=dtype, device=cuda) for _ in range(2))
        self.selected = torch.zeros(requests, 1, width * page_size, device=cuda)

    def step(self, qkv, new, max_new=None, tokens=None, finished=None):
        plan = self.s.step(sa.page_plan, new, tokens, finished)
        sa.paged_append(qkv[:, 1], qkv[:, 2], self.k, self.v, plan.slots)
        return sa.selective_attention_paged(qkv[:, 0], self.k, self.v, self.s.table, plan.lengths, plan.starts, self.selected,
                                            max_new=max_new)


def test_steps_follow_one_another(cuda):
    """Chunks and single tokens of several requests, step after step, equal each request's own prefill in one pass."""
    g = torch.Generator(device=cuda).manual_seed(5)
    layer, rows, outs = Layer(cuda), [[], [], []], [[], [], []]
    for new, max_new in (([20, 3, 0], None), ([1, 40, 5], 40), ([1, 1, 1], 1), ([2, 0, 33], 33), ([1, 1, 1], 1), ([1, 1, 1], 4)):
        qkv = torch.randn(sum(new) + 2, 3, 4, 64, device=cuda, generator=g).bfloat16()
        out = layer.step(qkv, new, max_new, tokens=sum(new) + 2)
        assert (out[-2:] == 0).all()
        at = 0
        for r, n in enumerate(new):
            rows[r].append(qkv[at:at + n])
            outs[r].append(out[at:at + n])
            at += n
    for r in range(3):
        q, k, v = torch.cat(rows[r]).permute(1, 2, 0, 3)[:, None].contiguous()
        y, aux = sa.selective_attention_forward(q, k, v, return_aux=True)
        got = torch.cat(outs[r]).transpose(0, 1)[None].float()
        assert (got - y).abs().max() < 2e-2
        assert torch.allclose(layer.selected[r, :, :q.shape[2]], aux["selected_total"], rtol=1e-5, atol=1e-5)


def test_a_row_starts_again_after_a_request_ended(cuda):
    g = torch.Generator(device=cuda).manual_seed(6)
    used, fresh = Layer(cuda), Layer(cuda)
    used.step(torch.randn(60, 3, 4, 64, device=cuda, generator=g).bfloat16(), [30, 20, 10])
    qkv = torch.randn(42, 3, 4, 64, device=cuda, generator=g).bfloat16()
    a = used.step(qkv, [20, 1, 21], finished=[True, False, True])
    b = fresh.step(torch.cat([qkv[:20], qkv[21:]]), [20, 0, 21])
    assert torch.equal(torch.cat([a[:20], a[21:]]), b)
    assert torch.equal(used.selected[0, :, :20], fresh.selected[0, :, :20])


@pytest.mark.parametrize("max_new,new", [(1, [1, 1, 0]), (6, [6, 2, 1])])
def test_captured_and_replayed(cuda, max_new, new):
    """Plan, append and attention in one graph, replayed with new inputs in the same buffers, eager work between."""
    g = torch.Generator(device=cuda).manual_seed(7)
    first = torch.randn(25, 3, 4, 64, device=cuda, generator=g).bfloat16()
    eager, captured = Layer(cuda), Layer(cuda)
    for layer in (eager, captured):
        layer.step(first, [9, 16, 0])
    s = captured.s
    qkv = torch.zeros(sum(new) + 1, 3, 4, 64, device=cuda, dtype=torch.bfloat16)
    counts = torch.tensor(new, dtype=torch.int32, device=cuda)

    def step():
        plan = sa.page_plan(s.cached, counts, s.table, s.free, s.taken, s.page_size, sum(new) + 1)
        sa.paged_append(qkv[:, 1], qkv[:, 2], captured.k, captured.v, plan.slots)
        out = sa.selective_attention_paged(qkv[:, 0], captured.k, captured.v, s.table, plan.lengths, plan.starts,
                                           captured.selected, max_new=max_new)
        s.cached.copy_(plan.cached)
        s.taken.copy_(plan.taken)
        return out

    s.cached, s.taken = s.cached.clone(), s.taken.clone()
    kept = [x.clone() for x in (s.cached, s.taken, s.table, captured.selected, captured.k, captured.v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()   # warm-up, undone below
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((s.cached, s.taken, s.table, captured.selected, captured.k, captured.v), kept):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(5):
        x = torch.randn(qkv.shape, device=cuda, generator=g).bfloat16()
        qkv.copy_(x)
        graph.replay()
        want = eager.step(x, new, max_new, tokens=sum(new) + 1)
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn
        assert torch.equal(captured.selected, eager.selected) and torch.equal(s.cached, eager.s.cached), turn


def test_on_another_stream(cuda):
    step = Step(*MIXED)
    want, state = attend(step, cuda)
    args = step.args(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = sa.selective_attention_paged(*args)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(args[-1].nan_to_num(-1), state.nan_to_num(-1))


def test_refusals_on_the_gpu(cuda):
    step = Step([3], [1], dtype=torch.float32)
    args = step.args(cuda)
    for i, wrong in ((0, step.q), (3, step.table), (4, torch.tensor([4], device=cuda)), (5, step.starts), (6, step.selected)):
        with pytest.raises(ValueError):
            sa.selective_attention_paged(*args[:i], wrong, *args[i + 1:])
    with pytest.raises(ValueError):
        sa.paged_append(args[0], args[0], args[1], args[2], torch.zeros(1, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        sa.page_plan(args[4], args[4].long(), args[3], args[4], args[4], 16, 1)


@pytest.mark.parametrize("attention", ["selective", "selective_x16", "selective_perhead"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_model_serves_requests_of_different_lengths(cuda, attention, dtype):
    """paged_step against each request alone through prefill and decode_step. fp32: both within fp32 rounding through two
    layers. bf16: two paths of two layers, whose activations (norm about 1, logits about 0.2) are each rounded to 2^-8 some
    ten times on the way: 10 * 2^-8 of a logit's size of 1 at most."""
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=211, n_layers=2, d_model=128, n_heads=4, context_length=64, attention=attention)
    model = SelectiveLM(cfg).to(cuda, dtype).eval()
    serve(model, cuda, dtype, rtol=0, atol=1e-4 if dtype == torch.float32 else 4e-2)


def test_a_mixed_step_with_many_single_tokens(cuda):
    """Requests with one new token take the single-token kernels, those with several the others, in one call."""
    rng = random.Random(2)
    cached = [rng.randrange(300) for _ in range(40)]
    new = [1 if r % 10 else 37 for r in range(40)]
    step = Step(cached, new, heads=4, width=400, pad=3)   # (the bound on positions decides: 6000 of them)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[torch.bfloat16])
    assert (out[-3:] == 0).all()
    step = Step([c + 40 for c in cached], [1] * 40, heads=4, width=400, pad=1)
    out, state = attend(step, cuda)   # (no bound given: every request turns out to have one)
    check(out, state, step)
    args = step.args(cuda)
    args[4][3], args[4][7] = 0, 10**7   # left out
    out = sa.selective_attention_paged(*args)
    assert (out[[3, 7, 40]] == 0).all() and (out[[2, 4, 6, 8, 39]].abs().sum(-1) > 0).all()


def outgrown(step, rate):
    """Histories as queries that select at `rate` would have left them: keys some hundred positions back carry no weight."""
    for r, c in enumerate(step.cached):
        step.selected[r, :, :c] = rate * (c - 1 - torch.arange(c)).clamp(min=0)
        step.selected[r, :, :step.exempt] = 0.0
    return step


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim,heads,groups,exempt", [(64, 4, 1, 1), (64, 2, 1, 40), (64, 2, 2, 1), (128, 2, 1, 1), (32, 2, 1, 3), (16, 2, 2, 1)])
def test_key_tiles_without_weight(cuda, dtype, head_dim, heads, groups, exempt):
    """Histories that leave most key tiles out, of requests that cross from such tiles into others, and that have none."""
    step = outgrown(Step([1500, 40, 3000, 0], [70, 200, 33, 130], heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, exempt=exempt,
                         seed=3), 0.4)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[dtype])
    # a little selection: the oldest tiles only
    step = outgrown(Step([4000], [50], heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, exempt=exempt, seed=4), 0.04)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[dtype])


@pytest.mark.parametrize("head_dim,heads", [(64, 4), (128, 2)])
def test_tiles_left_out_keep_the_bits(cuda, head_dim, heads):
    """A value that is not finite, in a tile whose weights are all zero, keeps the tile, of every request before and
    after: the outputs of the heads that do not hold it have the same bits, those of its own are NaN (0 times infinity)."""
    # (requests enough that no request's key tiles are shared out: a part's end would move with the tile that stays)
    step = outgrown(Step([1100] * 140, [40] * 140, heads=heads, head_dim=head_dim, seed=5), 0.4)
    out, state = attend(step, cuda)
    page, mine = int(step.table[100, 500 // 16]), slice(100 * 40, 101 * 40)
    rest = torch.ones(len(out), dtype=torch.bool)
    rest[mine] = False
    step.v_pages[page, 1, 500 % 16, 3] = float("inf")
    kept, again = attend(step, cuda)
    others = [h for h in range(heads) if h != 1]
    assert torch.equal(out[:, others], kept[:, others]) and torch.equal(out[rest], kept[rest])
    assert torch.equal(state.nan_to_num(-1), again.nan_to_num(-1))
    assert kept[mine, 1, 3].isnan().all() and torch.equal(kept[mine, 1, 4:], out[mine, 1, 4:])
    step.v_pages[page, 1, 500 % 16, 3] = 0.0
    step.k_pages[page, 1, 500 % 16, 3] = float("nan")   # a key: every weight of its head
    kept, _ = attend(step, cuda)
    assert kept[mine, 1].isnan().all() and torch.equal(out[:, others], kept[:, others]) and torch.equal(out[rest], kept[rest])
    step.k_pages[page, 1, 500 % 16, 3] = 0.0
    step.selected[100, 0, 500] = float("nan")   # a history: every weight of every head
    kept, _ = attend(step, cuda)
    assert kept[mine].isnan().all() and torch.equal(out[rest], kept[rest])


def test_more_query_tiles_than_a_grid_dimension(cuda):
    """65535 requests, a hundred of them with two new tokens: those, and some of one token, as in a small batch."""
    R, P, D, c = 65535, 8, 16, 20
    g = torch.Generator().manual_seed(0)
    two = torch.arange(100) * 661
    new = torch.ones(R, dtype=torch.int32)
    new[two] = 2
    N = int(new.sum())
    starts = torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0, dtype=torch.int32)]).int()
    table = torch.randint(0, 64, (R, 3), generator=g, dtype=torch.int32)   # pages that requests share
    k, v = (torch.randn(64, 1, P, D, generator=g).to(cuda, torch.bfloat16) for _ in range(2))
    q = torch.randn(N, 1, D, generator=g).to(cuda, torch.bfloat16)
    history = torch.rand(R, 1, 3 * P, generator=g)

    def call(rows):
        at = torch.cat([torch.arange(int(starts[r]), int(starts[r + 1])) for r in rows]) if len(rows) < R else torch.arange(N)
        begin = torch.cat([torch.zeros(1, dtype=torch.int32), new[rows].cumsum(0, dtype=torch.int32)]).int()
        selected = history[rows].to(cuda).contiguous()
        plan = [table[rows].to(cuda), (c + new[rows]).int().to(cuda), begin.to(cuda)]
        out = sa.selective_attention_paged(q[at.to(cuda)].contiguous(), k, v, *plan, selected, max_new=2, max_len=c + 2)
        torch.cuda.synchronize()
        return out, selected, at.to(cuda)

    out, state, _ = call(torch.arange(R))
    some = torch.cat([two, two + 1]).sort().values
    few, few_state, at = call(some)
    assert not out.isnan().any()
    # the two calls may take different kernels: weights rounded to bf16 (half a step, 2^-9, of values up to 4), and each
    # output; states of sums of sixteen fp32 products
    torch.testing.assert_close(out[at].float(), few.float(), rtol=2**-7, atol=2**-7)
    torch.testing.assert_close(state[some.to(cuda)], few_state, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_dim,heads,groups,exempt,rate", [(64, 4, 1, 1, 0.0), (32, 2, 2, 40, 0.1), (128, 1, 1, 1, 0.1)])
def test_long_prompts_whose_histories_are_made_in_segments(cuda, dtype, head_dim, heads, groups, exempt, rate):
    """Some three thousand queries of one request, few others: the walk along the queries is cut, at tiles that neither begin nor
    end a request; a request that ends within the first segment, and one token."""
    step = outgrown(Step([70, 300, 5], [2601, 1033, 1], heads=heads, head_dim=head_dim, groups=groups, dtype=dtype, exempt=exempt, seed=9),
                    rate)
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[dtype])


@pytest.mark.parametrize("head_dim,heads,new", [(64, 4, 34), (32, 1, 40)])
def test_more_key_tiles_than_a_mask_holds(cuda, head_dim, heads, new):
    """270000 positions, more than a workgroup's mask of 8192 key tiles; runs of keys with and without weight in turn, in
    the mask and past it, their ends anywhere in a tile."""
    step = Step([270000], [new], heads=heads, head_dim=head_dim, page_size=64, seed=11)
    j = torch.arange(270000)
    step.selected[0, 0, :270000] = torch.where((j // 997) % 3 == 0, 0.0, 300.0)
    step.selected[0, 0, 0] = 0.0
    out, state = attend(step, cuda)
    check(out, state, step, ROUNDED[torch.bfloat16])
