"""Edges of the paged operators and of the decoder's paged_step without a GPU."""

import random

import pytest
import torch

from paged_cases import Server, pages_of
from selective_attention import _lib, paged
from selective_attention.model import ModelConfig, SelectiveLM


def small_model(attention="selective", **kw):
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, n_layers=2, d_model=64, n_heads=4, context_length=64, attention=attention)
    return SelectiveLM(cfg).eval()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("precision", [None, "bf16", "ieee"])
def test_step_paged_passes_the_slots_precision_on(monkeypatch, precision):
    model = small_model()
    for block in model.transformer.h:
        block.attn.dot_precision = precision
    seen, plain = [], paged.selective_attention_paged_reference
    monkeypatch.setattr(paged, "selective_attention_paged_reference",
                        lambda *args, dot_precision="not passed", **kw: seen.append(dot_precision) or plain(*args, **kw))
    with torch.no_grad():
        model.paged_step(torch.arange(5), ints(3, 2), model.new_paged_cache(2, 4, 16))
    assert seen == [precision] * 2


def test_an_unknown_precision_is_refused():
    model = small_model()
    model.transformer.h[0].attn.dot_precision = "fp8"
    with pytest.raises(ValueError, match="dot_precision"), torch.no_grad():
        model.paged_step(torch.arange(5), ints(3, 2), model.new_paged_cache(2, 4, 16))


def continued(model, device, bounds, left_out):
    """Two prompts of which a bound leaves one out, the same prompt again without it, and a generated token of both: the
    logits are those of each request's own prefill. `bounds` of the first step, `left_out` the request past it."""
    g = torch.Generator().manual_seed(3)
    counts = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    prompts = [torch.randint(0, 97, (n,), generator=g).to(device) for n in (10, 3)]
    next_ids = torch.randint(0, 97, (2,), generator=g).to(device)
    cache = model.new_paged_cache(2, 8, 8, capacity=32)
    with torch.no_grad():
        _, plan = model.paged_step(torch.cat(prompts), counts(10, 3), cache, **bounds)
        want = [0 if r == left_out else len(p) for r, p in enumerate(prompts)]
        assert plan.lengths.tolist() == want and plan.cached.tolist() == want and cache["cached"].tolist() == want
        rows = [slice(0, 10), slice(10, 13)]
        assert (plan.slots[rows[left_out]] == -1).all() and (plan.slots[rows[1 - left_out]] >= 0).all()
        assert int(cache["taken"]) == sum(-(-n // 8) for n in want)
        again = [len(p) if r == left_out else 0 for r, p in enumerate(prompts)]
        model.paged_step(prompts[left_out], counts(*again), cache)
        logits, plan = model.paged_step(next_ids, counts(1, 1), cache, max_new=1)
        assert plan.lengths.tolist() == [11, 4]
        for r in range(2):
            want = model(torch.cat([prompts[r], next_ids[r:r + 1]])[None])[0][0, 0]
            torch.testing.assert_close(logits[r], want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("bounds", [dict(max_new=4), dict(max_len=8), dict(max_new=9, max_len=32)])
def test_a_request_past_a_bound_is_left_out_of_the_plan(bounds):
    continued(small_model(), "cpu", bounds, 0)


def test_plan_bounds_one_request_at_a_time():
    """Both bounds, met and passed by one; a request without new tokens is past none of them."""
    def plan(**kw):
        table, free = torch.full((4, 8), -1, dtype=torch.int32), torch.arange(20, dtype=torch.int32)
        for r, held in enumerate((2, 1, 1, 5)):
            table[r, :held] = 10 + 5 * r + torch.arange(held)
        return paged.page_plan_reference(ints(9, 4, 0, 40), ints(5, 6, 7, 0), table, free, ints(0), 8, 18, **kw)

    assert plan().lengths.tolist() == [14, 10, 7, 40]
    assert plan(max_new=7, max_len=14).lengths.tolist() == [14, 10, 7, 40]
    assert plan(max_new=6, max_len=14).lengths.tolist() == [14, 10, 0, 40]
    got = plan(max_new=7, max_len=13)
    assert got.lengths.tolist() == [0, 10, 7, 40] and got.cached.tolist() == [9, 10, 7, 40] and got.starts.tolist() == [0, 5, 11, 18, 18]
    assert got.slots[:5].eq(-1).all() and got.slots[5:].ge(0).all() and int(got.taken) == 2
    for wrong in (dict(max_new=0), dict(max_new=1.5), dict(max_len=0), dict(max_len=65), dict(max_len=7.5)):
        with pytest.raises(ValueError, match="max_"):
            plan(**wrong)


def test_a_refused_bound_leaves_the_cache_as_it_was():
    model = small_model()
    cache = model.new_paged_cache(2, 8, 8, capacity=32)
    for wrong in (dict(max_new=0), dict(max_len=33), dict(max_len=0)):
        with pytest.raises(ValueError, match="max_"), torch.no_grad():
            model.paged_step(torch.arange(5), ints(3, 2), cache, **wrong)
        assert not cache["cached"].any() and not cache["taken"].any() and (cache["table"] == -1).all()


def test_abi_refuses_bounds_before_any_launch():
    lib = _lib.load()
    fake = 1 << 20   # never dereferenced: validation fails first
    plan = [fake, fake, None, fake, 8, fake, fake, fake, fake, fake, fake, fake, 4, 8, 100, 10, 16, 10, 128, None]
    for i, value in ((0, None), (4, 7), (12, 0), (15, -1), (16, 24), (17, 0), (17, -1), (18, 0), (18, 129)):
        assert lib.sa_page_plan_within(*plan[:i], value, *plan[i + 1:]) == -1, i


def retired(model, device):
    """A step of no token, in which a request only ends; its pages serve the next."""
    counts = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    cache = model.new_paged_cache(2, 3, 8, capacity=24)
    ids = torch.arange(40, device=device)
    with torch.no_grad():
        model.paged_step(ids[:19], counts(16, 3), cache)   # every page taken
        logits, plan = model.paged_step(ids[:0], counts(0, 0), cache, torch.tensor([True, False], device=device))
        assert logits.shape == (2, 97) and logits.dtype == model.lm_head.weight.dtype and not logits.isnan().any()
        assert plan.lengths.tolist() == [0, 3] and cache["cached"].tolist() == [0, 3] and int(cache["taken"]) == 1
        assert plan.starts.tolist() == [0, 0, 0] and plan.slots.numel() == 0
        logits, plan = model.paged_step(ids[20:33], counts(12, 1), cache)
        assert plan.lengths.tolist() == [12, 4] and int(cache["taken"]) == 3
        for r, row in enumerate((ids[20:32], torch.cat([ids[16:19], ids[32:33]]))):
            torch.testing.assert_close(logits[r], model(row[None])[0][0, 0], rtol=1e-4, atol=1e-4)


def test_a_step_without_tokens():
    retired(small_model(), "cpu")


def test_ids_that_are_none_leave_the_cache_as_it_was():
    model = small_model()
    cache = model.new_paged_cache(2, 8, 8, capacity=32)
    for wrong in (torch.zeros(5), torch.full((5,), 97)):
        with pytest.raises((RuntimeError, IndexError)), torch.no_grad():
            model.paged_step(wrong, ints(3, 2), cache)
        assert not cache["cached"].any() and not cache["taken"].any() and (cache["table"] == -1).all()


def test_a_pending_negation():
    """Rows that are negated when read are laid out; what the kernels write or take whole can only be such a view with strides that
    are refused."""
    x = torch.randn(5, 4, 16).bfloat16()
    rows = paged._rows(torch._neg_view(-x))
    assert not rows.is_neg() and torch.equal(rows, x) and paged._rows(x) is x
    kp, vp = torch.zeros(3, 4, 8, 16), torch.zeros(3, 4, 8, 16)
    args = dict(q=torch.zeros(2, 4, 16), k_pages=kp, v_pages=vp, table=torch.zeros(1, 2, dtype=torch.int32), lengths=ints(2),
                starts=ints(0, 2), selected=torch.zeros(1, 1, 16), exempt=1, max_new=None, max_len=None)
    paged._check_step(**args)
    for name in ("k_pages", "v_pages", "selected"):
        view = torch.complex(args[name], args[name]).conj().imag
        assert view.is_neg() and view.shape == args[name].shape
        with pytest.raises(ValueError):
            paged._check_step(**{**args, name: view})


def one_holder(plan, device, seed):
    """A server's steps, with ends, bounds and a pool that runs out: every page is free or held by one request, once."""
    rng = random.Random(seed)
    s = Server(9, 6, 30, 8, device, seed)
    served = 0
    for _ in range(40):
        new = [rng.choice([0, 1, 1, rng.randrange(30)]) for _ in range(9)]
        ended = [rng.random() < 0.15 for _ in range(9)]
        kw = dict(max_new=rng.choice([None, 20]), max_len=rng.choice([None, 40]))
        made = s.step(lambda *args: plan(*args, **kw), new, None, ended)
        held = [s.table[r, :pages_of(int(s.cached[r]), 8)].tolist() for r in range(9)]
        assert sorted(sum(held, []) + s.free[int(s.taken):].tolist()) == list(range(30))
        served += int((made.lengths > 0).sum())
    assert served > 40


@pytest.mark.parametrize("seed", range(4))
def test_a_page_has_one_holder(seed):
    one_holder(paged.page_plan_reference, "cpu", seed)


def taken_back(ops, device, dtype, rtol, atol):
    """Drafted tokens verified in one step and two of four kept: with the counts and the state put back, and the kept tokens
    run again, all is as if the others had never been. The drafts cross into pages that the kept tokens do not reach."""
    plan, append, attend = ops
    g = torch.Generator().manual_seed(4)
    H, D, P = 2, 16, 8

    class Row(Server):
        def __init__(self):
            super().__init__(2, 4, 8, P, device)
            self.pages = [torch.zeros(8, H, P, D, dtype=dtype, device=device) for _ in range(2)]
            self.selected = torch.zeros(2, 1, 4 * P, device=device)

        def run(self, qkv, new):
            made = self.step(plan, new)
            append(qkv[:, 1], qkv[:, 2], *self.pages, made.slots)
            return attend(qkv[:, 0], *self.pages, self.table, made.lengths, made.starts, self.selected, max_new=max(new))

    tokens = lambda n: torch.randn(n, 3, H, D, generator=g).to(device, dtype)
    prompt, draft, after = tokens(14 + 7), tokens(4 + 4), tokens(2)
    kept = torch.cat([draft[:2], draft[4:6]])
    a, b = Row(), Row()
    a.run(prompt, [14, 7])
    b.run(prompt, [14, 7])
    before = a.cached, a.taken, a.selected.clone()
    first = a.run(draft, [4, 4])
    assert int(a.taken) == 5                      # one page more than the kept tokens need
    a.cached, a.taken = before[:2]
    a.selected.copy_(before[2])
    again, want = a.run(kept, [2, 2]), b.run(kept, [2, 2])
    assert torch.equal(again, want) and torch.equal(a.cached, b.cached) and torch.equal(a.taken, b.taken)
    torch.testing.assert_close(torch.cat([first[:2], first[4:6]]), again, rtol=rtol, atol=atol)
    assert torch.equal(a.run(after, [1, 1]), b.run(after, [1, 1])) and torch.equal(a.selected, b.selected)


def test_a_step_is_taken_back():
    taken_back((paged.page_plan_reference, paged.paged_append_reference, paged.selective_attention_paged_reference), "cpu",
               torch.float32, 1e-5, 1e-6)
