"""Requests over a paged cache for the tests: inputs, and the operator written out query by query in 64 bits."""

import math

import torch

from selective_attention import paged


def pages_of(n, page_size):
    return -(-n // page_size)


class Step:
    """One step of a batch: `cached` and `new` positions of every request, keys and values of all of them in pages of
    a scattered pool. What no request may read is NaN: pages that nobody holds, rows of a last page past the last position,
    table entries past it (which name a page of NaN), and the state of positions that are new."""

    def __init__(self, cached, new, heads=4, head_dim=64, groups=1, dtype=torch.bfloat16, page_size=16, exempt=1, pad=0,
                 seed=0, width=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.cached, self.new, self.exempt, self.page_size = list(cached), list(new), exempt, page_size
        self.heads, self.head_dim, self.groups, self.dtype = heads, head_dim, groups, dtype
        ts = self.lengths = [c + n for c, n in zip(cached, new)]
        held = [pages_of(t, page_size) for t in ts]
        self.pages = sum(held) + 2
        order = torch.randperm(self.pages - 1, generator=g) + 1   # page 0 is nobody's
        W = max(max(held), 1) + width
        self.table = torch.zeros(len(ts), W, dtype=torch.int32)
        nan = float("nan")
        self.k_pages = torch.full((self.pages, heads, page_size, head_dim), nan)
        self.v_pages = torch.full((self.pages, heads, page_size, head_dim), nan)
        self.k, self.v = [], []
        at = 0
        for r, t in enumerate(ts):
            mine = order[at:at + held[r]]
            at += held[r]
            self.table[r, :held[r]] = mine.int()
            k, v = (torch.randn(heads, t, head_dim, generator=g) * s for s in (spread, 1.0))
            self.k.append(k.to(dtype))
            self.v.append(v.to(dtype))
            pos = torch.arange(t)
            for x, rows in ((self.k_pages, k), (self.v_pages, v)):
                x[mine[pos // page_size], :, pos % page_size] = rows.transpose(0, 1)
        self.k_pages, self.v_pages = self.k_pages.to(dtype), self.v_pages.to(dtype)
        self.tokens = sum(new) + pad
        self.q = (torch.randn(self.tokens, heads, head_dim, generator=g) * spread).to(dtype)
        self.starts = torch.tensor([sum(new[:r]) for r in range(len(new) + 1)], dtype=torch.int32)
        L = max(W * page_size, 1)
        self.selected = torch.full((len(ts), groups, L), nan)
        for r, c in enumerate(cached):
            # decaying with the position, so that some keys' weights are gone and others' are not
            state = torch.rand(groups, c, generator=g) * (0.02 * (c - torch.arange(c))).clamp(max=30.0)
            state[:, :exempt] = 0.0
            self.selected[r, :, :c] = state

    def args(self, device="cpu"):
        """The operator's positional arguments on a device (the state a copy)."""
        lengths = torch.tensor(self.lengths, dtype=torch.int32)
        return [x.to(device) for x in (self.q, self.k_pages, self.v_pages, self.table, lengths, self.starts, self.selected.clone())]

    def exact(self, rounded=None):
        """((N, H, D) outputs, (R, G, L) state) in 64 bits, and for each how far fp32 arithmetic may be off, element by
        element. `rounded`: the relative rounding of the weights (half a step of their type), None: not rounded.

        With u = 2^-24 half a step of fp32. A logit s q.k (D products, D - 1 sums, the scale, each rounded) is off by at most
        e = (D + 2) u s sum |q k|, and a selection, its positive part, no more. A history of m such terms, summed in any
        order, is off by their errors and (m + 2) u of its value; the difference L - F, and its product with log2 e in the
        exponent, by 2 u (|L| + F + |max|) more: together d_j on key j's exponent. The weight is then off by d_j
        relative, 2^-22 for the exponential and its accumulation rescaled, the sum by the same mean over the keys,
        and t terms in fp32 sums by t u: so |out - exact| <= sum_j w_j |v_j| (rounded + d_j + sum_k w_k d_k + 2^-21 + 2 t u) to
        first order (second order: a tenth more), plus half a step of the output's type."""
        u = 2.0**-24
        N, H, D, G = self.tokens, self.heads, self.head_dim, self.groups
        s = 1.0 / math.sqrt(D)
        out, off = torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64)
        state, state_off = self.selected.double().clone(), torch.zeros(self.selected.shape, dtype=torch.float64)
        for r, t in enumerate(self.lengths):
            n, c, first = self.new[r], self.cached[r], int(self.starts[r])
            if n == 0:
                continue
            k, v = self.k[r].double(), self.v[r].double()
            for g in range(G):
                heads = range(g * H // G, (g + 1) * H // G)
                F = torch.cat([state[r, g, :c], torch.zeros(n, dtype=torch.float64)])
                F_off = u * F
                for i in range(n):
                    at = c + i
                    for h in heads:
                        qi = self.q[first + i, h].double()
                        L = s * (k[h, :at + 1] @ qi)
                        e = (D + 2) * u * s * (k[h, :at + 1].abs() @ qi.abs())
                        if h == heads[0]:
                            chosen, chosen_off = L.clamp(min=0.0), e.clone()
                            chosen[:self.exempt] = 0.0
                            chosen_off[:self.exempt] = 0.0
                            chosen[at:] = 0.0
                            chosen_off[at:] = 0.0
                        z = L - F[:at + 1]
                        w = torch.softmax(z, 0)
                        d = e + F_off[:at + 1] + (i + 2) * u * F[:at + 1] + 2 * u * (L.abs() + F[:at + 1] + z.max().abs())
                        lost = (rounded or 0.0) + d + (w * d).sum() + 2.0**-21 + 2 * t * u
                        out[first + i, h] = w @ v[h, :at + 1]
                        off[first + i, h] = 1.1 * ((w * lost) @ v[h, :at + 1].abs())
                    F[:at + 1] += chosen
                    F_off[:at + 1] += chosen_off
                state[r, g, :t] = F
                state_off[r, g, :t] = F_off + (n + 4) * u * F
        off += out.abs() * torch.finfo(self.dtype).eps / 2 + 2.0**-133
        return out, off, state, state_off


def check(got, state, step, rounded=None, what=""):
    """Outputs and state within their bounds; the state of what no request holds as it was."""
    out, off, want, want_off = step.exact(rounded)
    far = (got.double().cpu() - out).abs()
    assert not got.isnan().any(), f"{what}: NaN in the output"
    bad = far > off
    assert not bad.any(), f"{what}: output off by {far[bad].max():.3g} at {bad.nonzero()[0].tolist()}, allowed {off[bad][0]:.3g}"
    state = state.double().cpu()
    same = want.isnan() & state.isnan()
    far = (state - want).abs()
    bad = ~same & ~(far <= want_off)
    assert not bad.any(), f"{what}: state off at {bad.nonzero()[0].tolist()}: {state[bad][0]:.6g}, {want[bad][0]:.6g} +- {want_off[bad][0]:.2g}"


class Server:
    """A pool and its tables, for tests of page_plan: `plan` is page_plan or page_plan_reference."""

    def __init__(self, requests, width, pool, page_size, device="cpu", seed=0):
        g = torch.Generator().manual_seed(seed)
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)
        self.cached, self.taken = ints(requests), ints(1)
        self.table = ints(requests, width) - 1
        self.free = torch.randperm(pool, generator=g).int().to(device)
        self.page_size, self.device = page_size, device

    def step(self, plan, new, tokens=None, finished=None):
        ints = torch.tensor(new, dtype=torch.int32, device=self.device)
        ended = None if finished is None else torch.tensor(finished, device=self.device)
        made = plan(self.cached, ints, self.table, self.free, self.taken, self.page_size,
                    sum(max(n, 0) for n in new) if tokens is None else tokens, ended)
        assert isinstance(made, paged.PagePlan)
        self.cached, self.taken = made.cached, made.taken
        return made


def serve(model, device, dtype, rtol, atol):
    """A server's run through a decoder: two prompts, one of them in chunks, a request that comes later, one that ends and
    whose row another takes; every request's logits against its own prefill and decode steps."""
    g = torch.Generator().manual_seed(1)
    vocab = model.config.vocab_size
    cache = model.new_paged_cache(3, 14, 16, capacity=64, dtype=dtype)
    seen = [[], [], []]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    with torch.no_grad():
        for new, ended, max_new in (([17, 5, 0], None, None), ([1, 9, 0], None, 9), ([1, 1, 30], None, None), ([1, 1, 1], None, 1),
                                    ([1, 20, 1], [False, True, False], 20), ([1, 1, 1], None, 1)):
            ids = torch.randint(0, vocab, (sum(new),), generator=g)
            for r, part in enumerate(ids.split(new)):
                if ended and ended[r]:
                    seen[r] = []
                seen[r].append(part)
            logits, plan = model.paged_step(ids.to(device), ints(new), cache, None if ended is None else torch.tensor(ended, device=device),
                                            max_new=max_new)
            assert plan.lengths.tolist() == [sum(len(x) for x in row) for row in seen]
            for r, row in enumerate(seen):
                if new[r]:
                    ids = torch.cat(row)[None].to(device)
                    want = model.prefill(ids[:, :-1], capacity=64)[1] if ids.shape[1] > 1 else None
                    want = model.prefill(ids)[0] if want is None else model.decode_step(ids[:, -1:], 0, want)
                    torch.testing.assert_close(logits[r], want[0, 0].to(logits.dtype), rtol=rtol, atol=atol)
    held = [pages_of(int(n), 16) for n in cache["cached"].tolist()]
    assert int(cache["taken"]) == sum(held)
