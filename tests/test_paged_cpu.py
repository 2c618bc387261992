"""The paged cache without a GPU: the plain forms against the operator written out and against the oracle, the tables
against a pool kept by hand, and the refusals, in Python and at the C ABI."""

import pytest
import torch

import selective_attention as sa
from oracle import sa_oracle
from paged_cases import Server, Step, check, pages_of, serve
from selective_attention import _lib, paged
from selective_attention.model import ModelConfig, SelectiveLM


@pytest.mark.parametrize("groups,exempt,page_size", [(1, 1, 16), (2, 3, 8), (4, 16, 32)])
def test_plain_attention_is_the_operator(groups, exempt, page_size):
    step = Step([0, 5, 40, 0, 33], [7, 1, 12, 0, 3], groups=groups, exempt=exempt, page_size=page_size, dtype=torch.float32,
                head_dim=32, pad=2)
    args = step.args()
    out = sa.selective_attention_paged_reference(*args, exempt=exempt)
    check(out, args[-1], step)
    assert (out[-2:] == 0).all()


def test_a_prompt_is_the_oracles_attention():
    step = Step([0], [50], head_dim=16, dtype=torch.float64)
    args = step.args()
    args[-1] = args[-1].double()
    out = sa.selective_attention_paged_reference(*args)
    want = sa_oracle.attention(step.q.transpose(0, 1)[None], step.k[0][None], step.v[0][None])
    assert torch.allclose(out.transpose(0, 1)[None], want, rtol=1e-12, atol=1e-12)


def test_left_out_requests_and_missing_pages():
    step = Step([10, 20, 5], [3, 2, 4], dtype=torch.float32)
    args = step.args()
    args[4][1] = 1           # fewer positions than new tokens
    args[3][2, 0] = 10**6    # no such page: zero rows
    before = args[-1].clone()
    out = sa.selective_attention_paged_reference(*args)
    assert (out[3:5] == 0).all()
    assert torch.equal(args[-1][1].nan_to_num(-1.0), before[1].nan_to_num(-1.0))
    step.k[2][:, :16] = 0.0
    step.v[2][:, :16] = 0.0
    step.new[1], step.lengths[1] = 0, 20
    want = step.exact()
    assert ((out.double() - want[0]).abs() <= want[1])[[0, 1, 2, 5, 6, 7, 8]].all()


def test_plan_hands_out_and_takes_back_pages():
    s = Server(4, 8, 12, 8)
    pool = s.free.tolist()
    plan = s.step(sa.page_plan_reference, [9, 0, 8, 1])
    assert plan.starts.tolist() == [0, 9, 9, 17, 18] and plan.lengths.tolist() == [9, 0, 8, 1]
    assert s.table[0, :2].tolist() == pool[:2] and s.table[2, 0] == pool[2] and s.table[3, 0] == pool[3]
    assert plan.slots.tolist() == [pool[0] * 8 + i for i in range(8)] + [pool[1] * 8] + [pool[2] * 8 + i for i in range(8)] + [pool[3] * 8]
    plan = s.step(sa.page_plan_reference, [1, 1, 1, 1])       # positions 9, 0, 8, 1: pages for requests 1 and 2
    assert plan.slots.tolist() == [pool[1] * 8 + 1, pool[4] * 8, pool[5] * 8, pool[3] * 8 + 1] and s.taken.tolist() == [6]
    # request 0 ends and its row takes a prompt of 20; request 1's 60 tokens do not fit the 8 - 3 pages left
    plan = s.step(sa.page_plan_reference, [20, 60, 0, 1], finished=[True, False, False, False])
    assert plan.lengths.tolist() == [20, 0, 9, 3] and plan.cached.tolist() == [20, 1, 9, 3] and plan.slots[20:80].eq(-1).all()
    assert s.free.tolist()[4:6] == pool[:2] and s.table[0, :3].tolist() == [pool[0], pool[1], pool[6]] and s.taken.tolist() == [7]
    held = [s.table[r, :pages_of(int(s.cached[r]), 8)].tolist() for r in range(4)]
    assert sorted(sum(held, []) + s.free.tolist()[7:]) == sorted(pool)


def test_plan_leaves_out_what_does_not_fit():
    s = Server(3, 2, 10, 8)
    plan = s.step(sa.page_plan_reference, [17, 16, 3], tokens=35)   # wider than its row; fits; its rows past the batch
    assert plan.lengths.tolist() == [0, 16, 0] and plan.starts.tolist() == [0, 17, 33, 35] and s.taken.tolist() == [2]
    assert plan.slots[:17].eq(-1).all() and plan.slots[33:].eq(-1).all() and len(plan.slots) == 35


def test_append_rounds_and_leaves_out():
    kp, vp = torch.zeros(3, 2, 8, 16, dtype=torch.bfloat16), torch.zeros(3, 2, 8, 16, dtype=torch.bfloat16)
    k, v = torch.randn(4, 2, 16), torch.randn(4, 2, 16)
    sa.paged_append_reference(k, v, kp, vp, torch.tensor([9, -1, 23, 24]))
    assert torch.equal(kp[1, :, 1], k[0].bfloat16()) and torch.equal(vp[2, :, 7], v[2].bfloat16())
    assert kp.count_nonzero() == 64


def test_refusals():
    step = Step([3, 4], [1, 2], dtype=torch.float32)
    q, kp, vp, table, lengths, starts, selected = step.args()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        sa.selective_attention_paged(q, kp, vp, table, lengths, starts, selected)
    with pytest.raises(ValueError, match="CUDA"):
        sa.paged_append(q, q, kp, vp, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        sa.page_plan(ints(1), ints(1), ints(0).view(1, 1), ints(0), ints(0), 16, 1)
    check_step = lambda **kw: paged._check_step(**{**dict(q=q, k_pages=kp, v_pages=vp, table=table, lengths=lengths, starts=starts,
                                                         selected=selected, exempt=1, max_new=None, max_len=None), **kw})
    assert check_step()[6:10] == (16, 1, 3, 16)
    for wrong in (dict(q=q[0]), dict(q=q.half()), dict(q=q[:, :2]), dict(k_pages=kp[:, :, :5]), dict(v_pages=vp.half()),
                  dict(k_pages=kp[:, :, :12].contiguous(), v_pages=vp[:, :, :12].contiguous()),
                  dict(k_pages=kp.double(), v_pages=vp.double()), dict(k_pages=kp.transpose(1, 2), v_pages=vp.transpose(1, 2)),
                  dict(table=table.long()), dict(table=table[:1]), dict(lengths=lengths[:1]), dict(lengths=lengths.long()),
                  dict(starts=starts[:2]), dict(selected=selected.double()), dict(selected=selected[:1]),
                  dict(selected=selected.expand(2, 3, 16)), dict(selected=selected[:, :, ::2]), dict(exempt=0), dict(max_new=0),
                  dict(max_len=17), dict(max_len=0), dict(max_new=1.5)):
        with pytest.raises(ValueError):
            check_step(**wrong)
    with pytest.raises(ValueError, match="page_size"):
        paged._check_page_size(24)


def test_abi_refuses_before_any_launch():
    lib = _lib.load()
    fake = 1 << 20   # never dereferenced: validation fails first
    plan = [fake, fake, None, fake, 8, fake, fake, fake, fake, fake, fake, fake, 4, 8, 100, 10, 16, None]
    for i, value in ((0, None), (3, None), (4, 7), (12, 0), (12, 65536), (13, 0), (14, -1), (15, -1), (15, 1 << 24), (16, 4), (16, 24)):
        assert lib.sa_page_plan(*plan[:i], value, *plan[i + 1:]) == -1, i
    append = [fake, 256, 64, fake, 256, 64, fake, fake, fake, 10, 4, 64, 100, 16, 0, 0, None]
    for i, value, code in ((0, None, -1), (0, fake + 2, -1), (1, 3, -1), (8, None, -1), (9, -1, -1), (10, 0, -1), (11, 48, -2),
                           (12, 0, -1), (13, 17, -1), (14, 3, -3), (15, -1, -3)):
        assert lib.sa_paged_append(*append[:i], value, *append[i + 1:]) == code, i
    attend = [fake, 256, 64, fake, fake, fake, fake, 8, fake, fake, fake, 128, fake, 1 << 40, 4, 10, 4, 1, 64, 100, 16, 8, 5, 128,
              0.125, 0, 1, None]
    for i, value, code in ((0, None, -1), (1, 7, -1), (5, None, -1), (7, 7, -1), (11, 127, -1), (12, None, -4), (12, fake + 8, -4),
                           (13, 100, -4), (14, 0, -1), (15, 0, -1), (16, 0, -1), (17, 3, -1), (18, 48, -2), (19, 0, -1), (20, 12, -1),
                           (21, 7, -1), (22, 11, -1), (22, 0, -1), (23, 129, -1), (24, 0.0, -1), (24, float("nan"), -1), (25, 7, -3),
                           (26, 0, -1)):
        assert lib.sa_paged_attention(*attend[:i], value, *attend[i + 1:]) == code, i
    assert lib.sa_paged_attention_workspace_bytes(4, 10, 4, 3, 64, 5, 128, 0) == -1
    assert lib.sa_paged_attention_workspace_bytes(4, 10, 4, 1, 64, 5, 128, 0) > 0


@pytest.mark.parametrize("attention", ["selective", "selective_x16", "selective_perhead"])
def test_model_serves_requests_of_different_lengths(attention):
    """paged_step's logits after every step are those of each request alone in prefill and decode_step."""
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, n_layers=2, d_model=64, n_heads=4, context_length=64, attention=attention)
    model = SelectiveLM(cfg).double().eval()
    serve(model, "cpu", torch.float64, rtol=1e-4, atol=1e-5)   # (the state between steps is fp32)


def test_the_softmax_slot_has_no_pages():
    cfg = ModelConfig(vocab_size=97, n_layers=1, d_model=64, n_heads=4, context_length=64, attention="softmax")
    with pytest.raises(NotImplementedError, match="paged"):
        SelectiveLM(cfg).new_paged_cache(2, 4, 16)


def test_launches_past_a_grid_are_refused():
    """More workgroups or rows than a launch's first dimension holds (2^32 threads)."""
    lib = _lib.load()
    size = lambda requests, heads, max_len: lib.sa_paged_attention_workspace_bytes(requests, requests, heads, 1, 64, 1, max_len, 0)
    assert size(65535, 16, 4096) > 0 and size(65535, 255, 1024) > 0 and size(65535, 256, 1024) == -1 and size(65535, 16, 1 << 18) == -1
    fake = 1 << 20
    append = [fake, 64, 64, fake, 64, 64, fake, fake, fake, 1 << 23, 64, 64, 100, 16, 0, 0, None]
    assert lib.sa_paged_append(*append) == -1
    kp = torch.zeros(1, 1, 8, 16).expand(1, 256, 8, 16).contiguous()
    table, lengths = torch.zeros(65535, 128, dtype=torch.int32), torch.zeros(65535, dtype=torch.int32)
    with pytest.raises(ValueError, match="too large"):
        paged._check_step(torch.zeros(4, 256, 16), kp, kp, table, lengths, torch.zeros(65536, dtype=torch.int32),
                          torch.zeros(65535, 1, 8), 1, 1, 8)
