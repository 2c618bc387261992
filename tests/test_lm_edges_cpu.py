"""Edges of the operators around the attention layers that need no GPU."""

import socket

import torch

from selective_attention import _lib
from selective_attention.model import ModelConfig, SelectiveLM

A = 1 << 20   # an aligned address that nothing reads


def test_rows_of_probabilities_stay_within_a_tiles_offsets():
    """A piece of the vocabulary has as many words as a row of 2^22 bytes holds, however few the tokens: a tile's 256 rows of probabilities
    are then within 2^30 bytes. (The workspace: two pieces of one token's, in fp16 of two rows each, and 64 parts of its fp32 sums of dX at the most.)"""
    lib = _lib.load()
    for dtype in (1, 2):
        for vocab in (1 << 26, 1 << 27, (1 << 28) - 1):
            size = lib.sa_linear_xent_backward_workspace_bytes(A, 64, 1, vocab, 64, 1, 1, dtype, dtype)
            rows = 2 if dtype == 2 else 1
            assert 0 < size < rows * (2 * (1 << 22) + 64 * 64 * 4) + (1 << 16), (dtype, vocab, size)


class _Step(torch.nn.Module):
    """What a data-parallel wrapper wraps: a module whose forward is the model's loss."""

    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, idx, targets):
        return self.model.loss(idx, targets)


def _model_and_batch():
    torch.manual_seed(4)
    model = SelectiveLM(ModelConfig(vocab_size=61, n_layers=1, d_model=32, n_heads=2, context_length=40, attention="softmax"))
    return model, torch.randint(61, (4, 24)), torch.randint(61, (4, 24))


def _rank(rank, port, results):
    torch.set_num_threads(1)
    torch.distributed.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    model, idx, targets = _model_and_batch()
    step = torch.nn.parallel.DistributedDataParallel(_Step(model))
    step(idx[2 * rank:2 * rank + 2], targets[2 * rank:2 * rank + 2]).backward()
    results.put((rank, [p.grad.numpy() for p in model.parameters()]))
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


def test_loss_under_a_data_parallel_wrapper():
    """Two ranks with half of the batch each have the whole batch's gradients, through a module that calls `loss` in its forward."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = torch.multiprocessing.get_context("spawn")
    results = ctx.Queue()
    ranks = [ctx.Process(target=_rank, args=(r, port, results)) for r in range(2)]
    for p in ranks:
        p.start()
    got = dict(results.get(timeout=120) for _ in ranks)
    for p in ranks:
        p.join(60)
        assert p.exitcode == 0
    model, idx, targets = _model_and_batch()
    want = torch.autograd.grad(model.loss(idx, targets), tuple(model.parameters()))
    for grads in got.values():
        for a, b in zip(grads, want):
            torch.testing.assert_close(torch.from_numpy(a), b, rtol=1e-4, atol=1e-6)
