"""Histories take the tokens of THIS step from the sampler that has just written them, however early a kernel may start."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draw", ["argmax", "sorted"])
def test_every_step_counts_its_own_token(draw):
    from wick_b200 import ops
    rows, vocab, steps = 48, 3000, 40
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, vocab, (steps, rows), generator=g)
    logits = torch.zeros((steps, rows, vocab))
    logits.scatter_(2, tokens[:, :, None], 50.0)
    logits = logits.cuda()
    seen, counts = torch.zeros((rows, ops.bit_words(vocab)), dtype=torch.int32, device="cuda"), torch.zeros((rows, vocab), dtype=torch.int32, device="cuda")
    at, ids = torch.arange(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    u = torch.rand(rows, device="cuda")
    x, pen = torch.empty((rows, vocab), device="cuda"), torch.tensor([[1.0, 0.25, 0.5]] * rows, device="cuda")

    def step(i):
        ops.steer_logits(logits[i], at, seen=seen, counts=counts, penalties=pen, out=x)
        if draw == "argmax":
            ops.argmax(x, ids)
        else:
            vals, idx = ops.top_k(x, 8)
            ops.pick_sorted(vals, idx, u, 0.5, 0.0, 1.0, ids)
        ops.history_add(seen, counts, ids, at, generated=True)

    want = torch.zeros((rows, vocab), dtype=torch.int64)
    want.scatter_add_(1, tokens.T, torch.ones_like(tokens.T))
    step(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(steps):
            step(i)
    for _ in range(3):
        ops.history_clear(seen, counts, at)
        graph.replay()
        assert torch.equal(counts.cpu().long(), want)
        bits = (seen.cpu()[:, torch.arange(vocab) // 32] >> (torch.arange(vocab) % 32)) & 1
        assert torch.equal(bits.bool(), want > 0)
