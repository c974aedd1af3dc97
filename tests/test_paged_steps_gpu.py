"""Serving steps enqueued one behind the other give the bits of steps with a wait after every call: each call sees what
the one before it wrote, though it may be launched while that still runs. Lengths, tables, pages and queries
change from step to step, requests end and give pages up, and two layers share one workspace."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

STEPS, ROWS, HEADS, KV, DIM, VOCAB, PAGE = 24, 12, 16, 4, 128, 3000, 16


class Steps:
    def __init__(self, torch, rt, width, pages, most):  # noqa: F811
        self.rt, self.width, self.pages = rt, width, pages
        gen = torch.Generator(device="cuda").manual_seed(7)
        rng = np.random.default_rng(width)
        self.tokens = ROWS * most
        self.rope, _ = paged.rope_bits(torch, width * PAGE, DIM)
        self.norms = [(0.1 * torch.randn(DIM, generator=gen, device="cuda")).bfloat16() for _ in range(2)]
        self.qkv = torch.randn(STEPS, 2, self.tokens, (HEADS + 2 * KV) * DIM, generator=gen, device="cuda").bfloat16()
        self.head = torch.randn(STEPS, HEADS * DIM, VOCAB, generator=gen, device="cuda").bfloat16()
        self.u = torch.rand(STEPS, ROWS, generator=gen, device="cuda")
        append = rng.integers(1, most + 1, (STEPS, ROWS))
        append[0] = most
        append[rng.random((STEPS, ROWS)) < 0.1] = -1
        self.append = paged.ints(torch, append)
        self.work = torch.empty(rt.paged_attention_workspace(), dtype=torch.uint8, device="cuda")

    def run(self, torch, stream, wait):  # noqa: F811
        rt, ints = self.rt, lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        lens, counts, start = ints(STEPS + 1, ROWS), ints(STEPS + 1, 4), ints(STEPS, ROWS + 1)
        counts[0, 0] = self.pages
        table, free = ints(ROWS, self.width) - 1, torch.randperm(self.pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        slots, positions, ids = ints(STEPS, self.tokens), ints(STEPS, self.tokens), ints(STEPS, ROWS)
        caches = [[torch.zeros(self.pages, PAGE, KV, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2)]
        q, out = (torch.zeros(STEPS, 2, self.tokens, HEADS * DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        logits = torch.zeros(STEPS, ROWS, VOCAB, device="cuda")
        handles = [rt.PagedCache(k.data_ptr(), v.data_ptr(), 0, self.pages, PAGE, KV, DIM, PAGE * KV * DIM, KV * DIM, DIM) for k, v in caches]
        torch.cuda.synchronize()
        pause = torch.cuda.synchronize if wait else (lambda: None)
        for i in range(STEPS):
            rt.k_paged_plan(lens[i].data_ptr(), self.append[i].data_ptr(), ROWS, PAGE, self.pages, table.data_ptr(), self.width, free.data_ptr(),
                            counts[i].data_ptr(), lens[i + 1].data_ptr(), start[i].data_ptr(), slots[i].data_ptr(), positions[i].data_ptr(),
                            self.tokens, counts[i + 1].data_ptr(), stream)
            pause()
            for layer in range(2):
                rt.k_paged_qkv(handles[layer], self.qkv[i, layer].data_ptr(), (HEADS + 2 * KV) * DIM, self.tokens, HEADS, self.norms[0].data_ptr(),
                               self.norms[1].data_ptr(), 1e-6, self.rope.data_ptr(), self.width * PAGE, positions[i].data_ptr(),
                               slots[i].data_ptr(), q[i, layer].data_ptr(), HEADS * DIM, stream)
                pause()
                rt.k_paged_attention(handles[layer], q[i, layer].data_ptr(), HEADS * DIM, self.tokens, HEADS, table.data_ptr(), self.width,
                                     lens[i + 1].data_ptr(), ROWS, start[i].data_ptr(), self.width * PAGE, 0, DIM ** -0.5,
                                     out[i, layer].data_ptr(), HEADS * DIM, 0, self.work.data_ptr(), self.work.numel(), stream)
                pause()
            rows = out[i, 1, :ROWS].float()
            logits[i] = rows @ self.head[i].float()
            pause()
            rt.k_sample(logits[i].data_ptr(), 2, ROWS, VOCAB, VOCAB, 0, 0, 0, 0, self.u[i].data_ptr(), ids[i].data_ptr(), 0, 0, stream)
            pause()
        torch.cuda.synchronize()
        return [lens, counts, start, slots, positions, table, free, ids, q, out, logits, *caches[0], *caches[1]]


@pytest.mark.parametrize("width,pages,most", [(12, 100, 9), (300, 2000, 3), (8, 40, 6), (64, 600, 40)])
def test_steps_without_waits(torch, pkg, width, pages, most):  # noqa: F811
    steps = Steps(torch, pkg.runtime, width, pages, most)
    want = steps.run(torch, 0, True)
    assert int(want[1][1:, 1].sum()) > 0 and int((want[7] > 0).sum()) > 0
    for _ in range(5):
        for got, w in zip(steps.run(torch, 0, False), want):
            assert torch.equal(got, w)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for got, w in zip(steps.run(torch, side.cuda_stream, False), want):
            assert torch.equal(got, w)
