"""Attention over a paged cache right behind kernels that write what it reads."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def state(A, seqs, longest, kv, group, dim, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    width = -(-longest // page)
    cache = A.PagedCache.empty(seqs * width, page, kv, dim)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, generator=g).bfloat16())
    tables = torch.randperm(seqs * width, generator=g).view(seqs, width).int().cuda()
    q = torch.randn((seqs * 2, kv * group, dim), generator=g).bfloat16().cuda()
    return q, cache, tables


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("seqs,longest,kv,group", [(1, 6000, 1, 4), (6, 3000, 2, 4), (200, 120, 2, 1)])  # few heads in many parts, some, many in one
def test_lengths_and_counts_written_directly_in_front(A, captured, seqs, longest, kv, group):
    """Lengths and counts change by a kernel directly in front of the call, call after call, where the call before has read the old ones. The results are those of
    calls with the device idle in front of each."""
    q, cache, tables = state(A, seqs, longest, kv, group, 64, 16)
    steps = 8
    start = torch.randint(0, longest // 2, (seqs,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    step = (torch.arange(seqs, device="cuda", dtype=torch.int32) % 5 - 1) * (longest // 20)
    counts0 = (torch.arange(seqs, device="cuda", dtype=torch.int32) % 3)
    want, lengths, counts = [], start.clone(), counts0.clone()
    for _ in range(steps):
        lengths += step
        counts.copy_(2 - counts)
        torch.cuda.synchronize()
        want.append(A.paged_attention(q, cache, tables, lengths, counts=counts, return_lse=True))
        torch.cuda.synchronize()
    lengths, counts = start.clone(), counts0.clone()

    def all_steps():
        got = []
        for _ in range(steps):
            counts.neg_().add_(2)
            lengths.add_(step)
            got.append(A.paged_attention(q, cache, tables, lengths, counts=counts, return_lse=True))
        return got

    torch.cuda.synchronize()
    if captured:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = all_steps()
            graph.replay()
    else:
        got = all_steps()
    torch.cuda.synchronize()
    for i, (w, g) in enumerate(zip(want, got)):
        assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1]), i
