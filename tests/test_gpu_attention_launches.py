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


def test_two_threads_on_streams_of_their_own(A):
    """Rotations, appends and attention from two threads at once, in other forms each, give what they give one after the other."""
    import threading

    def work(seed):
        seqs, longest, kv, group, dim = ((4, 1500, 2, 8, 128), (40, 200, 1, 5, 64))[seed]
        g = torch.Generator().manual_seed(seed)
        table = A.RotaryTable(A.rotary_frequencies(dim)[0], layout=("half", "interleaved")[seed])
        _, cache, tables = state(A, seqs, longest, kv, group, dim, 16, seed)
        kept = cache.k.clone(), cache.v.clone()
        qkv = torch.randn((seqs, kv * (group + 2), dim), generator=g).bfloat16().cuda()
        starts = torch.randint(0, longest - 30, (seqs,), generator=g).cuda()

        def steps():
            cache.k.copy_(kept[0]), cache.v.copy_(kept[1])
            positions, got = starts.clone(), []
            for _ in range(25):
                q, k, v = qkv.split([kv * group, kv, kv], dim=1)
                turned = A.cache_append(cache, k, v, tables, positions, q=q, rotary=table)
                positions += 1
                out = A.paged_attention(turned, cache, tables, positions.int())
                got += [turned, out, A.rotary(out, positions, table)]
            return got

        return steps

    both = [work(0), work(1)]
    want = [f() for f in both]
    torch.cuda.synchronize()
    found, failed = [None, None], []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    found[i] = both[i]()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for w, f in zip(want, found):
        assert all(torch.equal(a, b) for a, b in zip(w, f, strict=True))
