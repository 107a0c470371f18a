"""Paged attention with more sequences, row tiles and parts than the other tests have: the search for a worker's place in a long list, joins of more items than blocks,
prompts, and splits that follow the lengths."""

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def run(A, lengths, queries, kv, group, dim, page, dtype, counts=None, window=0, seed=0):
    g = torch.Generator().manual_seed(seed + dim + queries)
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + 1, max(1, max(need))
    order = torch.randperm(pages, generator=g).int()
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv, page, dim)
    k, v = (torch.randn(shape, generator=g) for _ in range(2))
    scales = [None, None]
    if dtype == "e4m3":
        scales = [(torch.rand(kv, generator=g) + 0.5) / 20.0 for _ in range(2)]
        k, v = ((t * 20).to(R.E4M3).view(torch.uint8) for t in (k, v))
    else:
        k, v = k.bfloat16(), v.bfloat16()
    cache = A.PagedCache(k.cuda(), v.cuda(), *(s.cuda() if s is not None else None for s in scales))
    q = (torch.randn((len(lengths) * queries, kv * group, dim), generator=g) * 2).bfloat16()
    lengths = torch.tensor(lengths, dtype=torch.int32)
    ws = torch.full((A.attention_workspace_bytes(cache, len(lengths), queries, kv * group, width),), 0xFF, dtype=torch.uint8, device="cuda")
    out, lse = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), counts=counts.cuda() if counts is not None else None, window=window, return_lse=True, workspace=ws)
    R.check_attention(out, lse, R.attention(q, cache.k, cache.v, tables, lengths, counts, None, window, *scales))
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("seqs,kv,dim", [(1023, 1, 32), (1024, 1, 32), (1025, 2, 64), (1100, 1, 128), (4500, 1, 128), (2100, 2, 256)])
def test_more_sequences_than_the_lanes_look_at_once(A, dtype, seqs, kv, dim):
    """Short ones, many of them empty, runs of empty ones at the beginning and the end, and a few long ones that many workers share."""
    g = torch.Generator().manual_seed(seqs)
    lengths = torch.randint(0, 24, (seqs,), generator=g)
    lengths[torch.rand(seqs, generator=g) < 0.2] = 0
    lengths[:70] = 0
    lengths[-90:] = 0
    for i, n in ((100, 4000), (seqs // 2, 777), (seqs - 91, 2500)):
        lengths[i] = n
    out, lse = run(A, lengths.tolist(), 1, kv, 2, dim, 16, dtype)
    assert not out[:70].any() and (lse[-90:] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_joins_of_more_items_than_blocks(A, dtype):
    """64 rows of some 80 heads that seven workers share each: four warps to an item (an eight of rows and 32 elements), and more items than 16 blocks an SM."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    seqs = sms // 16 + 1
    assert seqs * 8 * 8 * 4 > 16 * sms
    run(A, [1900 + 13 * i for i in range(seqs)], 8, 8, 8, 128, 32, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("queries,kv,group,dim,context", [(65, 1, 1, 64, 0), (128, 2, 4, 128, 0), (200, 1, 8, 64, 150), (129, 2, 1, 256, 40), (300, 1, 3, 96, 7), (100, 1, 13, 32, 0)])
@pytest.mark.parametrize("window", [0, 70])
def test_prompts(A, dtype, queries, kv, group, dim, context, window):
    """More than 64 new tokens a sequence, on top of a context, with one that is shorter than its queries and one that is empty."""
    run(A, [queries + context, queries + context // 2, max(1, queries - 9), 0], queries, kv, group, dim, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_prompts_of_their_own_lengths(A, dtype):
    """Counts leave whole row tiles without a query."""
    counts = torch.tensor([190, 1, 0, 65, 128, 7], dtype=torch.int32)
    out, lse = run(A, [190, 300, 50, 65, 400, 7], 190, 2, 4, 64, 16, dtype, counts=counts, window=0)
    for b, n in enumerate(counts.tolist()):
        assert not out[b * 190 + n:(b + 1) * 190].any() and (lse[b * 190 + n:(b + 1) * 190] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_more_row_tiles_than_the_lanes_look_at_once(A, dtype):
    """Prompts of 60 sequences in 1500 row tiles."""
    run(A, [200] * 20 + [37] * 20 + [3] * 20, 200, 1, 8, 32, 16, dtype, counts=torch.tensor([200] * 20 + [37] * 20 + [3] * 20, dtype=torch.int32))


@pytest.mark.parametrize("setting", [0, 1])
@pytest.mark.parametrize("margin", [0, 16])
def test_launch_settings_change_no_result(A, setting, margin):
    """Appends, rotations and attention behind one another, as plain launches and as dependents, beside a margin of SMs or not."""
    from tilefish_b200 import _native as N

    lib = N.load()
    g = torch.Generator().manual_seed(4)
    table = A.RotaryTable(A.rotary_frequencies(64)[0])
    tables = torch.randperm(48, generator=g).view(3, 16).int().cuda()
    steps = [torch.randn((3 * n, 12, 64), generator=g).bfloat16().cuda() for n in (30, 1, 1, 4, 1, 90, 1)]

    def chain():
        cache = A.PagedCache.empty(48, 16, 2, 64)
        cache.k.zero_(), cache.v.zero_()
        lengths, got = torch.zeros(3, dtype=torch.int32, device="cuda"), []
        for x in steps:
            n = x.shape[0] // 3
            positions = (lengths.long()[:, None] + torch.arange(n, device="cuda")).flatten()
            lengths += n
            q, k, v = x.split([8, 2, 2], dim=1)
            turned = A.cache_append(cache, k, v, tables, positions, q=q, rotary=table)
            out, lse = A.paged_attention(turned, cache, tables, lengths, return_lse=True)
            back = A.rotary(turned, positions, table, inverse=True)
            got += [turned, out, lse, back, A.rotary(back, positions, table)]
        torch.cuda.synchronize()
        return got + [cache.k, cache.v]

    want = chain()
    try:
        N.check(lib.tf_set_programmatic_launch(setting), "tf_set_programmatic_launch")
        N.check(lib.tf_set_sm_margin(margin), "tf_set_sm_margin")
        eager = chain()
    finally:
        N.check(lib.tf_set_programmatic_launch(-1), "tf_set_programmatic_launch")
        N.check(lib.tf_set_sm_margin(0), "tf_set_sm_margin")
    for i, (a, b) in enumerate(zip(want, eager)):
        assert torch.equal(a, b), i
