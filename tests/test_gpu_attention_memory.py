"""What the attention operators write shares no memory with what else they use: refusals, and what is taken although it lies close by."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def refused(call, *args, **kwargs):
    from tilefish_b200 import TilefishPreconditionError

    with pytest.raises(TilefishPreconditionError) as e:
        call(*args, **kwargs)
    assert e.value.kind == "alias", (e.value.kind, str(e.value))


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16, device="cuda")


def test_a_cache_whose_keys_and_values_share_memory_is_refused(A):
    t = bf16(9, 2, 16, 64)
    refused(A.PagedCache, t[:8], t[1:])
    refused(A.PagedCache, t[:4], t[3:7])
    A.PagedCache(t[:4], t[4:8])
    A.PagedCache(t[::2][:4], t[1::2])
    both = bf16(4, 16, 2, 2, 64)  # slot, key or value, head
    A.PagedCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2))


def test_append_refuses_a_result_in_the_cache(A):
    cache = A.PagedCache(bf16(4, 2, 16, 64), bf16(4, 2, 16, 64))
    k, q = bf16(4, 2, 64), bf16(4, 2, 64)
    tables, positions = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.arange(4, device="cuda")
    for t in (cache.k, cache.v):
        refused(A.cache_append, cache, k, k, tables, positions, q=q, q_out=t[0, :, :4].transpose(0, 1))
        refused(A.cache_append, cache, k, k, tables, positions, q=t[0, :, :4].transpose(0, 1), q_out=t[0, :, :4].transpose(0, 1))
    refused(A.cache_append, cache, k, k, tables, positions, q=q, q_out=torch.as_strided(bf16(5, 64), (4, 2, 64), (64, 32, 1)))


def test_entries_move_within_a_cache(A):
    cache = A.PagedCache.empty(4, 16, 2, 64)
    cache.k.normal_(), cache.v.normal_()
    k, v = cache.k[3].clone(), cache.v[3].clone()
    kept = cache.k[:1].clone()
    tables = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")
    A.cache_append(cache, cache.k[3].transpose(0, 1), cache.v[3].transpose(0, 1), tables, torch.arange(16, 32, device="cuda"))
    assert torch.equal(cache.k[2], k) and torch.equal(cache.v[2], v) and torch.equal(cache.k[3], k) and torch.equal(cache.k[:1], kept)


def test_rotary_refuses_results_that_overlap_themselves(A):
    table = A.RotaryTable(A.rotary_frequencies(64)[0])
    x, positions = bf16(4, 2, 64), torch.arange(4, device="cuda")
    windows = torch.as_strided(bf16(9, 64), (4, 2, 64), (64, 64, 1))
    refused(A.rotary, x, positions, table, out=windows)
    refused(A.rotary, windows, positions, table, out=windows)
    windows.normal_()
    assert torch.equal(A.rotary(windows, positions, table), A.rotary(windows.contiguous(), positions, table))
    both = torch.randn((2, 2, 4, 64), device="cuda").bfloat16()  # heads outermost, x and out in turn
    want = A.rotary(both[:, 0].transpose(0, 1), positions, table)
    A.rotary(both[:, 0].transpose(0, 1), positions, table, out=both[:, 1].transpose(0, 1))
    assert torch.equal(both[:, 1].transpose(0, 1), want)


def test_attention_refuses_results_and_workspaces_in_what_it_reads(A):
    g = torch.Generator().manual_seed(0)
    cache = A.PagedCache.empty(8, 16, 2, 64)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, generator=g).bfloat16())
    q = torch.randn((2, 4, 64), generator=g).bfloat16().cuda()
    tables, lengths = torch.randperm(8, generator=g).view(2, 4).int().cuda(), torch.tensor([60, 33], dtype=torch.int32, device="cuda")
    need = A.attention_workspace_bytes(cache, 2, 1, 4, 4)
    want = A.paged_attention(q, cache, tables, lengths, return_lse=True)
    for t in (cache.k, cache.v):
        refused(A.paged_attention, q, cache, tables, lengths, out=t[:1].view(8, 4, 64)[:2])
        refused(A.paged_attention, q, cache, tables, lengths, lse=t.view(torch.float32).flatten()[:8].view(2, 4))
    store = torch.zeros(need + 8 * 2 * 16 * 64 * 4, dtype=torch.uint8, device="cuda")
    k, v = (store[i:i + 8 * 2 * 16 * 64 * 2].view(torch.bfloat16).view(8, 2, 16, 64) for i in (need - 32, need - 32 + 8 * 2 * 16 * 64 * 2))
    refused(A.paged_attention, q, A.PagedCache(k, v), tables, lengths, workspace=store)
    out = torch.empty_like(q)
    refused(A.paged_attention, q, cache, tables, lengths, out=out, lse=out.view(torch.float32).flatten()[:8].view(2, 4))
    refused(A.paged_attention, q, cache, tables, lengths, lse=q.view(torch.float32).flatten()[:8].view(2, 4))
    arena = torch.empty(4096 + need, dtype=torch.uint8, device="cuda")
    inside = arena[2048:2048 + 2 * 4 * 64 * 2].view(torch.bfloat16).view(2, 4, 64)
    refused(A.paged_attention, q, cache, tables, lengths, workspace=arena, out=inside)
    refused(A.paged_attention, inside.copy_(q), cache, tables, lengths, workspace=arena)
    refused(A.paged_attention, q, cache, tables, lengths, workspace=arena, lse=arena[:32].view(torch.float32).view(2, 4))
    for name, t in (("tables", tables), ("lengths", lengths)):
        there = arena[:t.numel() * 4].view(torch.int32).view(t.shape).copy_(t)
        refused(A.paged_attention, q, cache, *(there if n == name else x for n, x in (("tables", tables), ("lengths", lengths))), workspace=arena)
    there = arena[:8].view(torch.int32).fill_(1)
    refused(A.paged_attention, q, cache, tables, lengths, counts=there, workspace=arena)
    # behind the bytes that the call needs the rest of a workspace is the caller's
    behind = arena[-4096:]
    out, lse = behind[:1024].view(torch.bfloat16).view(2, 4, 64), behind[1024:1056].view(torch.float32).view(2, 4)
    assert (need % 16) == 0
    got = A.paged_attention(q, cache, tables, lengths, workspace=arena, out=out, lse=lse)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    R.check_attention(*got, R.attention(q, cache.k, cache.v, tables, lengths))
