"""What the multiplications of paged attention keep of softmax weights and queries, where the result's own rounding does not hide it."""

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


def one_sequence(A, k, v, dtype):
    """A cache of one sequence with keys and values [entries, dim], in pages of 16."""
    n, dim = k.shape
    pages = -(-n // 16)
    caches = []
    for x in (k, v):
        t = torch.zeros((pages * 16, dim))
        t[:n] = x
        t = t.view(pages, 1, 16, dim)
        caches.append((t.to(R.E4M3).view(torch.uint8) if dtype == "e4m3" else t.bfloat16()).cuda())
    return A.PagedCache(*caches), torch.arange(pages, dtype=torch.int32).view(1, pages), torch.tensor([n], dtype=torch.int32)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("entries,group", [(2, 8), (33, 3), (333, 8), (333, 40), (5000, 8), (5000, 1)])
def test_weights_of_16_bits_for_a_bf16_cache(A, dim, entries, group):
    """Values of plus and minus one whose weighted sum nearly cancels: what the weights lose is as large as the result's own rounding, or larger."""
    g = torch.Generator().manual_seed(entries + dim)
    k = torch.randn((entries, dim), generator=g).bfloat16().float() * 0.25
    v = torch.ones((entries, dim))
    v[1::2] = -1.0
    q = (torch.randn((1, group, dim), generator=g) * 0.5).bfloat16()
    cache, tables, lengths = one_sequence(A, k, v, "bf16")
    out = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda())
    want, _, _, _ = R.attention(q, cache.k, cache.v, tables, lengths)
    s = q[0].double() @ cache.k.double().cpu().view(-1, dim)[:entries].T * dim**-0.5
    ds = (dim + 6) * 2.0**-24 * dim**-0.5 * (q[0].double().abs() @ cache.k.double().cpu().view(-1, dim)[:entries].abs().T).amax(-1)
    # two bf16 terms: each keeps half a step, 2^-8, of what is left; twice the score's error; exp2's two steps; additions as in the reference; sum w |v| is 1
    bound = 2.0**-16 + 2 * ds + 2.0**-22 + (entries / 8 + 64) * 2.0**-24
    got = out.double().cpu()[0]
    off = (got - want[0]).abs()
    assert (off <= bound[:, None] + R.rounding(want[0], torch.bfloat16) * (1 + 2.0**-8)).all()
    if entries == 2:  # weights of 11 bits would not do: the same sum with f16 weights leaves the bound in some row
        w = torch.exp(s - s.amax(-1, keepdim=True))
        half = (w.half().double() * v[:, 0].double()).sum(-1) / w.sum(-1)
        assert ((half - want[0, :, 0]).abs() > bound).any()


def test_a_weight_that_differs_in_its_thirteenth_bit(A):
    """Two keys whose weights are 1 and 1 - 2^-13, values 1 and -1: the result is that difference alone."""
    dim = 64
    k = torch.zeros((2, dim))
    k[1, 0] = 1.0
    v = torch.ones((2, dim))
    v[1] = -1.0
    q = torch.zeros((1, 1, dim)).bfloat16()
    q[0, 0, 0] = -(2.0**-13)
    cache, tables, lengths = one_sequence(A, k, v, "bf16")
    out = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), scale=1.0).double().cpu()
    want = math.tanh(2.0**-14)
    assert ((out - want).abs() <= 2.0**-17 + 2.0**-22).all()  # 16 bits of one weight in a sum of two: half of 2^-16


@pytest.mark.parametrize("group", [1, 8, 20, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("below,counts", [(20, True), (31, True), (40, False)])
def test_small_elements_of_queries_over_an_e4m3_cache(A, group, dim, below, counts):
    """One element of a query is far above the others and meets keys of zero: the scores come from elements 2^-below of it, exact down to 2^-31 and zero below 2^-39."""
    g = torch.Generator().manual_seed(below)
    n = 70
    k = torch.randn((n, dim), generator=g).to(R.E4M3).float()
    k[:, 5] = 0.0
    v = torch.randn((n, dim), generator=g).to(R.E4M3).float()
    small = 1.0 + torch.randint(0, 128, (1, group, dim), generator=g) / 128.0  # eight bits, in [1, 2)
    q = (small * torch.where(torch.rand((1, group, dim), generator=g) < 0.5, -1.0, 1.0)).bfloat16()
    q[:, :, 5] = 2.0**below * 1.0
    scale = 0.25 * dim**-0.5
    cache, tables, lengths = one_sequence(A, k, v, "e4m3")
    out = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), scale=scale)
    seen = q.clone()
    seen[:, :, 5] = 0  # it meets zeros only, and would swell the bound
    if not counts:
        seen.zero_()
    ref = R.attention(seen, cache.k, cache.v, tables, lengths, scale=scale)
    R.check_attention(out, None, ref)
    apart = R.attention(q, cache.k, cache.v, tables, lengths, scale=scale)[0]
    assert counts == bool(((apart - ref[0]).abs().amax(-1) < 1e-9).all())
