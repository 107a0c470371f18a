"""Rotations and appends large enough for the forms that long calls take: two rows of a head to a thread, several blocks to an SM, loops over the grid."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def tokens_for(heads, dim, more=1.0):
    """As many tokens as two blocks of two rows a thread on every SM do not hold, times ``more``; the last block is part empty where the number of
    heads allows it."""
    lanes = 1
    while lanes < dim // 16:
        lanes *= 2
    rows = 2 * (256 // lanes)  # of a block
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tokens = int(2 * rows * sms * more) // heads + 1
    return tokens + (tokens * heads % rows == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,dim,rot,layout", [(1, 128, 128, "half"), (7, 128, 64, "half"), (40, 64, 64, "half"), (3, 96, 48, "half"), (5, 256, 256, "half"), (2, 1024, 512, "half"),
                                                  (1, 16, 16, "half"), (64, 128, 128, "interleaved"), (3, 80, 32, "interleaved"), (9, 64, 26, "interleaved"), (1, 48, 46, "interleaved"),
                                                  (6, 64, 46, "half"), (1, 112, 26, "half")])
@pytest.mark.parametrize("inverse", [False, True])
def test_long_rotations(A, dtype, heads, dim, rot, layout, inverse):
    tokens = tokens_for(heads, dim)
    g = torch.Generator(device="cuda").manual_seed(heads + dim)
    wide = torch.empty((tokens, heads + 1, dim), dtype=dtype, device="cuda").normal_(generator=g)
    x, positions = wide[:, :heads], torch.randint(-5000, 200000, (tokens,), generator=g, device="cuda")
    inv, _ = A.rotary_frequencies(rot)
    table = A.RotaryTable(inv, layout=layout, magnitude=1.25)
    out = A.rotary(x, positions, table, inverse=inverse)
    before, last = x.clone(), wide[:, heads:].clone()
    want, size = R.rotated(x, positions, inv, layout, 1.25, inverse)
    # the oracle's angle is a product in 64 bits: off by half a step of it
    error = (R.TURN_ERROR + 200000 * 2.0**-53) * size
    R.check(out, want, torch.where(size > 0, R.rounding(want, dtype) + 1.01 * error, 0.0), "rotary")
    assert torch.equal(x, before)
    A.rotary(x, positions, table, out=x, inverse=inverse)
    assert torch.equal(x, out) and torch.equal(wide[:, heads:], last)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_long_rotations_of_any_alignment(A, dtype, layout):
    """Single pairs, more than the grid takes in one pass."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    heads, dim, rot = 3, 100, 50
    tokens = 8 * sms * 256 * 5 // 2 // (heads * (dim - rot // 2)) + 1
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(tokens * heads * dim + 1, dtype=dtype, device="cuda").normal_(generator=g)[1:].view(tokens, heads, dim)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") * 3
    inv, _ = A.rotary_frequencies(rot)
    table = A.RotaryTable(inv, layout=layout)
    out = A.rotary(x, positions, table)
    want, size = R.rotated(x, positions, inv, layout)
    R.check(out, want, torch.where(size > 0, R.rounding(want, dtype) + 1.01 * R.TURN_ERROR * size, 0.0), "rotary")
    assert A.rotary(x, positions, table, out=x) is x and torch.equal(x, out)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("q_heads,kv,dim,rot,layout,page", [(8, 2, 128, 128, "half", 16), (0, 1, 64, 32, "half", 24), (5, 3, 80, 80, "interleaved", 7), (3, 1, 256, 128, "half", 64),
                                                            (2, 1, 16, 16, "interleaved", 32), (1, 1, 96, 0, "half", 16), (4, 2, 64, 46, "half", 16)])
def test_long_appends(A, dtype, q_heads, kv, dim, rot, layout, page):
    """Prompts of several sequences with padding, far positions, and rows and pages that do not exist between their tokens."""
    tokens, seqs = tokens_for(q_heads + 2 * kv, dim), 5
    each = -(-tokens // seqs)
    width = -(-each // page)
    pages = seqs * width + 2
    g = torch.Generator().manual_seed(dim + page)
    qkv = torch.randn((tokens, q_heads + 2 * kv, dim), generator=g).bfloat16()
    tables = torch.randperm(pages, generator=g)[:seqs * width].view(seqs, width).int()
    tables[1, 0], tables[2, width - 1] = -1, pages
    rows, positions = (torch.arange(tokens) // each).int(), torch.arange(tokens) % each
    odd = torch.randperm(tokens, generator=g)[:40]
    positions[odd[:10]], positions[odd[10:20]] = -1 - torch.arange(10), width * page + torch.arange(10)
    rows[odd[20:30]], rows[odd[30:]] = -1, seqs
    codes = dtype == "e4m3"
    scales = [torch.rand(kv, generator=g) * 0.05 + 0.01 for _ in range(2)] if codes else [None, None]
    cache = A.PagedCache.empty(pages, page, kv, dim, dtype, k_scale=scales[0].cuda() if codes else None, v_scale=scales[1].cuda() if codes else None)
    for t in (cache.k, cache.v):
        t.fill_(7)
    inv, _ = A.rotary_frequencies(rot) if rot else ([], 1.0)
    gpu = qkv.cuda()
    q, k, v = gpu.split([q_heads, kv, kv], dim=1)
    out = A.cache_append(cache, k, v, tables.cuda(), positions.cuda(), rows=rows.cuda(), q=q if q_heads else None, rotary=A.RotaryTable(inv, layout=layout) if rot else None)
    turn = (lambda x: R.rotated(x, positions, inv, layout)) if rot else (lambda x: (x.double(), torch.zeros_like(x.double())))
    if q_heads:
        want, size = turn(qkv[:, :q_heads])
        R.check(out, want, torch.where(size > 0, R.rounding(want, torch.bfloat16) + 1.01 * R.TURN_ERROR * size, 0.0), "q")
    inside = (positions >= 0) & (positions < width * page) & (rows >= 0) & (rows < seqs)
    page_of = tables[rows.clamp(0, seqs - 1).long(), positions.clamp(0, width * page - 1) // page].long()
    inside &= (page_of >= 0) & (page_of < pages)
    assert 0 < int(inside.sum()) < tokens
    at = page_of[inside], positions[inside] % page
    for name, got, (x, size), scale in (("k", cache.k.cpu(), turn(qkv[:, q_heads:q_heads + kv]), scales[0]), ("v", cache.v.cpu(), (qkv[:, q_heads + kv:].double(), torch.zeros(1).double()), scales[1])):
        untouched = torch.ones((pages, page), dtype=torch.bool)
        untouched[at] = False
        assert (got.transpose(1, 2)[untouched] == 7).all(), name
        x, size = x[inside], size.expand(x.shape)[inside]
        entries = got.transpose(1, 2)[at]
        if codes:
            y = x / scale.double()[:, None]
            # 1 / scale and its product are rounded once each, on top of the turn's error
            error = 2.0**-23 * y.abs() + R.TURN_ERROR * size / scale.double()[:, None]
            y = y.clamp(-448, 448)
            R.check(entries.view(R.E4M3), y, R.rounding(y, R.E4M3) + 1.07 * error, name)
        else:
            R.check(entries, x, torch.where(size > 0, R.rounding(x, torch.bfloat16) + 1.01 * R.TURN_ERROR * size, 0.0), name)
