"""The write into a paged cache against the rotation in 64 bits: every written entry, every other byte as it was."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def order_view(order, pages, heads, page, dim, dtype):
    """Two filled tensors [pages, heads, page, dim] in memory of another order."""
    if order == "heads first":
        k, v = (torch.empty((pages, heads, page, dim), dtype=dtype, device="cuda") for _ in range(2))
    elif order == "slots first":
        k, v = (torch.empty((pages, page, heads, dim), dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        k, v = torch.empty((pages, 2, page, heads, dim + 16), dtype=dtype, device="cuda")[..., :dim].transpose(2, 3).unbind(1)
    for t, x in ((k, 3), (v, 5)):
        t.fill_(x)
    return k, v


def run(A, tokens, heads, kv, dim, rot, layout, page, dtype, order="heads first", table_pages=6, seqs=3, positions=None, rows=None, tables=None, wide=True, magnitude=1.0):
    g = torch.Generator().manual_seed(tokens + dim)
    qkv = torch.randn((tokens, (heads + 2 * kv) * dim), generator=g).bfloat16()
    if positions is None:
        positions = torch.randperm(page * table_pages, generator=g)[:tokens]
        rows = torch.randint(0, seqs, (tokens,), generator=g, dtype=torch.int32)
    pages = seqs * table_pages + 2
    if tables is None:
        tables = torch.randperm(pages, generator=g)[:seqs * table_pages].view(seqs, table_pages).int()
    codes = dtype == "e4m3"
    k0, v0 = order_view(order, pages, kv, page, dim, torch.uint8 if codes else torch.bfloat16)
    scales = [torch.rand(kv, generator=g) * 0.05 + 0.01 for _ in range(2)] if codes else [None, None]
    cache = A.PagedCache(k0, v0, *(s.cuda() if s is not None else None for s in scales))
    before = [k0.clone(), v0.clone()]
    inv, _ = A.rotary_frequencies(rot) if rot else ([], 1.0)
    table = A.RotaryTable(inv, layout=layout, magnitude=magnitude) if rot else None
    q, k, v = (t.view(tokens, -1, dim) for t in qkv.cuda().split([heads * dim, kv * dim, kv * dim], dim=1))
    positions = positions.to(torch.int64 if wide else torch.int32)
    out = A.cache_append(cache, k, v, tables.cuda(), positions.cuda(), rows=rows.cuda() if rows is not None else None, q=q if heads else None, rotary=table)

    qc, kc, vc = (t.view(tokens, -1, dim) for t in qkv.split([heads * dim, kv * dim, kv * dim], dim=1))
    turn = (lambda x: R.rotated(x, positions, inv, layout, magnitude)) if rot else (lambda x: (x.double(), torch.zeros_like(x.double())))
    if heads:
        want, size = turn(qc)
        R.check(out, want, torch.where(size > 0, R.rounding(want, torch.bfloat16) + 1.01 * R.TURN_ERROR * size, 0.0), "q")
    else:
        assert out is None
    got = [t.cpu() for t in (k0, v0)]
    want, untouched = [b.cpu().clone() for b in before], torch.ones((pages, kv, page, dim), dtype=torch.bool)
    share = tokens // tables.shape[0]
    for x, size, i in ((*turn(kc), 0), (vc.double(), torch.zeros(tokens, kv, dim, dtype=torch.float64), 1)):
        for t in range(tokens):
            row, e = int(rows[t]) if rows is not None else t // share, int(positions[t])
            if not 0 <= row < tables.shape[0] or not 0 <= e < page * tables.shape[1] or not 0 <= int(tables[row, e // page]) < pages:
                continue
            at = (int(tables[row, e // page]), slice(None), e % page)
            untouched[at] = False
            if codes:
                y = x[t] / scales[i].double()[:, None]
                # 1 / scale and its product are rounded once each, on top of the turn's error
                error = 2.0**-23 * y.abs() + R.TURN_ERROR * size[t] / scales[i].double()[:, None]
                y = y.clamp(-448, 448)
                R.check(got[i][at].view(R.E4M3), y, R.rounding(y, R.E4M3) + 1.07 * error, f"entry of token {t}")
            else:
                R.check(got[i][at], x[t], torch.where(size[t] > 0, R.rounding(x[t], torch.bfloat16) + 1.01 * R.TURN_ERROR * size[t], 0.0), f"entry of token {t}")
    for i in range(2):
        assert torch.equal(got[i][untouched], want[i][untouched]), "an entry that no token names has changed"
    return cache, k0, v0


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,page", [(1, 8, 2, 128, 128, 16), (5, 4, 4, 64, 64, 7), (70, 6, 2, 80, 32, 24), (33, 3, 1, 96, 26, 16), (40, 0, 3, 128, 64, 64),
                                                          (9, 5, 5, 16, 16, 3), (20, 2, 1, 256, 256, 100), (6, 1, 1, 48, 0, 1), (129, 16, 2, 112, 112, 32)])
def test_append(A, dtype, layout, tokens, heads, kv, dim, rot, page):
    positions = rows = None
    if tokens > 6 * page:  # tokens of one sequence after the other, one entry each
        positions, rows = torch.arange(tokens) % (6 * page), (torch.arange(tokens) // (6 * page)).int()
    run(A, tokens, heads, kv, dim, rot, layout, page, dtype, positions=positions, rows=rows)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("order", ["heads first", "slots first", "both in one"])
def test_orders_of_the_axes(A, dtype, order):
    run(A, 25, 4, 2, 64, 64, "half", 16, dtype, order=order, magnitude=1.5, wide=False)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_padding_and_what_lies_outside_is_left_out(A, dtype):
    """Negative and far positions, rows and pages that do not exist."""
    tables = torch.tensor([[0, 5, -1], [7, 100, 3], [2, 2**31 - 1, 6]], dtype=torch.int32)
    positions = torch.tensor([-1, 0, 8, 15, 16, 23, 24, 10**12, 9, 17, 8, -(2**40)])
    rows = torch.tensor([0, 0, 0, 0, 0, 1, 1, 1, 1, 2, 2, 2], dtype=torch.int32)
    run(A, 12, 4, 2, 64, 64, "half", 8, dtype, table_pages=3, positions=positions, rows=rows, tables=tables)
    rows = torch.tensor([0, -1, 3, 2**31 - 1, -(2**31), 1, 1, 2, 2, 2, 2, 0], dtype=torch.int32)
    positions = torch.arange(12)
    run(A, 12, 4, 2, 64, 32, "interleaved", 8, dtype, table_pages=3, positions=positions, rows=rows, tables=tables)


def test_without_rows_tokens_belong_to_the_sequences_in_turn(A):
    positions = torch.tensor([4, 5, 6, 0, 1, 2, 17, 18, 19])
    run(A, 9, 4, 2, 64, 64, "half", 8, "bf16", table_pages=3, positions=positions)


def test_specials(A):
    """Infinities saturate, NaN stays NaN in an e4m3 cache; both stay what they are in bf16."""
    inv, _ = A.rotary_frequencies(32)
    k = torch.ones((1, 1, 32), dtype=torch.bfloat16, device="cuda")
    v = torch.tensor([float("inf"), float("-inf"), float("nan"), 1e30, -0.0, 449.0, 2.0**-10, 2.0**-11] * 4, dtype=torch.bfloat16, device="cuda").view(1, 1, 32)
    tables, positions = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = A.PagedCache.empty(1, 4, 1, 32, "e4m3")
    A.cache_append(cache, k, v, tables, positions, rotary=A.RotaryTable(inv))
    got = cache.v[0, 0, 0, :8].view(R.E4M3).float().cpu()
    assert got[2].isnan() and got[[0, 1, 3, 4, 5, 6, 7]].tolist() == [448.0, -448.0, 448.0, 0.0, 448.0, 0.0, 0.0]
    cache = A.PagedCache.empty(1, 4, 1, 32)
    A.cache_append(cache, k, v, tables, positions, rotary=A.RotaryTable(inv))
    assert torch.equal(cache.v[0, 0, 0].view(torch.int16), v[0, 0].view(torch.int16))


def test_pages_behind_32_bits(A):
    """Entries whose byte offset in the cache passes 2^32."""
    cache = A.PagedCache.empty(5000, 256, 8, 128, "bf16")  # 2.6 GB of k: 1.3e9 elements
    far = A.PagedCache.empty(9000, 256, 16, 128, "e4m3")  # 4.7 GB, 4.7e9 elements
    for c, page in ((cache, 4999), (far, 8999)):
        k, v = (torch.randn((1, c.kv_heads, 128), device="cuda").bfloat16() for _ in range(2))
        tables = torch.tensor([[0, page]], dtype=torch.int32, device="cuda")
        A.cache_append(c, k, v, tables, torch.tensor([511], device="cuda"))
        want = (v[0].clamp(-448, 448).to(R.E4M3).view(torch.uint8)) if c.dtype == "e4m3" else v[0]
        assert torch.equal(c.v[page, :, 255], want)


def test_captured_with_new_positions(A):
    cache = A.PagedCache.empty(8, 16, 2, 64)
    cache.k.zero_(), cache.v.zero_()
    inv, _ = A.rotary_frequencies(64)
    table = A.RotaryTable(inv)
    k, v, q = (torch.randn((2, n, 64), device="cuda").bfloat16() for n in (2, 2, 4))
    tables, positions = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), torch.tensor([3, 20], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = A.cache_append(cache, k, v, tables, positions, q=q, rotary=table)
    torch.cuda.synchronize()
    assert not cache.k.any()
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, A.rotary(q, positions, table))
        turned = A.rotary(k, positions, table)
        for b in range(2):
            e = int(positions[b])
            assert torch.equal(cache.k[int(tables[b, e // 16]), :, e % 16], turned[b]) and torch.equal(cache.v[int(tables[b, e // 16]), :, e % 16], v[b])
        positions += 1


def test_empty_and_refusals(A):
    from tilefish_b200 import TilefishPreconditionError

    cache = A.PagedCache.empty(4, 16, 2, 64)
    k = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    tables, positions = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.arange(4, device="cuda")
    inv, _ = A.rotary_frequencies(64)
    table = A.RotaryTable(inv)
    assert A.cache_append(cache, k[:0], k[:0], tables, positions[:0], q=k[:0]).shape == (0, 2, 64)

    def refused(kind, *args, **kwargs):
        with pytest.raises(TilefishPreconditionError) as e:
            A.cache_append(*args, **kwargs)
        assert e.value.kind == kind, (e.value.kind, str(e.value))

    refused("dtype", (cache.k, cache.v), k, k, tables, positions)
    refused("shape", cache, k[:, :1], k, tables, positions)
    refused("shape", cache, k, k[:3], tables, positions)
    refused("shape", cache, k[..., :32], k, tables, positions)
    refused("dtype", cache, k.float(), k, tables, positions)
    refused("device", cache, k.cpu(), k, tables, positions)
    refused("shape", cache, k, k, tables, positions[:2])
    refused("dtype", cache, k, k, tables.long(), positions)
    refused("contiguous", cache, k, k, torch.zeros((2, 4), dtype=torch.int32, device="cuda")[:, ::2], positions)
    refused("divisible", cache, k[:3], k[:3], tables, positions[:3])
    refused("shape", cache, k, k, tables, positions, rows=tables[0])
    refused("argument", cache, k, k, tables, positions, q_out=k)
    refused("alias", cache, k, k, tables, positions, q=k, q_out=torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda").expand(4, 2, 64))
    wide = torch.zeros((4, 8, 64), dtype=torch.bfloat16, device="cuda")
    refused("alias", cache, wide[:, 4:6], wide[:, 6:], tables, positions, q=torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda"), q_out=wide[:, 1:5])
    assert A.cache_append(cache, wide[:, 4:6], wide[:, 6:], tables, positions, q=wide[:, :4], q_out=wide[:, :4]) is not None  # columns of one matrix
    refused("shape", cache, k, k, tables, positions, rotary=A.RotaryTable(A.rotary_frequencies(128)[0]))
    refused("alignment", cache, torch.zeros((4, 2, 68), dtype=torch.bfloat16, device="cuda")[..., :64], k, tables, positions)
    refused("pointer_alignment", cache, torch.zeros(4 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 2, 64), k, tables, positions)
    t = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    for kind, args in (("divisible", (t[..., :40], t[..., :40])), ("shape", (t, t[:2])), ("contiguous", (t, t.transpose(1, 2).contiguous().transpose(1, 2))), ("alias", (t, t)),
                       ("alias", (t[:1].expand(4, 2, 16, 64), t[1:2].expand(4, 2, 16, 64))), ("dtype", (t.float(), t.float())), ("dtype", (t, t.view(torch.int16))),
                       ("argument", (t, t.clone(), torch.ones(2, device="cuda"))), ("contiguous", (t.transpose(2, 3), t.clone().transpose(2, 3)))):
        with pytest.raises(TilefishPreconditionError) as e:
            A.PagedCache(*args)
        assert e.value.kind == kind, (kind, e.value.kind, str(e.value))
