"""Attention over a paged cache against the formula in 64 bits: lengths, head layouts, windows, padding, what is not seen, and its refusals."""

import math

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

NAN8 = 0x7F


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def setup(A, lengths, queries, kv, group, dim, page, dtype, order="heads first", seed=0, stale="nan", peak=2.0, width=None, scales=True):
    """q, a cache whose entries that nobody sees are NaN, tables and lengths. Pages lie anywhere, those behind a length do not exist."""
    g = torch.Generator().manual_seed(seed + 31 * dim + queries)
    need = [-(-max(0, n) // page) for n in lengths]
    width = width or max(1, max(need))
    pages = sum(need) + 2
    perm = torch.randperm(pages, generator=g).int()
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    tables[:, 0] = 2**30
    codes = dtype == "e4m3"
    shape = (pages, kv, page, dim)
    if order == "heads first":
        k, v = (torch.empty(shape, dtype=torch.bfloat16) for _ in range(2))
    elif order == "slots first":
        k, v = (torch.empty((pages, page, kv, dim), dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    else:
        k, v = torch.empty((pages, 2, page, kv, dim), dtype=torch.bfloat16).transpose(2, 3).unbind(1)
    at = 0
    k.fill_(math.nan if stale == "nan" else 1.0), v.fill_(math.nan if stale == "nan" else 1.0)
    for b, (n, x) in enumerate(zip(lengths, need)):
        tables[b, :x] = perm[at:at + x]
        at += x
        for j in range(x):
            many = min(page, n - j * page)
            for t in (k, v):
                t[int(tables[b, j]), :, :many] = torch.randn((kv, many, dim), generator=g).bfloat16()
    k_scale = v_scale = None
    if codes:
        spread = 20.0 if scales else 1.0
        strides = k.stride()
        k, v = ((t.float() * spread).to(R.E4M3).view(torch.uint8) for t in (k, v))
        assert k.stride() == strides or order != "heads first"
        if scales:
            k_scale, v_scale = ((torch.rand(kv, generator=g) + 0.5) / spread for _ in range(2))
    q = (torch.randn((len(lengths) * queries, kv * group, dim), generator=g) * peak).bfloat16()
    to = lambda t: t.cuda() if t is not None else None  # noqa: E731
    kc, vc = torch.empty_strided(k.shape, k.stride(), dtype=k.dtype, device="cuda").copy_(k), torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda").copy_(v)
    if order == "both in one":
        both = torch.empty((pages, 2, page, kv, dim), dtype=k.dtype, device="cuda").transpose(2, 3)
        kc, vc = both.unbind(1)
        kc.copy_(k), vc.copy_(v)
    cache = A.PagedCache(kc, vc, to(k_scale), to(v_scale))
    return q, cache, tables, torch.tensor(lengths, dtype=torch.int32)


def run(A, q, cache, tables, lengths, **kwargs):
    counts = kwargs.pop("counts", None)
    need = A.attention_workspace_bytes(cache, len(lengths), q.shape[0] // len(lengths), q.shape[1], tables.shape[1])
    workspace = torch.full((max(16, need),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN: what the call did not write shows
    out, lse = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), counts=counts.cuda() if counts is not None else None, return_lse=True,
                                 workspace=workspace, **kwargs)
    R.check_attention(out, lse, R.attention(q, cache.k, cache.v, tables, lengths, counts, kwargs.get("scale"), kwargs.get("window", 0), cache.k_scale, cache.v_scale))
    return out, lse


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 128, 144, 192, 256])
def test_head_dims(A, dtype, dim):
    run(A, *setup(A, [0, 1, 17, 65, 130], 1, 2, 4, dim, 16, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("kv,group,queries", [(1, 1, 1), (3, 1, 1), (8, 8, 1), (2, 16, 1), (1, 17, 1), (2, 5, 2), (1, 8, 4), (1, 8, 5), (2, 16, 4), (1, 13, 5), (1, 32, 4), (1, 3, 64), (4, 1, 16),
                                              (1, 71, 1), (1, 130, 1)])
def test_heads_and_queries(A, dtype, kv, group, queries):
    run(A, *setup(A, LENGTHS[::2] if queries < 10 else [0, 5, 64, 70, 100], queries, kv, group, 64, 16, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [48, 96, 128, 240])
@pytest.mark.parametrize("group,queries", [(8, 1), (3, 5), (8, 3), (8, 4), (8, 5), (16, 3), (7, 9), (13, 10)])
def test_every_number_of_rows(A, dtype, dim, group, queries):
    """8 to 130 rows of a kv head in every head size's kernels, with sequences that several workers share, empty ones and padding."""
    q, cache, tables, lengths = setup(A, [400, 0, 33, 2, 90], queries, 2, group, dim, 16 if group % 2 else 48, dtype)
    run(A, q, cache, tables, lengths)
    run(A, q, cache, tables, lengths, counts=torch.tensor([queries, 1, queries - 1, queries, 1], dtype=torch.int32), window=50)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 100, 1000])
def test_page_sizes(A, dtype, page):
    run(A, *setup(A, LENGTHS, 2, 2, 3, 64, page, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("order", ["heads first", "slots first", "both in one"])
def test_orders_of_the_axes(A, dtype, order):
    run(A, *setup(A, [40, 0, 129, 7], 1, 4, 2, 128, 16, dtype, order=order))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 1000])
@pytest.mark.parametrize("queries", [1, 6])
def test_windows(A, dtype, window, queries):
    run(A, *setup(A, LENGTHS, queries, 2, 4, 64, 16, dtype), window=window)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [0, 20])
def test_counts_pad_a_batch(A, dtype, window):
    q, cache, tables, lengths = setup(A, [50, 50, 50, 3, 0, 64, 65, 128], 5, 2, 4, 64, 16, dtype)
    counts = torch.tensor([5, 0, 1, 5, 2, 4, 9, -3], dtype=torch.int32)
    q[1 * 5:2 * 5] = math.nan  # what pads may hold anything
    out, lse = run(A, q, cache, tables, lengths, counts=counts, window=window)
    assert not out[5:10].any() and (lse[5:10] == -math.inf).all() and not out[2 * 5 + 1:3 * 5].any()


@pytest.mark.parametrize("dtype,dim,length", [("bf16", 128, 5000), ("e4m3", 128, 5001), ("bf16", 256, 3333), ("e4m3", 64, 9000), ("bf16", 64, 12345)])
@pytest.mark.parametrize("queries,kv,group", [(1, 1, 8), (3, 2, 8), (1, 4, 1)])
def test_long_sequences_are_split_and_joined(A, dtype, dim, length, queries, kv, group):
    q, cache, tables, lengths = setup(A, [length, 3], queries, kv, group, dim, 32, dtype)
    out, lse = run(A, q, cache, tables, lengths)
    again, lse2 = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2), "the same call gave other bits"


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_many_sequences(A, dtype):
    g = torch.Generator().manual_seed(3)
    run(A, *setup(A, torch.randint(0, 90, (300,), generator=g).tolist(), 1, 2, 3, 32, 8, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("level", [-30000.0, 30000.0])
def test_parts_of_high_and_low_scores_are_joined_as_they_are(A, dtype, level):
    """A large common level of the scores (an element of q and k apart from the others) changes no weight, in one worker or between the parts of many."""
    q, cache, tables, lengths = setup(A, [3000], 1, 1, 4, 32, 16, dtype, scales=False, peak=0.25)
    q[:, :, 0] = level / 128
    cache.k[..., 0] = torch.tensor(128.0).to(R.E4M3).view(torch.uint8).cuda() if dtype == "e4m3" else 128.0
    run(A, q, cache, tables, lengths, scale=1.0)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("peak", [0.0, 30.0, 1000.0])
def test_flat_and_peaked_scores(A, dtype, peak):
    run(A, *setup(A, [129, 1000], 1, 2, 4, 64, 16, dtype, peak=peak))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scale(A, scale):
    run(A, *setup(A, [77], 2, 1, 4, 64, 16, "bf16"), scale=scale)


def test_e4m3_without_scales(A):
    run(A, *setup(A, [77, 5], 1, 2, 4, 64, 16, "e4m3", scales=False))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_rising_scores(A, dtype):
    """Each key's score passes the ones before it by less than 2^8, in steps that add up to far more: the exponents' reference has to follow."""
    q, cache, tables, lengths = setup(A, [600], 1, 1, 2, 32, 16, dtype, scales=False)
    for e in range(600):
        row = torch.full((32,), 0.0)
        row[e % 32] = min(448.0, 0.75 * e)
        cache.k[int(tables[0, e // 16]), 0, e % 16] = row.to(R.E4M3).view(torch.uint8).cuda() if dtype == "e4m3" else row.bfloat16().cuda()
    q.fill_(1.0)
    run(A, q, cache, tables, lengths, scale=1.0)
    run(A, q, cache, tables, lengths, scale=-1.0)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_what_is_not_seen_does_not_matter(A, dtype):
    """Keys and values of later tokens and outside the window hold NaN and infinities: only the queries that see them get any."""
    q, cache, tables, lengths = setup(A, [70], 4, 2, 4, 64, 16, dtype)
    clean = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), window=40)
    for e, value in ((69, math.nan), (68, math.inf), (29, math.nan), (27, -math.inf)):  # the last query sees [30, 70), the first [27, 67)
        for t in (cache.k, cache.v):
            bad = torch.tensor(value, dtype=torch.bfloat16)
            t[int(tables[0, e // 16]), :, e % 16] = NAN8 if dtype == "e4m3" else bad
    out = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), window=40)
    sees = [[e for e in (69, 68, 29, 27) if 27 + i <= e < 67 + i] for i in range(4)]
    assert sees == [[29, 27], [29], [68, 29], [69, 68]]
    assert out.isnan().any(-1).all(), "all four see one of them"
    for e in (29, 27):
        for t in (cache.k, cache.v):
            t[int(tables[0, e // 16]), :, e % 16] = 0
    out = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), window=40)
    assert out[:2].isfinite().all() and not out[2:].isfinite().all()
    R.check_attention(out[:2], None, tuple(r[:2] for r in R.attention(q, cache.k, cache.v, tables, lengths, None, None, 40, cache.k_scale, cache.v_scale)))
    assert clean.isfinite().all()


def test_infinite_scores(A):
    """A key of minus infinity has weight zero; one of plus infinity makes the row NaN, as the formula does."""
    q, cache, tables, lengths = setup(A, [20, 20], 1, 1, 2, 32, 32, "bf16")
    q = q.abs() + 0.5
    low = q.new_full((32,), -math.inf)
    cache.k[int(tables[0, 0]), 0, 7] = low.cuda()
    cache.k[int(tables[1, 0]), 0, 7] = -low.cuda()
    out, lse = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), return_lse=True)
    keep = [e for e in range(20) if e != 7]
    want = torch.softmax((q[0].double() @ cache.k[int(tables[0, 0]), 0, keep].double().cpu().T) * 32**-0.5, -1) @ cache.v[int(tables[0, 0]), 0, keep].double().cpu()
    R.check(out[0], want, 2.0**-8 * want.abs() + 2.0**-9, "out")
    assert out[1].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_pages_outside_the_cache_are_seen_by_nobody(A, dtype):
    q, cache, tables, lengths = setup(A, [100, 100, 40], 2, 2, 4, 64, 16, dtype)
    tables[0, 2], tables[0, 6], tables[1] = -1, cache.pages, 2**31 - 1
    out, lse = run(A, q, cache, tables, lengths)
    assert not out[2:4].any() and (lse[2:4] == -math.inf).all()


def test_lengths_are_taken_within_the_table(A):
    q, cache, tables, _ = setup(A, [64, 64, 64], 1, 2, 2, 64, 16, "bf16")
    out, _ = run(A, q, cache, tables, torch.tensor([10**9, -5, 64], dtype=torch.int32))
    assert not out[1].any()


def test_shared_pages(A):
    """Two sequences with the same beginning."""
    q, cache, tables, lengths = setup(A, [64, 64], 1, 2, 2, 64, 16, "bf16")
    tables[1, :2] = tables[0, :2]
    run(A, q, cache, tables, lengths)


def test_strided_queries_and_results(A):
    q, cache, tables, lengths = setup(A, [33, 65, 9], 1, 2, 4, 64, 16, "bf16")
    wide = torch.full((3, 14 * 64), 9.0, dtype=torch.bfloat16, device="cuda")
    qs = wide[:, 64:9 * 64].view(3, 8, 64).copy_(q)
    to = torch.full((8, 3, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    ref = R.attention(q, cache.k, cache.v, tables, lengths)
    out = A.paged_attention(qs, cache, tables.cuda(), lengths.cuda(), out=to[..., :64].transpose(0, 1))
    R.check_attention(out, None, ref)
    assert (to[..., 64:] == 7).all()
    tall = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    tall[:, 2:2 + tables.shape[1]] = tables.cuda()
    R.check_attention(A.paged_attention(qs, cache, tall[:, 2:2 + tables.shape[1]], lengths.cuda()), None, ref)
    R.check_attention(A.paged_attention(qs[:, :1].expand(3, 8, 64), cache, tables.cuda(), lengths.cuda()), None,
                      R.attention(q[:, :1].expand(3, 8, 64), cache.k, cache.v, tables, lengths))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_pages_behind_32_bits(A, dtype):
    """Entries whose offset in the cache passes 2^32 elements."""
    cache = A.PagedCache.empty(17000, 128, 16, 128, dtype)  # 4.5e9 elements: 8.9 or 4.5 GB each
    pages = [16999, 0, 16998]
    g = torch.Generator().manual_seed(1)
    small = [torch.randn((3, 16, 128, 128), generator=g).to(R.E4M3).view(torch.uint8) if dtype == "e4m3" else torch.randn((3, 16, 128, 128), generator=g).bfloat16() for _ in range(2)]
    for t, s in zip((cache.k, cache.v), small):
        t[pages] = s.cuda()
    q = torch.randn((1, 16, 128), generator=g).bfloat16()
    lengths = torch.tensor([300], dtype=torch.int32)
    out, lse = A.paged_attention(q.cuda(), cache, torch.tensor([pages], dtype=torch.int32).cuda(), lengths.cuda(), return_lse=True)
    R.check_attention(out, lse, R.attention(q, *small, torch.tensor([[0, 1, 2]]), lengths))


def test_captured_with_new_lengths_and_two_graphs(A):
    """The split follows the lengths that stand in memory at replay; two graphs and an eager call each have a workspace of their own."""
    q, cache, tables, lengths = setup(A, [3000, 700, 1], 2, 2, 4, 64, 16, "bf16")
    qs, ts, ls = q.cuda(), tables.cuda(), lengths.cuda()
    graphs = []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for window in (0, 900):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = A.paged_attention(qs, cache, ts, ls, window=window)
            graphs.append((graph, out, window))
    for now in ([3000, 700, 1], [1, 700, 0], [2999, 0, 0]):
        ls.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = A.paged_attention(qs, cache, ts, ls)
        torch.cuda.synchronize()
        for _, out, window in graphs:
            R.check_attention(out, None, R.attention(q, cache.k, cache.v, tables, torch.tensor(now), window=window))
        assert torch.equal(eager, graphs[0][1])


def test_captured_on_a_forked_stream(A):
    """Both launches behind an event, a copy and a memset of another stream, and in front of a kernel of it."""
    q, cache, tables, lengths = setup(A, [2000, 70, 5], 1, 2, 4, 64, 16, "bf16")
    qs, ts, ls = q.cuda(), tables.cuda(), lengths.cuda()
    source, held = qs.clone(), torch.empty_like(qs)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    main.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(main):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            held.zero_()
            held.copy_(source)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                out = A.paged_attention(held, cache, ts, ls)
                twice = A.paged_attention(held, cache, ts, ls, window=33)
            main.wait_stream(side)
            total = out.float() + twice.float()
    for scale in (1.0, 0.5):
        source.copy_(qs * scale)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for o, window in ((out, 0), (twice, 33)):
            R.check_attention(o, None, R.attention(q * scale, cache.k, cache.v, tables, lengths, window=window))
        assert torch.equal(total, out.float() + twice.float())


def test_own_workspace_of_any_content(A):
    q, cache, tables, lengths = setup(A, [3000, 70], 1, 2, 8, 128, 16, "bf16")
    need = A.attention_workspace_bytes(cache, 2, 1, 16, tables.shape[1])
    ws = torch.full((max(need, 1),), 0xFF, dtype=torch.uint8, device="cuda")
    lse = torch.empty((2, 16), device="cuda")
    out, same = A.paged_attention(q.cuda(), cache, tables.cuda(), lengths.cuda(), workspace=ws, lse=lse)
    assert same is lse
    R.check_attention(out, lse, R.attention(q, cache.k, cache.v, tables, lengths))


def test_on_another_stream(A):
    q, cache, tables, lengths = setup(A, [500, 70], 1, 2, 8, 128, 16, "bf16")
    stream = torch.cuda.Stream()
    qs, ts, ls = q.cuda(), tables.cuda(), lengths.cuda()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = A.paged_attention(qs, cache, ts, ls)
    stream.synchronize()
    R.check_attention(out, None, R.attention(q, cache.k, cache.v, tables, lengths))


def test_empty_and_refusals(A):
    from tilefish_b200 import TilefishPreconditionError

    q, cache, tables, lengths = setup(A, [40, 5], 2, 2, 4, 64, 16, "bf16")
    q, tables, lengths = q.cuda(), tables.cuda(), lengths.cuda()
    assert A.paged_attention(q[:0], cache, tables, lengths).shape == (0, 8, 64)
    assert A.paged_attention(q[:0], cache, tables[:0], lengths[:0]).shape == (0, 8, 64)

    def refused(kind, *args, **kwargs):
        with pytest.raises(TilefishPreconditionError) as e:
            A.paged_attention(*args, **kwargs)
        assert e.value.kind == kind, (e.value.kind, str(e.value))

    refused("dtype", q, (cache.k, cache.v), tables, lengths)
    refused("dtype", q.float(), cache, tables, lengths)
    refused("device", q.cpu(), cache, tables, lengths)
    refused("shape", q[..., :32], cache, tables, lengths)
    refused("divisible", q[:, :7], cache, tables, lengths)
    refused("divisible", q[:, :0], cache, tables, lengths)
    refused("divisible", q[:3], cache, tables, lengths)
    refused("divisible", q, cache, tables[:0], lengths[:0])
    refused("dtype", q, cache, tables.long(), lengths)
    refused("rank", q, cache, tables[0], lengths)
    refused("contiguous", q, cache, tables[:, :0], lengths)
    refused("shape", q, cache, tables, lengths[:1])
    refused("dtype", q, cache, tables, lengths.long())
    refused("shape", q, cache, tables, lengths, counts=lengths[:1])
    refused("argument", q, cache, tables, lengths, window=-1)
    refused("argument", q, cache, tables, lengths, window=2**64 + 5)
    refused("argument", q, cache, tables, lengths, scale=math.nan)
    refused("argument", q, cache, tables, lengths, scale=1e39)
    assert torch.equal(A.paged_attention(q, cache, tables, lengths, window=2**62), A.paged_attention(q, cache, tables, lengths))
    refused("alias", q, cache, tables, lengths, out=q)
    refused("shape", q, cache, tables, lengths, out=q[:2].clone())
    refused("shape", q, cache, tables, lengths, lse=torch.empty((4, 7), device="cuda"))
    refused("alignment", torch.zeros((4, 8, 68), dtype=torch.bfloat16, device="cuda")[..., :64], cache, tables, lengths)
    refused("argument", q, cache, tables, lengths, stream=torch.cuda.Stream())


@pytest.mark.parametrize("sequences,queries,heads,width", [(2, 0, 8, 3), (-1, 1, 8, 3), (2, 1, 7, 3), (2, 1, 0, 3), (2, 1, 8, 0), (2**31, 1, 8, 3)])
def test_no_workspace_for_what_is_not_taken(A, sequences, queries, heads, width):
    from tilefish_b200 import TilefishPreconditionError

    _, cache, _, _ = setup(A, [40, 5], 2, 2, 4, 64, 16, "bf16")
    with pytest.raises(TilefishPreconditionError) as e:
        A.attention_workspace_bytes(cache, sequences, queries, heads, width)
    assert e.value.kind == "unsupported"
    with pytest.raises(TilefishPreconditionError):
        A.attention_workspace_bytes((cache.k, cache.v), 2, 1, 8, 3)
