"""The attention operators together, as a decoder layer runs them: prompts, then single tokens, then drafted tokens over one cache."""

import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


H, HEADS, KV, DIM, F = 512, 8, 2, 64, 256


def weights(A, fmt, seed):
    from tilefish_b200 import mlp

    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(s, generator=g) * s[-1] ** -0.5).bfloat16().cuda()  # noqa: E731
    norm = lambda: (1 + 0.1 * torch.randn(H, generator=g)).bfloat16().cuda()  # noqa: E731
    return (A.quantize_attention_weights(norm(), r((HEADS + 2 * KV) * DIM, H), r(H, HEADS * DIM), fmt, q_heads=HEADS, kv_heads=KV),
            mlp.quantize_weights(norm(), r(2 * F, H), r(H, F), fmt))


def make_cache(A, dtype):
    scale = [torch.full((KV,), 0.02, device="cuda") for _ in range(2)] if dtype == "e4m3" else [None, None]
    return A.PagedCache.empty(20, 16, KV, DIM, dtype, k_scale=scale[0], v_scale=scale[1])


@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_the_block_is_its_operators(A, fmt, dtype):
    """attention_block against the same operators called one by one, with the attention against the formula in 64 bits over the cache that the block wrote."""
    from tilefish_b200 import kernels as K

    w, _ = weights(A, fmt, 1)
    cache, table = make_cache(A, dtype), A.RotaryTable(A.rotary_frequencies(DIM)[0])
    tables = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:18].view(3, 6).int().cuda()
    g = torch.Generator().manual_seed(5)
    start = torch.zeros(3, dtype=torch.int64)
    for new in (20, 1, 1, 4):  # a prompt, two steps, four drafted tokens
        x, res = torch.randn((3 * new, H), generator=g).bfloat16().cuda(), torch.randn((3 * new, H), generator=g).cuda()
        positions = (start[:, None] + torch.arange(new)).view(-1).cuda()
        start += new
        lengths = start.int().cuda()
        mine = res.clone()
        y = A.attention_block(x, mine, w, cache, tables, positions, lengths, table)
        if fmt == "nvfp4":
            amax = torch.zeros(1, device="cuda")
            hq = K.quantize(K.residual_add_rmsnorm(x, res, w.w_n, amax_out=amax), fmt, amax=amax)
        else:
            _, hq = K.residual_add_rmsnorm(x, res, w.w_n, quantize_to=fmt, want_bf16=False)
        assert torch.equal(mine, res)
        q, k, v = K.gemm_blockscaled(hq, w.w_qkv).view(3 * new, -1, DIM).split([HEADS, KV, KV], dim=1)
        q = A.rotary(q, positions, table)
        turned = A.rotary(k, positions, table)
        for t in range(3 * new):
            e = int(positions[t])
            at = (int(tables[t // new, e // 16]), slice(None), e % 16)
            if dtype == "bf16":
                assert torch.equal(cache.k[at], turned[t]) and torch.equal(cache.v[at], v[t])
        o = A.paged_attention(q, cache, tables, lengths)
        R.check_attention(o, None, R.attention(q, cache.k, cache.v, tables, lengths, None, None, 0, cache.k_scale, cache.v_scale))
        assert torch.equal(y, K.gemm(o.view(3 * new, -1), w.w_o))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_tokens_one_by_one_give_what_a_prompt_gives(A, dtype):
    """The keys, values and attention of a sequence do not depend on how many tokens come at once. Row kernels and GEMMs are left out: their launch forms
    differ with the number of rows."""
    g = torch.Generator().manual_seed(3)
    n = 37
    qkv = torch.randn((n, HEADS + 2 * KV, DIM), generator=g).bfloat16().cuda()
    table = A.RotaryTable(A.rotary_frequencies(DIM)[0], layout="interleaved")
    tables = torch.tensor([[4, 0, 7]], dtype=torch.int32, device="cuda")
    whole, steps = make_cache(A, dtype), make_cache(A, dtype)
    for c in (whole, steps):
        c.k.zero_(), c.v.zero_()
    positions = torch.arange(n, device="cuda")
    q, k, v = qkv.split([HEADS, KV, KV], dim=1)
    turned = A.cache_append(whole, k, v, tables, positions, q=q, rotary=table)
    out = A.paged_attention(turned, whole, tables, torch.tensor([n], dtype=torch.int32, device="cuda"))
    for t in range(n):
        one = A.cache_append(steps, k[t:t + 1], v[t:t + 1], tables, positions[t:t + 1], q=q[t:t + 1], rotary=table)
        assert torch.equal(one[0], turned[t])
        lengths = torch.tensor([t + 1], dtype=torch.int32, device="cuda")
        o = A.paged_attention(one, steps, tables, lengths)
        ref = R.attention(one, steps.k, steps.v, tables, lengths, None, None, 0, steps.k_scale, steps.v_scale)
        R.check_attention(o, None, ref)
        R.check_attention(out[t:t + 1], None, ref)
    assert torch.equal(whole.k, steps.k) and torch.equal(whole.v, steps.v)


@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
def test_a_captured_decode_step(A, fmt):
    """A whole layer in a CUDA graph, replayed for token after token, against the eager calls."""
    att, mlp = weights(A, fmt, 7)
    table = A.RotaryTable(A.rotary_frequencies(DIM)[0])
    tables = torch.arange(18, dtype=torch.int32, device="cuda").view(3, 6)
    g = torch.Generator().manual_seed(8)
    xs = torch.randn((6, 3, H), generator=g).bfloat16().cuda()

    def fresh():
        c = make_cache(A, "bf16")
        c.k.zero_(), c.v.zero_()
        return c, torch.zeros((3, H), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")

    def step(x, cache, res, positions, lengths):
        lengths += 1
        y = A.decoder_layer(x, res, att, mlp, cache, tables, positions, lengths, table)
        positions += 1
        return y

    eager = fresh()
    want = [step(x, *eager).clone() for x in xs]
    state, x = fresh(), torch.empty_like(xs[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x.copy_(xs[0])
        step(x, *fresh())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = step(x, *state)
        for i in range(6):
            x.copy_(xs[i])
            graph.replay()
            assert torch.equal(y, want[i]), i
    torch.cuda.synchronize()
    assert torch.equal(state[0].k, eager[0].k) and torch.equal(state[1], eager[1])


def test_the_weights_have_to_match_the_cache(A):
    from tilefish_b200 import TilefishPreconditionError

    w, _ = weights(A, "mxfp8", 1)
    x, res = torch.zeros((1, H), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, H), device="cuda")
    args = (torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(TilefishPreconditionError):
        A.attention_block(x, res, w, A.PagedCache.empty(2, 16, KV, 128), *args)
    with pytest.raises(TilefishPreconditionError):
        A.quantize_attention_weights(w.w_n, torch.zeros((100, H), dtype=torch.bfloat16, device="cuda"), torch.zeros((H, 64), dtype=torch.bfloat16, device="cuda"), "mxfp8",
                                     q_heads=8, kv_heads=3)
