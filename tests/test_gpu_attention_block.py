"""attention_block and decoder_layer at their edges: a refused call changes nothing."""

import pytest
import torch

pytestmark = pytest.mark.gpu

H, HEADS, KV, DIM, F = 512, 8, 2, 64, 256


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def parts(A, fmt="mxfp8", h=H, f=F):
    from tilefish_b200 import mlp

    g = torch.Generator().manual_seed(2)
    r = lambda *s: (torch.randn(s, generator=g) * s[-1] ** -0.5).bfloat16().cuda()  # noqa: E731
    return (A.quantize_attention_weights(r(h), r((HEADS + 2 * KV) * DIM, h), r(h, HEADS * DIM), fmt, q_heads=HEADS, kv_heads=KV), mlp.quantize_weights(r(h), r(2 * f, h), r(h, f), fmt))


def test_a_refused_call_changes_nothing(A):
    from tilefish_b200 import TilefishPreconditionError
    from tilefish_b200.attention import AttentionWeights
    from tilefish_b200.mlp import MlpWeights

    att, mlp = parts(A)
    cache = A.PagedCache.empty(8, 16, KV, DIM)
    cache.k.fill_(1.0), cache.v.fill_(2.0)
    x, res = torch.ones((4, H), dtype=torch.bfloat16, device="cuda"), torch.full((4, H), 3.0, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(tables=ints(0, 1, 2, 3).view(2, 2), positions=torch.arange(4, device="cuda"), lengths=ints(2, 2), rotary=A.RotaryTable(A.rotary_frequencies(DIM)[0]))
    other, other_mlp = parts(A, h=256)
    bad = [("tables", good["tables"].long(), "dtype"), ("tables", good["tables"].cpu(), "device"), ("tables", good["tables"][0], "rank"), ("tables", good["tables"].t(), "contiguous"),
           ("tables", ints(0, 1, 2).view(3, 1), "shape"), ("positions", good["positions"][:3], "shape"), ("positions", good["positions"].float(), "dtype"), ("rows", ints(0, 1), "shape"),
           ("rotary", A.rotary_frequencies(DIM), "dtype"), ("rotary", A.RotaryTable(A.rotary_frequencies(128)[0]), "shape"), ("lengths", ints(2, 2).long(), "dtype"), ("lengths", ints(2), "shape"),
           ("counts", ints(2, 2, 2), "shape"), ("counts", ints(2, 2).float(), "dtype"), ("window", -1, "argument"), ("window", 2.5, "argument"), ("cache", (cache.k, cache.v), "dtype"),
           ("cache", A.PagedCache.empty(8, 16, KV, 32), "shape"), ("x", x.float(), "dtype"), ("residual", res[:2], "shape"),
           ("w", AttentionWeights(att.w_n, att.w_qkv, other.w_o, HEADS, KV), "shape"), ("w", AttentionWeights(att.w_n, other.w_qkv, att.w_o, HEADS, KV), "shape"),
           ("w", AttentionWeights(other.w_n, att.w_qkv, att.w_o, HEADS, KV), "shape")]
    for name, value, kind in bad:
        arguments = {"x": x, "residual": res, "w": att, "cache": cache, **good, name: value}
        first = [arguments.pop(n) for n in ("x", "residual", "w", "cache", "tables", "positions", "lengths", "rotary")]
        for call in (lambda: A.attention_block(*first, **arguments), lambda: A.decoder_layer(*first[:3], mlp, *first[3:], **arguments)):
            with pytest.raises(TilefishPreconditionError) as e:
                call()
            assert e.value.kind == kind, (name, e.value.kind, str(e.value))
    odd = dict(good, tables=ints(0, 1, 2).view(3, 1), lengths=ints(1, 1, 1))  # four tokens of three sequences
    for m in (MlpWeights(mlp.w_n, other_mlp.w_gu, mlp.w_d), MlpWeights(mlp.w_n, mlp.w_gu, other_mlp.w_d), MlpWeights(mlp.w_n, parts(A, f=128)[1].w_gu, mlp.w_d), MlpWeights(mlp.w_n, mlp.w_gu, parts(A, "mxfp4")[1].w_d),
              MlpWeights(other_mlp.w_n, mlp.w_gu, mlp.w_d), MlpWeights(mlp.w_n.float(), mlp.w_gu, mlp.w_d)):
        with pytest.raises(TilefishPreconditionError):
            A.decoder_layer(x, res, att, m, cache, *(good[n] for n in ("tables", "positions", "lengths", "rotary")))
    with pytest.raises(TilefishPreconditionError) as e:
        A.attention_block(x, res, att, cache, *(odd[n] for n in ("tables", "positions", "lengths", "rotary")))
    assert e.value.kind == "divisible"
    assert (res == 3).all() and (x == 1).all() and (cache.k == 1).all() and (cache.v == 2).all()
    y = A.decoder_layer(x, res, att, mlp, cache, *(good[n] for n in ("tables", "positions", "lengths", "rotary")))
    assert y.shape == (4, H) and not (res == 3).all() and not (cache.k == 1).all()


@pytest.mark.parametrize("sequences", [0, 2])
def test_a_batch_without_tokens_is_refused_as_the_mlp_block_refuses_it(A, sequences):
    from tilefish_b200 import TilefishPreconditionError
    from tilefish_b200 import mlp as MLP

    att, mlp = parts(A)
    cache = A.PagedCache.empty(8, 16, KV, DIM)
    cache.k.fill_(1.0), cache.v.fill_(2.0)
    x, res = torch.ones((0, H), dtype=torch.bfloat16, device="cuda"), torch.ones((0, H), device="cuda")
    tables, lengths = torch.zeros((sequences, 2), dtype=torch.int32, device="cuda"), torch.zeros(sequences, dtype=torch.int32, device="cuda")
    for call in (lambda: MLP.decoder_block(x, res, mlp), lambda: A.decoder_layer(x, res, att, mlp, cache, tables, torch.arange(0, device="cuda"), lengths)):
        with pytest.raises(TilefishPreconditionError):
            call()
    assert (cache.k == 1).all() and (cache.v == 2).all()
