"""Rotary positions against the rotation in 64 bits, its gradient, and its refusals."""

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


def inputs(tokens, heads, dim, dtype, seed, start=0, step=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((tokens, heads, dim), generator=g).to(dtype), start + step * torch.arange(tokens)


def check(out, x, positions, inv, layout, magnitude=1.0, inverse=False):
    want, size = R.rotated(x, positions, inv, layout, magnitude, inverse)
    error = R.TURN_ERROR * size
    R.check(out, want, torch.where(size > 0, R.rounding(want, x.dtype) + 1.01 * error, 0.0), "rotary")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 1, 128, 128), (3, 5, 128, 128), (65, 64, 128, 64), (33, 7, 80, 32), (17, 3, 80, 80), (5, 9, 96, 26),
                                                  (9, 2, 100, 50), (2, 3, 40, 16), (40, 1, 256, 256), (300, 2, 64, 62), (7, 40, 112, 96), (2, 1, 1024, 1024)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotation(A, dtype, layout, tokens, heads, dim, rot, inverse):
    x, positions = inputs(tokens, heads, dim, dtype, tokens + rot, start=3)
    inv, _ = A.rotary_frequencies(rot)
    table = A.RotaryTable(inv, layout=layout)
    out = A.rotary(x.cuda(), positions.cuda(), table, inverse=inverse)
    check(out, x, positions, inv, layout, inverse=inverse)


@pytest.mark.parametrize("position", [0, 1, 131071, 10**6 + 7, 2**31 - 1, -1, -5000])
@pytest.mark.parametrize("wide", [False, True])
def test_far_positions_keep_their_angle(A, position, wide):
    x, _ = inputs(4, 3, 64, torch.float32, 5)
    positions = torch.full((4,), position, dtype=torch.int64 if wide else torch.int32)
    inv, _ = A.rotary_frequencies(64)
    out = A.rotary(x.cuda(), positions.cuda(), A.RotaryTable(inv))
    # the oracle's angle is a 64-bit product: off by half a step of it
    want, size = R.rotated(x, positions, inv, "half")
    R.check(out, want, R.rounding(want, torch.float32) + (R.TURN_ERROR + abs(position) * 2.0**-53) * size, "rotary")


@pytest.mark.parametrize("scaling", ["linear", "ntk", "bands", "yarn"])
def test_scaled_frequencies(A, scaling):
    inv, magnitude = A.rotary_frequencies(64, base=500000.0, scaling=scaling, factor=8.0, length=4096)
    x, positions = inputs(50, 4, 64, torch.bfloat16, 2, start=30000)
    out = A.rotary(x.cuda(), positions.cuda(), A.RotaryTable(inv, layout="interleaved", magnitude=magnitude))
    check(out, x, positions, inv, "interleaved", magnitude)


@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (96, 26)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strided_in_place_and_out(A, layout, dim, rot):
    heads = 6
    wide = torch.randn((11, (heads + 3) * dim), generator=torch.Generator().manual_seed(1)).bfloat16()
    positions = torch.arange(11, dtype=torch.int32) * 17
    inv, _ = A.rotary_frequencies(rot)
    table = A.RotaryTable(inv, layout=layout)
    gpu = wide.cuda()
    x = gpu[:, dim:(heads + 1) * dim].view(11, heads, dim)
    fresh = A.rotary(x, positions.cuda(), table)
    check(fresh, wide[:, dim:(heads + 1) * dim].reshape(11, heads, dim), positions, inv, layout)
    by_heads = torch.full((heads, 11, dim), 7.0, dtype=torch.bfloat16, device="cuda")  # heads outside, tokens inside
    A.rotary(x, positions.cuda(), table, out=by_heads.transpose(0, 1))
    assert torch.equal(by_heads.transpose(0, 1), fresh)
    both = torch.cat([x, torch.full_like(x, 5.0)], dim=1)  # into other columns of the same matrix
    A.rotary(both[:, :heads], positions.cuda(), table, out=both[:, heads:])
    assert torch.equal(both[:, heads:], fresh) and torch.equal(both[:, :heads], x)
    assert A.rotary(x, positions.cuda(), table, out=x) is x
    assert torch.equal(x, fresh)
    assert torch.equal(gpu[:, :dim].cpu(), wide[:, :dim]) and torch.equal(gpu[:, (heads + 1) * dim:].cpu(), wide[:, (heads + 1) * dim:])


def test_unaligned_and_broadcast_inputs(A):
    inv, _ = A.rotary_frequencies(32)
    table = A.RotaryTable(inv)
    flat = torch.randn(5 * 3 * 48 + 1, generator=torch.Generator().manual_seed(4)).bfloat16()
    x = flat[1:].view(5, 3, 48)
    positions = torch.arange(5)
    gpu = flat.cuda()[1:].view(5, 3, 48)  # two bytes behind a 16-byte boundary
    check(A.rotary(gpu, positions.cuda(), table), x, positions, inv, "half")
    one = x[:, :1].expand(5, 7, 48)
    check(A.rotary(gpu[:, :1].expand(5, 7, 48), positions.cuda(), table), one, positions, inv, "half")


def test_the_gradient_is_the_way_back(A):
    """<g, R x> = <R^T g, x>, with R^T the inverse call, and against differences of the exact rotation."""
    inv, _ = A.rotary_frequencies(48)
    table = A.RotaryTable(inv, layout="interleaved", magnitude=1.25)
    x, positions = inputs(6, 3, 64, torch.float32, 8, start=100)
    g, _ = inputs(6, 3, 64, torch.float32, 9)
    back = A.rotary(g.cuda(), positions.cuda(), table, inverse=True)
    check(back, g, positions, inv, "interleaved", 1.25, inverse=True)
    y, _ = R.rotated(x, positions, inv, "interleaved", 1.25)
    step = 0.5  # the map is linear: a difference is exact whatever its step
    for at in [(0, 0, 0), (3, 2, 47), (5, 1, 60), (2, 0, 13)]:
        moved = x.clone().double()
        moved[at] += step
        difference = ((R.rotated(moved, positions, inv, "interleaved", 1.25)[0] - y) * g.double()).sum() / step
        assert abs(float(difference) - float(back[at])) <= 2 * R.TURN_ERROR * 1.25 * float(g.abs().max()) * 2 + 1e-12


def test_specials_stay_in_their_pair(A):
    inv, _ = A.rotary_frequencies(64)
    x, positions = inputs(3, 2, 64, torch.bfloat16, 3)
    x[1, 0, 5], x[2, 1, 40] = math.nan, math.inf
    out = A.rotary(x.cuda(), positions.cuda(), A.RotaryTable(inv)).cpu()
    assert out[1, 0, [5, 37]].isnan().all() and not out[2, 1, [8, 40]].isfinite().any()
    rest = torch.ones_like(x, dtype=torch.bool)
    rest[1, 0, [5, 37]] = rest[2, 1, [8, 40]] = False
    assert out[rest].isfinite().all()


def test_captured_with_new_positions(A):
    inv, _ = A.rotary_frequencies(128)
    table = A.RotaryTable(inv)
    x, positions = inputs(4, 8, 128, torch.bfloat16, 6)
    xs, ps = x.cuda(), positions.cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        A.rotary(xs, ps, table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = A.rotary(xs, ps, table)
    for start in (5, 70000):
        ps.copy_(positions + start)
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, positions + start, inv, "half")


def test_empty_and_refusals(A):
    from tilefish_b200 import TilefishPreconditionError

    inv, _ = A.rotary_frequencies(64)
    table = A.RotaryTable(inv)
    x, positions = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.arange(4, device="cuda")
    assert A.rotary(x[:0], positions[:0], table).shape == (0, 2, 64) and A.rotary(x[:, :0], positions, table).shape == (4, 0, 64)

    def refused(kind, *args, **kwargs):
        with pytest.raises(TilefishPreconditionError) as e:
            A.rotary(*args, **kwargs)
        assert e.value.kind == kind, (e.value.kind, str(e.value))

    refused("dtype", x.half(), positions, table)
    refused("device", x.cpu(), positions, table)
    refused("rank", x[0], positions, table)
    refused("shape", x, positions[:3], table)
    refused("dtype", x, positions.float(), table)
    refused("shape", x[..., :32], positions, table)
    refused("contiguous", x.transpose(1, 2).contiguous().transpose(1, 2), positions, table)
    refused("dtype", x, positions, inv)
    refused("alias", x[1:], positions[1:], table, out=x[:3])
    refused("alias", x, positions, table, out=torch.empty((1, 2, 64), dtype=torch.bfloat16, device="cuda").expand(4, 2, 64))
    refused("dtype", x, positions, table, out=x.float())
    refused("contiguous", x, torch.arange(8, device="cuda")[::2], table)
