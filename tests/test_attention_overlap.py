"""Which results share memory with what a call reads, byte by byte (no GPU: views of CPU memory)."""

import random

import pytest
import torch

from tilefish_b200 import TilefishPreconditionError
from tilefish_b200 import attention as A


def elements(t):
    at = torch.zeros(t.shape, dtype=torch.int64)
    for axis, (n, st) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * st).view([-1 if i == axis else 1 for i in range(t.dim())])
    return set(((at + t.storage_offset()).flatten()).tolist())


def view(base, shape, strides, offset):
    return torch.as_strided(base, shape, strides, offset)


def test_slices_of_one_tensor():
    base = torch.zeros(2, 6, 4, 5, 16)
    both = [base[:, :, :2], base[:, :, 2:]], [base[:, :3], base[:, 3:]], [base[..., :8], base[..., 8:]], [base[0:1], base[1:2]], [base[:, ::2], base[:, 1::2]]
    for a, b in both:
        for t in ((a, b), (a.transpose(1, 2), b.transpose(1, 2)), (a.transpose(0, 3), b.transpose(0, 3)), (b, a)):
            assert not A._overlap(*t)
        assert A._overlap(a, a) and A._overlap(a, base)
    heads_first = torch.zeros(8, 2, 9, 16)  # two tensors with their tokens between one another's
    assert not A._overlap(heads_first[:, 0].transpose(0, 1), heads_first[:, 1].transpose(0, 1))
    assert A._overlap(heads_first[:, 0].transpose(0, 1)[1:], heads_first[:, 0].transpose(0, 1)[:-1])


def test_nothing_shared_is_said_to_be_apart():
    """Boxes of the same strides: said to overlap exactly where they do."""
    rng = random.Random(3)
    base = torch.zeros(4000)
    seen = [0, 0]
    for _ in range(4000):
        dim = rng.choice((2, 4, 8))
        width = dim + rng.choice((0, 0, 2, 8))
        inner, outer = rng.randint(1, 4), rng.randint(1, 4)
        strides = (width * inner + rng.choice((0, 0, dim, 5)), width)
        shapes = [(rng.randint(1, outer), rng.randint(1, inner), rng.randint(1, dim)) for _ in range(2)]
        order = rng.random() < 0.5
        a, b = (view(base, s, (*strides, 1), rng.randint(0, 120)) for s in shapes)
        if order:
            a, b = a.transpose(0, 1), b.transpose(0, 1)
        want = bool(elements(a) & elements(b))
        seen[want] += 1
        assert A._overlap(a, b) == want, (a.shape, b.shape, strides, a.storage_offset(), b.storage_offset(), order)
    assert min(seen) > 500


def test_other_strides_are_never_said_to_be_apart_wrongly():
    rng = random.Random(4)
    base = torch.zeros(4000)
    for _ in range(3000):
        a, b = (view(base, (rng.randint(1, 3), rng.randint(1, 3), 4), (rng.randint(0, 20), rng.randint(0, 20), 1), rng.randint(0, 80)) for _ in range(2))
        if elements(a) & elements(b):
            assert A._overlap(a, b)


def test_empty_tensors_share_nothing():
    t = torch.zeros(4, 2, 16)
    assert not A._overlap(t[:0], t) and not A._overlap(t, t[:, :0])


def test_results_do_not_overlap_themselves():
    base = torch.zeros(4000)
    for shape, strides, fine in (((5, 3, 8), (24, 8, 1), True), ((5, 3, 8), (8, 40, 1), True), ((5, 3, 8), (24, 0, 1), False), ((5, 3, 8), (0, 8, 1), False), ((5, 3, 8), (16, 8, 1), False),
                                 ((5, 3, 8), (24, 4, 1), False), ((1, 3, 8), (0, 8, 1), True), ((5, 1, 8), (8, 0, 1), True), ((5, 1, 8), (4, 0, 1), False), ((5, 3, 8), (8, 24, 1), False),
                                 ((0, 3, 8), (0, 0, 1), True), ((4, 0, 8), (0, 0, 1), True)):
        t = view(base, shape, strides, 0)
        if fine:
            A._result(t, "out")
        else:
            with pytest.raises(TilefishPreconditionError) as e:
                A._result(t, "out")
            assert e.value.kind == "alias"


def test_ranges():
    A._apart(100, 200, "out", (((200, 300), "b"), ((0, 100), "c")))
    for span in ((199, 300), (0, 101), (120, 130), (0, 1000)):
        with pytest.raises(TilefishPreconditionError) as e:
            A._apart(100, 200, "out", ((span, "b"),))
        assert e.value.kind == "alias"


def test_columns_of_one_matrix():
    """The short look says that two tensors are apart only where they are, and says so of the slices of a qkv product."""
    rng = random.Random(5)
    base = torch.zeros(4000, dtype=torch.bfloat16)
    said = 0
    for _ in range(4000):
        step = rng.choice((0, 24, 40, 64))
        rows = []
        for _ in range(2):
            shape, strides = (rng.randint(1, 4), rng.randint(1, 3), 8), (rng.choice((step, step, step, 56)), rng.choice((0, 8, 16, 24)), 1)
            t = view(base, shape, strides, rng.randint(0, 150))
            rows.append((t, (t.shape, *A._strides(t.shape, t.stride()), t.data_ptr())))
        (a, ra), (b, rb) = rows
        assert A._ends(ra, 2) == A._span(a)
        if A._columns(ra, rb, 2):
            said += 1
            assert not elements(a) & elements(b)
    assert said > 200
    q, k, v = torch.zeros(5, 12, 16, dtype=torch.bfloat16).split([8, 2, 2], dim=1)
    q, k, v = ((t.shape, *A._strides(t.shape, t.stride()), t.data_ptr()) for t in (q, k, v))
    assert A._columns(q, k, 2) and A._columns(q, v, 2) and A._columns(v, k, 2) and not A._columns(k, k, 2)
