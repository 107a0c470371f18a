"""A cache's handle goes by the addresses of the tensors that it was made with, so it does not let them be exchanged."""

import pytest

from tilefish_b200 import attention as A


@pytest.mark.parametrize("name", A.PagedCache.__slots__)
def test_nothing_of_a_cache_is_exchanged(name):
    cache = object.__new__(A.PagedCache)
    with pytest.raises(AttributeError, match=name):
        setattr(cache, name, None)


@pytest.mark.gpu
def test_scales_are_followed_where_they_change_in_place():
    import torch

    scale = torch.ones(2, device="cuda")
    cache = A.PagedCache.empty(2, 16, 2, 64, "e4m3", k_scale=scale, v_scale=scale)
    with pytest.raises(AttributeError):
        cache.v_scale = torch.full((2,), 0.5, device="cuda")
    x = torch.full((1, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    tables, positions, lengths = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for s in (1.0, 0.5, 2.0):  # 3, 6 and 1.5 are codes
        scale.fill_(s)
        A.cache_append(cache, x, x, tables, positions)
        assert (cache.v[0, :, 0].view(torch.float8_e4m3fn).float() == 3.0 / s).all()
        assert (A.paged_attention(x, cache, tables, lengths) == 3.0).all()


@pytest.mark.gpu
def test_copies_go_by_their_own_tensors():
    import copy

    import torch

    cache = A.PagedCache.empty(2, 16, 2, 64)
    cache.k.fill_(1.0), cache.v.fill_(1.0)
    same, other = copy.copy(cache), copy.deepcopy(cache)
    assert same.k is cache.k and other.k.data_ptr() != cache.k.data_ptr()
    x = torch.full((1, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    A.cache_append(same, x, x, tables, torch.tensor([0], device="cuda"))
    A.cache_append(other, x, x, tables, torch.tensor([1], device="cuda"))
    assert (cache.v[0, :, 0] == 3).all() and (cache.v[0, :, 1] == 1).all() and (other.v[0, :, 0] == 1).all() and (other.v[0, :, 1] == 3).all()
