"""Two tokens that name one entry: what that entry holds is unspecified, all others are as they have to be."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
def test_only_the_entry_named_twice_is_unspecified(dtype):
    from tilefish_b200 import attention as A

    cache = A.PagedCache.empty(8, 16, 4, 64, dtype)
    for t in (cache.k, cache.v):
        t.fill_(1)
    before = cache.k.clone(), cache.v.clone()
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randint(-8, 9, (40, 4, 64), generator=g).bfloat16().cuda() for _ in range(2))  # whole numbers: e4m3 codes as they are
    tables = torch.tensor([[3, 1], [6, 2]], dtype=torch.int32, device="cuda")
    positions = torch.arange(20).repeat(2)
    positions[7] = positions[9] = 31  # two of the first sequence
    positions[25] = 4  # entry 4 of the second, which token 24 has too
    A.cache_append(cache, k, v, tables, positions.cuda())
    as_numbers = lambda t: t.view(torch.float8_e4m3fn).float() if dtype == "e4m3" else t.float()  # noqa: E731
    for x, got, old in ((k, cache.k, before[0]), (v, cache.v, before[1])):
        want, sure = as_numbers(old).clone(), torch.ones((8, 16), dtype=torch.bool, device="cuda")
        for t in range(40):
            e, b = int(positions[t]), t // 20
            want[tables[b, e // 16], :, e % 16] = x[t].float()
        sure[tables[0, 1], 15] = sure[tables[1, 0], 4] = False
        same = (as_numbers(got) == want).all(3).all(1)
        assert same[sure].all()
