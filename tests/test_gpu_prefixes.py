"""Shared prefixes: which slots begin with the same pages, against lists."""
import pytest
import torch

import step_ref as R
from lazy_compiler_b200 import serving as S

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(table, lens, pages, page):
    maps = S.CacheMaps(ints(table).reshape(len(lens), -1), ints(lens), torch.zeros(pages, dtype=torch.int32, device="cuda"))
    got = S.cache_prefixes(maps, page_size=page)
    for name, x, want in zip(got._fields, got, R.prefixes(maps.table.cpu(), lens, pages, page)):
        assert x.tolist() == list(want), name
    return got


def test_groups():
    table = [[0, 1, 2, 9], [3, 4, 5, 6], [0, 1, 7, 8], [3, 4, 5, 10], [0, 1, 2, 11], [12, 1, 2, 9], [13, -1, -1, -1]]
    got = check(table, [64, 50, 64, 49, 60, 64, 16], 20, 16)
    assert got.leader.tolist() == [0, 1, 0, 1, 0, 5, 6] and got.shared.tolist() == [32, 48, 32, 48, 32, 0, 0]


def test_what_is_not_shared():
    """Empty slots, last pages that are not full, pages that do not exist, lengths outside the table."""
    table = [[0, 1], [0, 1], [0, 1], [-1, 1], [-1, 1], [99, 1], [99, 1], [4, 5], [4, 6], [0, 1]]
    check(table, [0, 15, 16, 32, 32, 32, 32, 31, 31, 1000], 10, 16)
    check(table, [-5, 16, 31, 32, 32, 32, 32, 16, 31, 2 ** 31 - 1], 10, 16)
    check([[0], [0], [0]], [1, 1, 1], 1, 1)
    check([[]], [0], 4, 16)
    maps = S.CacheMaps(ints([]).reshape(0, 3), ints([]), ints([0, 0]))
    assert [x.numel() for x in S.cache_prefixes(maps, page_size=16)] == [0, 0, 0]


@pytest.mark.parametrize("slots,width,groups", [(1, 5, 1), (33, 3, 4), (64, 2500, 3), (257, 513, 20), (1000, 40, 999), (8192, 2, 50)])
def test_random(slots, width, groups):
    g = torch.Generator().manual_seed(slots)
    prompt = torch.randint(0, groups, (slots,), generator=g)
    agree = torch.randint(max(1, width // 2), width + 1, (slots,), generator=g)
    table = prompt.view(-1, 1) * width + torch.arange(width)
    own = groups * width + torch.arange(slots * width).view(slots, width)
    table = torch.where(torch.arange(width) < agree.view(-1, 1), table, own)
    lens = torch.randint(0, 8 * width + 1, (slots,), generator=g)
    lens[::3] = 8 * width
    check(table.tolist(), lens.tolist(), (groups + slots) * width, 8)


def test_a_fork_and_what_follows():
    cache = S.PagedCache(1, 64, 16, 1, 16, 6, 8, dtype=torch.float16)
    cache.extend(ints([40, 33, 0, 0, 0, 0]))
    cache.fork(ints([0, 1, 0, 1, 0, -1]))
    got = cache.prefixes()
    assert got.leader.tolist() == [0, 1, 0, 1, 0, 5] and got.shared.tolist() == [32, 32, 32, 32, 32, 0]
    assert got.order.tolist() == [0, 2, 4, 1, 3, 5]
    cache.extend(ints([20, 1, 1, 1, 7, 0]))
    cache.compact()
    again = cache.prefixes(into=S.CachePrefixes(*(torch.zeros_like(x) for x in got)))
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    cache.release(ints([1, 0, 0, 0, 0, 0]))
    assert cache.prefixes().leader.tolist() == [0, 1, 2, 1, 2, 5]
    cache.check()
