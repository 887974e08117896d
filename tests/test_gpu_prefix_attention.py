"""Attention over shared prefixes against the plain 64-bit form, and against the form that shares nothing."""
import numpy as np
import pytest
import torch

import serving_ref as R
from lazy_compiler_b200 import runtime
from lazy_compiler_b200 import serving as S

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# all slots' tables together hold what makes the prefixes worth a kernel of their own
CAPACITY = 200 << 20


def ints(v):
    return torch.as_tensor(v, dtype=torch.int32).cuda()


def cache(groups, page, h, d, dtype, seed=0, mix=True):
    """groups: (prefix tokens, [suffix tokens of each slot]).  Slots of a group share the prefix's full pages.  Returns k and v
    pages, table, lens, and the prefixes."""
    g = torch.Generator().manual_seed(seed)
    slots = [(i, s) for i, (_, suffixes) in enumerate(groups) for s in suffixes]
    if mix:
        slots = [slots[i] for i in torch.randperm(len(slots), generator=g).tolist()]
    lens = [groups[i][0] + s for i, s in slots]
    width = max(max(-(-n // page) for n in lens), CAPACITY // (len(slots) * page * h * d * 4) + 1)
    need = sum(-(-n // page) for n in lens) + 3
    ids, at = torch.randperm(need, generator=g).tolist(), 0
    table = torch.full((len(slots), width), -1, dtype=torch.int32)
    shared = {}
    for x, (i, _) in enumerate(slots):
        full = groups[i][0] // page
        if i not in shared:
            shared[i] = ids[at:at + full]
            at += full
        own = -(-lens[x] // page) - full
        table[x, :full] = torch.tensor(shared[i], dtype=torch.int32)
        table[x, full:full + own] = torch.tensor(ids[at:at + own], dtype=torch.int32)
        at += own
    cuda = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(need, h, page, d, generator=cuda, device="cuda").to(TYPES[dtype]) for _ in range(2))
    maps = S.CacheMaps(table.cuda(), ints(lens), torch.ones(need, dtype=torch.int32, device="cuda"))
    return k, v, maps, S.cache_prefixes(maps, page_size=page)


def queries(slots, hq, d, dtype, seed=1):
    return torch.randn(slots, hq, d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(TYPES[dtype])


def check(q, k, v, maps, prefixes, dtype, window=0, sinks=0, slots=None, **options):
    o, lse = S.shared_decode(q, k, v, maps.table, maps.lens, prefixes, window=window, sinks=sinks, return_lse=True, **options)
    pick = list(range(len(q)))[:: max(1, len(q) // 12)] if slots is None else slots
    f = lambda x: x.double().cpu().numpy()  # noqa: E731
    ref = R.paged_decode(f(q[pick]), f(k), f(v), maps.table[pick].cpu().numpy(), maps.lens[pick].cpu().numpy(), 1 / np.sqrt(q.shape[2]), window, sinks)
    got, infinite = f(o[pick]), np.isinf(ref[0])  # infinite outputs are the same ones; the others within the bound
    assert (got[infinite] == ref[0][infinite]).all()
    R.check_attention(np.where(infinite, 0, got), f(lse[pick]), (np.where(infinite, 0, ref[0]), ref[1], np.where(infinite, 0, ref[2])), dtype)
    # every slot alone: two roundings of the same values
    p, p_lse = S.paged_decode(q, k, v, maps.table, maps.lens, window=window, sinks=sinks, return_lse=True)
    both = torch.isfinite(p.float())
    assert torch.equal(both, torch.isfinite(o.float()))
    off = ((o.float() - p.float()).abs() - 3 * R.U[dtype] * p.float().abs().clamp(min=0.25))[both]
    assert not len(off) or float(off.max()) <= 0, float(off.max())
    runtime.call("lc_device_status", None)
    return o, lse


SHAPES = [(8, 2, 64, 16), (4, 4, 128, 16), (32, 8, 128, 16), (10, 2, 96, 8), (6, 1, 40, 7), (16, 1, 128, 64), (24, 2, 64, 128), (1, 1, 8, 1)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hq,h,d,page", SHAPES)
def test_shapes(dtype, hq, h, d, page):
    groups = [(500, [1, 40, 7]), (1000, [3]), (129, [1, 1]), (300, [20, 200, 5, 6, 90]), (60, [8, 9])]
    k, v, maps, prefixes = cache(groups, page, h, d, dtype)
    check(queries(13, hq, d, dtype), k, v, maps, prefixes, dtype)


@pytest.mark.parametrize("samples,prefix", [(16, 400), (33, 1025), (40, 250), (64, 2000), (130, 140)])
def test_rows_of_several_tiles(samples, prefix):
    """Four heads a group: 64 rows, 132 (two tiles), 160, 256, 520 (three blocks of 256 rows, the last of 8)."""
    k, v, maps, prefixes = cache([(prefix, [1 + 7 * (i % 9) for i in range(samples)]), (300, [1, 2])], 16, 2, 64, "f16")
    check(queries(samples + 2, 8, 64, "f16"), k, v, maps, prefixes, "f16", slots=[0, 1, samples // 2, samples, samples + 1])


@pytest.mark.parametrize("dtype,h,d", [("f16", 1, 128), ("bf16", 2, 64)])
def test_long_prefix(dtype, h, d):
    """More blocks than a CTA's run: parts of many CTAs to a row, of one group, and with others beside it."""
    k, v, maps, prefixes = cache([(30000, [5, 1, 3000])], 16, h, d, dtype)
    check(queries(3, 4 * h, d, dtype), k, v, maps, prefixes, dtype)
    k, v, maps, prefixes = cache([(9000, [5] * 40), (20000, [1, 2]), (128, [1, 1, 1])], 32, h, d, dtype)
    check(queries(45, 4 * h, d, dtype), k, v, maps, prefixes, dtype, slots=[0, 11, 22, 33, 44])


def test_many_groups():
    k, v, maps, prefixes = cache([(128 + 16 * (i % 7), [1 + i % 5, 3]) for i in range(150)], 16, 2, 64, "bf16")
    check(queries(300, 4, 64, "bf16"), k, v, maps, prefixes, "bf16")


@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 0), (300, 4), (700, 130), (5000, 4), (64, 600), (900, 1)])
def test_windows(window, sinks):
    """Windows that end in the suffixes, in the prefix, and differ between the slots of a group; sinks within and beyond."""
    groups = [(800, [1, 200, 640]), (256, [10, 300]), (1500, [2, 2, 2, 900])]
    k, v, maps, prefixes = cache(groups, 16, 2, 64, "f16")
    q = queries(9, 8, 64, "f16")
    check(q, k, v, maps, prefixes, "f16", window, sinks)
    k, v, maps, prefixes = cache(groups, 12, 1, 128, "bf16")
    check(queries(9, 5, 128, "bf16"), k, v, maps, prefixes, "bf16", window, sinks)


def test_prefixes_of_the_callers():
    """Any number of tokens, also all that a slot has; a slot that has fewer now, or none; no plan at all."""
    k, v, maps, _ = cache([(640, [0, 0, 30, 30, 30]), (320, [1])], 16, 2, 64, "f16", mix=False)
    q, zero = queries(6, 8, 64, "f16"), ints([0] * 6)
    for tokens in (640, 639, 333, 129, 128, 127, 1, 0, 100000):
        given = S.CachePrefixes(ints([0, 0, 0, 0, 0, 5]), ints([min(tokens, 640)] * 5 + [0]), ints([0, 1, 2, 3, 4, 5]))
        check(q, k, v, maps, given, "f16")
    given = S.CachePrefixes(ints([0, 0, 0, 0, 0, 5]), ints([640] * 5 + [0]), ints([0, 1, 2, 3, 4, 5]))
    fewer = maps._replace(lens=ints([640, 200, 0, 650, 127, 0]))
    o, lse = check(q, k, v, fewer, given, "f16")
    assert float(o[2].abs().max()) == 0 and bool((lse[[2, 5]] == -np.inf).all())
    alone = S.CachePrefixes(ints(range(6)), zero, ints(range(6)))
    check(q, k, v, maps, alone, "f16")
    one = S.CachePrefixes(ints(range(6)), ints([640, 0, 0, 640, 0, 320]), ints(range(6)))  # groups of one, with a prefix
    check(q, k, v, maps, one, "f16")


def test_pages_that_are_not_there():
    k, v, maps, prefixes = cache([(800, [1, 20, 7]), (512, [9, 9])], 16, 2, 64, "bf16", mix=False)
    for at in (0, 3, 17, 40):
        maps.table[:3, at] = maps.table[0, at] * 0 - 1
    maps.table[:3, 20] = k.shape[0]
    maps.table[3:, 5:30] = -1
    check(queries(5, 8, 64, "bf16"), k, v, maps, prefixes, "bf16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinite_and_unseen_values(dtype):
    """What no slot sees (behind the ends, outside the window) may be NaN; infinite values that are seen come out as they
    do where nothing is shared."""
    nan, inf = float("nan"), float("inf")
    k, v, maps, prefixes = cache([(400, [5, 30, 77])], 16, 1, 64, dtype, mix=False)
    q = queries(3, 4, 64, dtype)
    for x, n in enumerate(maps.lens.tolist()):
        last = int(maps.table[x, (n - 1) // 16])
        if n % 16:
            k[last, :, n % 16:] = nan
            v[last, :, n % 16:] = inf
    check(q, k, v, maps, prefixes, dtype)
    windowed_k, windowed_v = k.clone(), v.clone()
    windowed_k[maps.table[0, :6].long()] = nan  # the first 96 tokens, unseen in a window of 300
    windowed_v[maps.table[0, :6].long()] = nan
    check(q, windowed_k, windowed_v, maps, prefixes, dtype, window=300)
    v[maps.table[0, 9].long(), 0, 3, 17] = inf
    v[maps.table[1, 25].long(), 0, 1, 5] = -inf
    o, _ = check(q, k, v, maps, prefixes, dtype)
    assert bool((o[:, :, 17] == inf).all()) and bool((o[1, :, 5] == -inf).all())


def test_weights_that_leave_each_other_far():
    """The prefix outweighs the suffix by far, and the other way round; values at the type's end."""
    for dtype in ("f16", "bf16"):
        k, v, maps, prefixes = cache([(256, [16, 40])], 16, 1, 64, dtype, mix=False)
        q = queries(2, 2, 64, dtype)
        for first, rest in ((8.0, 0.1), (0.1, 8.0), (0.0, 0.0)):
            kk, vv = k * rest, v.clone()
            kk[maps.table[0, :16].long()] = k[maps.table[0, :16].long()] * first
            check(q, kk, vv, maps, prefixes, dtype)
        big = torch.sign(v.float()) * torch.finfo(TYPES[dtype]).max
        o, _ = S.shared_decode(q, k, big.to(TYPES[dtype]), maps.table, maps.lens, prefixes, return_lse=True)
        p = S.paged_decode(q, k, big.to(TYPES[dtype]), maps.table, maps.lens)
        assert bool(torch.isfinite(o.float()).all()) and bool(((o.float() - p.float()).abs() <= 2e-2 * torch.finfo(TYPES[dtype]).max).all())


def test_strides():
    """Pages in another order of axes, queries and outputs in wider rows, a table's slice."""
    k, v, maps, prefixes = cache([(300, [5, 30, 77]), (200, [1, 1])], 16, 2, 64, "f16")
    q = queries(5, 8, 64, "f16")
    want, _ = check(q, k, v, maps, prefixes, "f16")
    other = lambda x: torch.nn.functional.pad(x.permute(0, 2, 1, 3).contiguous(), (0, 8)).permute(0, 2, 1, 3)[..., :64]  # noqa: E731
    wide_q = torch.nn.functional.pad(q, (2, 6))[..., 2:66]
    wide_table = torch.nn.functional.pad(maps.table, (0, 3), value=7)[:, :maps.table.shape[1]]
    out = torch.full((5, 9, 70), 5.0, dtype=torch.float16, device="cuda")
    got = S.shared_decode(wide_q, other(k), other(v), wide_table, maps.lens, prefixes, out=out[:, 1:, 3:67])
    assert torch.equal(got, want) and bool((out[:, 0] == 5).all()) and bool((out[:, :, :3] == 5).all()) and bool((out[:, :, 67:] == 5).all())


def test_what_the_tensor_form_does_not_take():
    """Heads over 128, odd sizes and small caches run as if nothing were shared."""
    for hq, h, d, page in ((4, 2, 256, 16), (4, 2, 36, 16), (3, 1, 20, 8)):
        k, v, maps, prefixes = cache([(200, [5, 30]), (200, [1])], page, h, d, "f16")
        check(queries(3, hq, d, "f16"), k, v, maps, prefixes, "f16")
    k, v, maps, prefixes = cache([(64, [1, 1])], 16, 2, 64, "f16")
    small = maps._replace(table=maps.table[:, :6].contiguous())
    check(queries(2, 4, 64, "f16"), k, v, small, prefixes, "f16")


def test_repeats_bit_for_bit():
    k, v, maps, prefixes = cache([(3000, [5] * 20), (700, [1, 2, 3])], 16, 2, 128, "bf16")
    q = queries(23, 8, 128, "bf16")
    first = S.shared_decode(q, k, v, maps.table, maps.lens, prefixes)
    for _ in range(5):
        assert torch.equal(first, S.shared_decode(q, k, v, maps.table, maps.lens, prefixes))


@pytest.mark.parametrize("d", [64, 128])
def test_most_slots(d):
    slots = 8192
    table = torch.zeros((slots, 17), dtype=torch.int32)
    table[:, :9] = torch.arange(9)
    table[:, 9] = 9 + torch.arange(slots)
    k, v = (torch.randn(9 + slots, 1, 16, d, generator=torch.Generator(device="cuda").manual_seed(x), device="cuda").half() for x in (0, 1))
    lens = 144 + torch.arange(slots) % 16 + 1
    maps = S.CacheMaps(table.cuda(), ints(lens), torch.ones(9 + slots, dtype=torch.int32, device="cuda"))
    prefixes = S.cache_prefixes(maps, page_size=16)
    assert int(prefixes.shared.min()) == 144
    check(queries(slots, 1, d, "f16"), k, v, maps, prefixes, "f16", slots=[0, 4000, 8191])


def test_streams_and_graphs():
    """On another stream; captured once, replayed with other queries, lengths and pages' contents; an eager call beside it."""
    k, v, maps, prefixes = cache([(600, [5, 30, 77]), (200, [1, 1])], 16, 2, 64, "f16")
    q, side, graph = queries(5, 8, 64, "f16"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    call = lambda **o: S.shared_decode(q, k, v, maps.table, maps.lens, prefixes, **o)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    got = call(stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    with torch.cuda.graph(graph, stream=side):
        call(out=out)
    for seed in (5, 6):
        q.copy_(queries(5, 8, 64, "f16", seed))
        maps.lens.sub_(1)
        v.mul_(0.5)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    runtime.call("lc_device_status", None)


def test_two_streams_at_once():
    """Calls that run beside each other keep to workspaces of their own."""
    k, v, maps, prefixes = cache([(2000, [5, 30, 77] * 6), (700, [1, 1])], 16, 2, 64, "f16")
    q = [queries(20, 8, 64, "f16", seed) for seed in range(4)]
    want = [S.shared_decode(x, k, v, maps.table, maps.lens, prefixes) for x in q]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [S.shared_decode(x, k, v, maps.table, maps.lens, prefixes, stream=s.cuda_stream) for x, s in zip(q, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_leaders_that_are_none():
    """A plan whose leaders are no slots shares nothing."""
    k, v, maps, prefixes = cache([(2000, [5, 30, 77] * 6)], 16, 2, 64, "f16")
    q = queries(18, 8, 64, "f16")
    want = S.paged_decode(q, k, v, maps.table, maps.lens).float()
    for no in (-1, 18, 1 << 30):
        plan = S.CachePrefixes(torch.full_like(prefixes.leader, no), torch.full_like(prefixes.shared, 1 << 30), torch.full_like(prefixes.order, no))
        got = S.shared_decode(q, k, v, maps.table, maps.lens, plan).float()
        assert (got - want).abs().max() <= 2.0 ** -10 * want.abs().max()  # each is off by a rounding, its sums by less


def test_refusals():
    k, v, maps, prefixes = cache([(300, [5, 30])], 16, 2, 64, "f16")
    q = queries(2, 8, 64, "f16")
    call = lambda q=q, p=prefixes, **o: S.shared_decode(q, k, v, maps.table, maps.lens, p, **o)  # noqa: E731
    for wrong in (prefixes._replace(leader=prefixes.leader.long()), prefixes._replace(shared=prefixes.shared[:1]),
                  prefixes._replace(order=prefixes.order.cpu()), prefixes._replace(order=ints([0, 0, 1, 1])[::2])):
        with pytest.raises(ValueError, match="prefixes"):
            call(p=wrong)
    with pytest.raises(ValueError, match="out"):
        call(out=torch.zeros(2, 8, 63, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError, match="expanded"):
        call(out=torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda").expand(2, 8, 64))
    with pytest.raises(runtime.LcError, match="scale"):
        call(scale=0.0)


def test_a_loop_of_samples():
    """Prompts, samples of them, tokens one by one: what the cache's operations leave is what the attention takes."""
    c = S.PagedCache(1, 400, 16, 2, 64, 8, 4000, dtype=torch.float16)
    assert 8 * 4000 * 16 * 2 * 64 * 4 > CAPACITY
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    rotary = S.Rotary(64)
    add = ints([300, 170] + [0] * 6)
    c.extend(add)
    c.append(0, None, rand(8, 300, 2, 64), rand(8, 300, 2, 64), add, rotary)
    c.fork(ints([0, 1, 0, 0, 1, 0, -1, 1]))
    prefixes, one = c.prefixes(), ints([1] * 8)
    assert prefixes.shared.tolist() == [288, 160, 288, 288, 160, 288, 0, 160]
    for _ in range(20):
        c.extend(one)
        q = c.append(0, rand(8, 1, 8, 64), rand(8, 1, 2, 64), rand(8, 1, 2, 64), one, rotary)[:, 0]
        o = c.shared_decode(0, q, prefixes)
        p = c.decode(0, q)
        assert float((o.float() - p.float()).abs().max()) <= 3 * 2.0 ** -11
    check(q, c.pool[0], c.pool[1], c.maps, prefixes, "f16")
    c.check()
