"""Rotations and rotated cache writes against exact angles and 64-bit arithmetic."""
import numpy as np
import pytest
import torch

import step_ref as R
from lazy_compiler_b200 import runtime
from lazy_compiler_b200 import serving as S

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def check(got, ref, size, dtype):
    """The output's rounding, u |o|; and of each pair's |a| + |b|, 2^-21: an angle's fraction in f32 (an eighth of a turn at
    most, 2^-26 of it is 2^-25.5 radians), sincospif within 1 ulp (2^-24 of 1), the magnitude's product, one product and
    one sum in f32 (2^-24 each): 4.4 * 2^-24 together.  2^-24: the least f16."""
    got = got.double().cpu().numpy()
    tol = U[dtype] * np.abs(ref) * 1.01 + 2.0 ** -21 * size + (2.0 ** -24 if dtype == "f16" else 0)
    assert got.shape == ref.shape
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - ref).max()))


def normal(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[dtype])


def rotated(x, positions, rotary):
    b, t, h, d = x.shape
    o, size = R.rotate(x.double().cpu().numpy().reshape(b * t, h, d), positions.cpu().numpy().reshape(-1), rotary.frequencies.numpy(),
                       rotary.interleaved, rotary.magnitude)
    return o.reshape(b, t, h, d), size.reshape(b, t, h, d)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,d,rot", [(3, 128, 128), (2, 64, 32), (5, 96, 24), (1, 80, 80), (4, 7, 6), (2, 9, 2), (1, 66, 66), (2, 256, 64), (1, 16, 0), (3, 1024, 1024)])
def test_layouts(dtype, interleaved, heads, d, rot):
    x = normal((2, 5, heads, d), dtype)
    positions = torch.tensor([[0, 1, 2, 777, 100003], [-1, -4096, 2 ** 31 - 1, -2 ** 31, 1 << 20]], dtype=torch.int32, device="cuda")
    rotary = S.Rotary(rot, interleaved=interleaved)
    check(S.rotate(x, positions, rotary), *rotated(x, positions, rotary), dtype)


@pytest.mark.parametrize("batch,tokens,heads", [(1, 1, 1), (1, 1, 40), (300, 1, 3), (3, 333, 2), (1, 4097, 1), (2, 70, 48)])
def test_sizes(batch, tokens, heads):
    x = normal((batch, tokens, heads, 64), "bf16", 1)
    positions = torch.randint(0, 5000, (batch, 1), device="cuda", dtype=torch.int32) + torch.arange(tokens, device="cuda", dtype=torch.int32)
    rotary = S.Rotary(64)
    got = S.rotate(x, positions, rotary)
    pick = torch.arange(tokens, device="cuda")[:: max(1, tokens // 37)]
    check(got[:, pick], *rotated(x[:, pick], positions[:, pick], rotary), "bf16")
    # every token the same way: all of it against the same in f32 from torch's sine and cosine of the exact angles
    if batch * tokens <= 400:
        check(got, *rotated(x, positions, rotary), "bf16")


@pytest.mark.parametrize("dtype,d,shift", [("f16", 64, 0), ("f16", 64, 4), ("f16", 64, 1), ("f32", 32, 2), ("f32", 32, 1), ("bf16", 128, 3)])
def test_strides_and_alignment(dtype, d, shift):
    """Heads before tokens, a slice of a wider row, bases off their alignment."""
    rotary = S.Rotary(d // 2)
    flat = normal((2 * 3 * 7 * (d + 24) + 64,), dtype, 2)
    x = flat[shift:shift + 2 * 3 * 7 * (d + 24)].view(2, 3, 7, d + 24)[..., :d].transpose(1, 2)  # batch, tokens, heads, d
    positions = torch.arange(28, device="cuda", dtype=torch.int32).view(2, 14)[:, ::2]
    out = torch.full((2, 3, 7, d + 8), 3.0, dtype=TYPES[dtype], device="cuda")
    view = out[..., 8 - shift:8 - shift + d].transpose(1, 2)
    ref = rotated(x, positions, rotary)
    got = S.rotate(x, positions, rotary, out=view)
    assert got is view
    check(got, *ref, dtype)
    rest = torch.cat([out[..., :8 - shift], out[..., 8 - shift + d:]], -1)
    assert bool((rest == 3).all())


def test_in_place_and_back():
    x = normal((3, 11, 4, 64), "f32", 3)
    positions = torch.arange(33, device="cuda", dtype=torch.int32).view(3, 11) * 1001
    rotary, before, version = S.Rotary(64, interleaved=True), x.clone(), x._version
    ref = rotated(x, positions, rotary)
    assert S.rotate(x, positions, rotary, out=x) is x and x._version > version
    check(x, *ref, "f32")
    S.rotate(x, -positions, rotary, out=x)
    assert float((x - before).abs().max()) < 1e-5


def test_nothing():
    rotary = S.Rotary(8)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        assert S.rotate(torch.zeros(shape, device="cuda"), torch.zeros(shape[:2], dtype=torch.int32, device="cuda"), rotary).shape == shape


@pytest.mark.parametrize("scaling", ["linear", "base", "bands"])
def test_scaled(scaling):
    x = normal((1, 6, 2, 64), "f32", 4)
    positions = torch.tensor([[0, 1, 100, 8191, 65536, 262143]], dtype=torch.int32, device="cuda")
    rotary = S.Rotary(64, 500000.0, scaling=scaling, factor=8.0, trained=8192)
    assert (scaling == "bands") == (rotary.magnitude != 1)
    check(S.rotate(x, positions, rotary), *rotated(x, positions, rotary), "f32")


def test_refusals():
    x, positions, rotary = torch.zeros(2, 3, 4, 16, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), S.Rotary(16)
    for call in (lambda: S.rotate(x, positions.long(), rotary), lambda: S.rotate(x, positions[:, :2], rotary), lambda: S.rotate(x, positions, S.Rotary(18)),
                 lambda: S.rotate(x, positions, S.Rotary(16, device="cpu")), lambda: S.rotate(x[0], positions, rotary),
                 lambda: S.rotate(x.transpose(2, 3), positions, S.Rotary(4)), lambda: S.rotate(x, positions, rotary, out=x.half()),
                 lambda: S.rotate(x, positions, rotary, out=x[:, :1].expand(-1, 3, -1, -1))):
        with pytest.raises(ValueError):
            call()
    maps = S.CacheMaps(ints([[0], [1]]), ints([1, 1]), ints([1, 1]))
    pages, add = torch.zeros(2, 4, 16, 16, device="cuda"), ints([1, 1])
    k = x[:, :1].contiguous()
    for call in (lambda: S.cache_append(k.half(), k, k, pages, pages, maps, add, rotary), lambda: S.cache_append(None, k, k, pages, pages, maps, add, rotary, out=k),
                 lambda: S.cache_append(None, k, k[..., :8], pages, pages, maps, add, rotary), lambda: S.cache_append(None, k, k, pages, pages[:1].expand(2, -1, -1, -1), maps, add, rotary),
                 lambda: S.cache_append(None, k, k, pages, pages, maps, add.long(), rotary)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- into the cache

def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def appended(q, k, v, pool, table, lens, add, rotary, refused=False):
    """(queries, their sizes, pool, its sizes): the definition token by token; pool float64."""
    pool, size = pool.double().cpu().numpy(), np.zeros(pool.shape)
    page, width = pool.shape[3], table.shape[1]
    o, o_size = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, a) in enumerate(zip(lens.tolist(), add.tolist())):
        new = min(max(a, 0), k.shape[1])
        if refused or n - a < 0 or new == 0:
            continue
        pos = np.arange(n - a, n - a + new)
        f = (rotary.frequencies.numpy(), rotary.interleaved, rotary.magnitude)
        o[s, :new], o_size[s, :new] = R.rotate(q[s, :new].double().cpu().numpy(), pos, *f)
        kk, kk_size = R.rotate(k[s, :new].double().cpu().numpy(), pos, *f)
        vv = v[s, :new].double().cpu().numpy()
        for t, p in enumerate(pos):
            at = int(table[s, p // page]) if p // page < width else -1
            if 0 <= at < pool.shape[1]:
                pool[0, at, :, p % page], pool[1, at, :, p % page], size[0, at, :, p % page] = kk[t], vv[t], kk_size[t]
    return o, o_size, pool, size


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("page,hq,h,d,rot", [(16, 8, 2, 64, 64), (7, 3, 1, 40, 20), (1, 4, 4, 16, 16), (128, 32, 8, 128, 32)])
def test_append(dtype, page, hq, h, d, rot):
    adds, before = [0, 1, 40, 13, 2], [5, 0, 16 * 3 - 1, 100, 31]
    lens, most = [a + b for a, b in zip(adds, before)], 40
    width = -(-max(lens) // page) + 1
    table = torch.full((5, width), -1, dtype=torch.int32)
    held = [-(-n // page) for n in lens]
    order = torch.randperm(sum(held), generator=torch.Generator().manual_seed(0)).int()
    for i, n in enumerate(held):
        table[i, :n] = order[sum(held[:i]):sum(held[:i]) + n]
    if page < 64:
        table[2, held[2] - 1] = -1  # a page that is not there: its tokens are skipped
    maps = S.CacheMaps(table.cuda(), ints(lens), torch.ones(sum(held), dtype=torch.int32, device="cuda"))
    qkv = normal((5, most, hq + 2 * h, d), dtype, 5)
    q, k, v = qkv.split([hq, h, h], 2)
    pool = normal((2, sum(held), h, page, d), dtype, 6)
    rotary = S.Rotary(rot, interleaved=page == 7)
    o, o_size, want, want_size = appended(q, k, v, pool, table, maps.lens, ints(adds), rotary)
    got = S.cache_append(q, k, v, pool[0], pool[1], maps, ints(adds), rotary)
    check(got, o, o_size, dtype)
    check(pool, want, want_size, dtype)
    # the same into the queries themselves: what is not new stays
    rest = q.clone()
    got = S.cache_append(q, k, v, pool[0], pool[1], maps, ints(adds), rotary, out=q)
    assert got is q
    for i, a in enumerate(adds):
        check(q[i, :a], o[i, :a], o_size[i, :a], dtype)
        assert torch.equal(q[i, a:], rest[i, a:])
    check(pool, want, want_size, dtype)
    assert S.cache_append(None, k, v, pool[0], pool[1], maps, ints(adds), rotary) is None
    check(pool, want, want_size, dtype)


def test_append_beyond_the_buffers():
    """Lengths that pass the table, more tokens than there are rows, a negative start."""
    table = ints([[0, 1], [2, 9], [3, -1], [4, 5]])
    lens, add = ints([40, 32, 20, 3]), ints([10, 90, 4, 5])  # slot 1: 90 new of 32; slot 3: 5 new of 3
    q, k, v = (normal((4, 12, h, 32), "f16", 7) for h in (4, 2, 2))
    pool = normal((2, 6, 2, 16, 32), "f16", 8)
    rotary = S.Rotary(32)
    o, o_size, want, size = appended(q, k, v, pool, table.cpu(), lens, add, rotary)
    got = S.cache_append(q, k, v, pool[0], pool[1], S.CacheMaps(table, lens, ints([1] * 6)), add, rotary)
    check(got, o, o_size, "f16")
    check(pool, want, size, "f16")


def test_append_after_a_refusal():
    cache = S.PagedCache(1, 2, 16, 2, 32, 2, 4, dtype=torch.float16)
    rotary = S.Rotary(32)
    q, k, v = (normal((2, 40, h, 32), "f16", 9) for h in (4, 2, 2))
    add = ints([20, 3])
    cache.extend(add)  # three pages of two
    before = cache.pool.clone()
    assert float(cache.append(0, q, k, v, add, rotary).abs().max()) == 0 and torch.equal(cache.pool, before)
    with pytest.raises(RuntimeError, match="1 pages are missing"):
        cache.check()
    add = ints([20, 0])
    cache.extend(add)
    o, o_size, want, size = appended(q, k, v, cache.pool, cache.maps.table.cpu(), cache.maps.lens, add, rotary)
    check(cache.append(0, q, k, v, add, rotary), o, o_size, "f16")
    check(cache.pool, want, size, "f16")
    assert cache.check() == 0


def test_far_offsets():
    """A plane whose pages lie 2^31 elements apart."""
    step = (1 << 31) + 64
    base = torch.zeros(2 * step + 4096, dtype=torch.float16, device="cuda")
    planes = [base.as_strided((3, 1, 16, 32), (step, 512, 32, 1), x) for x in (0, 2048)]
    table, lens, add = ints([[2, 1]]), ints([20]), ints([20])
    q, k, v = (normal((1, 20, 1, 32), "f16", x) for x in (10, 11, 12))
    rotary = S.Rotary(32)
    small = torch.zeros((2, 3, 1, 16, 32), dtype=torch.float16, device="cuda")
    _, _, want, size = appended(q, k, v, small, table.cpu(), lens, add, rotary)
    S.cache_append(q, k, v, planes[0], planes[1], S.CacheMaps(table, lens, ints([0, 1, 1])), add, rotary)
    check(torch.stack([p.clone() for p in planes]), want, size, "f16")


def test_on_a_stream_and_in_a_graph():
    rotary, side = S.Rotary(64), torch.cuda.Stream()
    x = normal((4, 9, 3, 64), "bf16", 13)
    positions = torch.arange(36, device="cuda", dtype=torch.int32).view(4, 9)
    want = S.rotate(x, positions, rotary)
    torch.cuda.synchronize()
    got = S.rotate(x, positions, rotary, stream=side.cuda_stream)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(x)
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.graph(graph, stream=side):
        S.rotate(x, positions, rotary, out=out)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)
    runtime.call("lc_device_status", None)
