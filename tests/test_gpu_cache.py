"""The page operations of the key-value cache against a model on lists: whole numbers and moved values are equal."""
import numpy as np
import pytest

import serving_ref as R

pytestmark = pytest.mark.gpu


def ints(values, shape=None):
    import torch
    t = torch.tensor(values, dtype=torch.int32, device="cuda")
    return t if shape is None else t.reshape(shape)


def maps_of(model, width):
    from lazy_compiler_b200 import serving as S
    return S.CacheMaps(ints(model.table, (len(model.lens), width)), ints(model.lens), ints(model.refs))


def same(model, maps, status, pool=None):
    assert maps.status.tolist() == status
    assert maps.lens.tolist() == model.lens
    assert maps.refs.tolist() == model.refs
    assert maps.table.tolist() == model.table
    if pool is not None:
        np.testing.assert_array_equal(pool.float().cpu().numpy(), model.pool)


def random_cache(rng, slots, width, pages, page, planes=2, heads=2, d=8, dtype="float16", fill=0.5):
    import torch
    pool = torch.from_numpy(rng.integers(-100, 100, (planes, pages, heads, page, d)).astype(np.float32)).cuda().to(getattr(torch, dtype))
    ids, at = rng.permutation(pages), 0
    table, lens, refs = np.full((slots, width), -1), np.zeros(slots, int), np.zeros(pages, int)
    for i in rng.permutation(slots):
        n = int(rng.integers(0, width * page + 1))
        held = -(-n // page)
        if at + held > fill * pages:
            continue
        table[i, :held] = ids[at:at + held]
        refs[ids[at:at + held]] = 1
        lens[i] = n
        at += held
    return pool, R.Pages(table, lens, refs, page, pool.float().cpu().numpy())


SIZES = [(1, 1, 1, 1), (4, 7, 20, 16), (64, 20, 700, 16), (3, 400, 900, 5), (1500, 3, 2500, 8), (40, 30, 70000, 64)]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("seed", [0, 1])
def test_extend(sizes, seed, cuda_device):
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(seed)
    slots, width, pages, page = sizes
    pool, model = random_cache(rng, slots, width, pages, page, planes=1, heads=1, d=1)
    maps = maps_of(model, width)
    room = [width * page - n for n in model.lens]
    adds = [[min(1, r) for r in room], [0] * slots, [int(rng.integers(0, r + 1)) if rng.random() < 0.4 else 0 for r in room],
            [r + (i == slots - 1) for i, r in enumerate(room)], [-1] + [0] * (slots - 1), room]
    for k, add in enumerate(adds):
        status = model.extend(add)
        maps = S.cache_extend(maps, ints(add), page_size=page, into=maps if k % 2 else None)
        same(model, maps, status)


def test_extend_when_pages_run_out(cuda_device):
    from lazy_compiler_b200 import serving as S
    model = R.Pages([[-1] * 9] * 3, [0] * 3, [0] * 20, 4)
    maps = maps_of(model, 9)
    for add in ([36, 36, 9], [36, 36, 8], [0, 0, 1], [0, 0, 0]):
        status = model.extend(add)
        maps = S.cache_extend(maps, ints(add), page_size=4, into=maps)
        same(model, maps, status)
    assert status == [0, 0]


@pytest.mark.parametrize("dtype,heads,d,page,order", [("float16", 2, 128, 16, "hnd"), ("bfloat16", 3, 64, 5, "nhd"), ("float32", 1, 7, 4, "hnd"),
                                                      ("uint8", 2, 5, 3, "nhd"), ("float16", 1, 1, 1, "hnd")])
@pytest.mark.parametrize("most", [1, 70])
def test_write(dtype, heads, d, page, order, most, cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(most)
    slots, width = 6, 120 // page + 1
    pages = slots * width + 3
    shape = (2, pages, heads, page, d) if order == "hnd" else (2, pages, page, heads, d)
    pool = torch.zeros(shape, dtype=getattr(torch, dtype), device="cuda")
    pool = pool if order == "hnd" else pool.transpose(2, 3)
    model = R.Pages([[-1] * width] * slots, [0] * slots, [0] * pages, page, np.zeros((2, pages, heads, page, d), np.float32))
    maps = maps_of(model, width)
    for add in ([0, 1, 1, 0, 1, 1], rng.integers(0, most + 1, slots).tolist(), [min(most, 50)] * slots):
        add = [min(a, most) for a in add]
        k, v = (rng.integers(0, 200, (slots, most, heads, d)).astype(np.float32) for _ in range(2))
        assert model.extend(add)[0] == 0
        model.write(k, v, add)
        maps = S.cache_extend(maps, ints(add), page_size=page, into=maps)
        tk, tv = (torch.from_numpy(x).cuda().to(pool.dtype) for x in (k, v))
        tk = torch.cat([tk, tk], 2)[:, :, heads:]  # a stride that is not the shape's
        S.cache_write(tk, tv, pool[0], pool[1], maps, ints(add))
        same(model, maps, model.status(), pool)


def test_write_skips_what_has_no_page(cuda_device):
    """Lengths beyond the table, pages trimmed away, lengths below the count: nothing else is touched."""
    import torch
    from lazy_compiler_b200 import serving as S
    pool = torch.zeros((2, 4, 1, 4, 16), dtype=torch.float16, device="cuda")
    maps = S.CacheMaps(ints([[0, -1], [1, 2], [77, 3]]), ints([8, 12, 3]), ints([1, 1, 1, 1]))
    k = torch.ones((3, 8, 1, 16), dtype=torch.float16, device="cuda")
    S.cache_write(k, k, pool[0], pool[1], maps, ints([8, 8, 5]))
    assert pool[:, 0].eq(1).all() and pool[:, 1].eq(0).all() and pool[:, 2].eq(1).all() and pool[:, 3].eq(0).all()


@pytest.mark.parametrize("sizes", SIZES[:5])
@pytest.mark.parametrize("dtype,d", [("float16", 8), ("bfloat16", 3), ("float32", 128)])
def test_fork(sizes, dtype, d, cuda_device):
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(d)
    slots, width, pages, page = sizes
    pool, model = random_cache(rng, slots, width, pages, page, planes=4, d=d, dtype=dtype)
    maps = maps_of(model, width)
    for parent in (list(range(slots)), rng.integers(0, slots, slots).tolist(), rng.integers(-1, min(slots, 3), slots).tolist(),
                   [0] * (slots - 1) + [slots], [-2] + [0] * (slots - 1), [int(np.argmax(model.lens))] * slots, [-1] * slots):
        status = model.fork(parent)
        new = S.cache_fork(pool, maps, ints(parent))
        same(model, new, status, pool)
        maps = new


def test_fork_when_pages_run_out(cuda_device):
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(0)
    pool, _ = random_cache(rng, 1, 1, 4, 4, planes=2)
    model = R.Pages([[3, 1], [-1, -1], [-1, -1], [-1, -1]], [6, 0, 0, 0], [0, 1, 0, 1], 4, pool.float().cpu().numpy())
    maps = maps_of(model, 2)
    for parent in ([0, 0, 0, 0], [0, 0, -1, 0], [1, -1, -1, 0]):
        status = model.fork(parent)
        maps = S.cache_fork(pool, maps, ints(parent))
        same(model, maps, status, pool)


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype,d", [("float16", 8), ("uint8", 1)])
def test_compact_release_and_trim(sizes, dtype, d, cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(d)
    slots, width, pages, page = sizes
    pool, model = random_cache(rng, slots, width, pages, page, planes=2, heads=1, d=d, dtype="float16", fill=0.8)
    if dtype == "uint8":
        model.pool = np.abs(model.pool)
        pool = pool.abs().to(torch.uint8)
    maps = maps_of(model, width)
    for k in range(3):
        parent = rng.integers(-1, slots, slots).tolist()  # shared pages
        status = model.fork(parent)
        maps = S.cache_fork(pool, maps, ints(parent))
        same(model, maps, status, pool)
        status = model.compact()
        maps = S.cache_compact(pool, maps, into=maps if k % 2 else None)
        same(model, maps, status, pool)
        assert status[1] == pages - sum(n > 0 for n in model.refs)
        window, sinks = int(rng.integers(1, 2 * page + 2)), int(rng.integers(0, 2 * page))
        status = model.trim(window, sinks)
        maps = S.cache_trim(maps, window=window, sinks=sinks, page_size=page)
        same(model, maps, status)
        gone = rng.integers(0, 2, slots).tolist()
        status = model.release(gone)
        maps = S.cache_release(maps, ints(gone), page_size=page)
        same(model, maps, status)
        status = model.compact()
        maps = S.cache_compact(pool, maps, into=maps)
        same(model, maps, status, pool)


@pytest.mark.parametrize("heads,page,d,dtype", [(2, 16, 64, "float16"), (1, 3, 5, "uint8"), (3, 1, 8, "float32")])
def test_copy(heads, page, d, dtype, cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    pool = torch.randint(0, 100, (6, 50, heads, page, d), device="cuda").to(getattr(torch, dtype))
    want = pool.clone()
    ids = np.random.default_rng(0).permutation(50)
    src, dst = ids[:20].tolist(), ids[20:40].tolist()
    want[:, dst] = want[:, src]
    S.cache_copy(pool, ints(src + [-1, 3, 50]), ints(dst + [3, 50, 3]))
    assert torch.equal(pool, want)
    S.cache_copy(pool, ints([]), ints([]))
    part = torch.zeros((6, 50, heads + 1, page, d), dtype=pool.dtype, device="cuda")[:, :, 1:]
    part.copy_(pool)
    S.cache_copy(part, ints([ids[0]]), ints([ids[45]]))
    want[:, ids[45]] = want[:, ids[0]]
    assert torch.equal(part, want)


def test_paged_cache_steps_in_a_graph(cuda_device):
    """Extend, write and decode of every step replayed from one captured graph; samples fork, windows are trimmed."""
    import torch
    from lazy_compiler_b200 import serving as S
    slots, h, hq, d, page, width, window, sinks = 3, 2, 4, 64, 8, 40, 24, 3
    cache = S.PagedCache(2, 80, page, h, d, slots, width, dtype=torch.float16)
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    add = ints([30, 7, 0])
    k, v = rand(2, slots, 30, h, d), rand(2, slots, 30, h, d)
    cache.extend(add)
    for layer in range(2):
        cache.write(layer, k[layer], v[layer], add)
    keys = [[[k[l, i, :n].float(), v[l, i, :n].float()] for i, n in enumerate((30, 7, 0))] for l in range(2)]
    cache.fork(ints([0, 1, 0]))
    for layer in keys:
        layer[2] = list(layer[0])
    assert cache.check() == 80 - 4 - 1 - 1
    one = ints([1, 1, 1])
    new_k, new_v, q = rand(2, slots, 1, h, d), rand(2, slots, 1, h, d), rand(2, slots, hq, d)
    outs = torch.empty((2, slots, hq, d), dtype=torch.float16, device="cuda")

    def step():
        cache.extend(one)
        for layer in range(2):
            cache.write(layer, new_k[layer], new_v[layer], one)
            cache.decode(layer, q[layer], window=window, sinks=sinks, out=outs[layer])
        cache.trim(window, sinks)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = None
    for t in range(40):
        new_k.copy_(rand(2, slots, 1, h, d)), new_v.copy_(rand(2, slots, 1, h, d)), q.copy_(rand(2, slots, hq, d))
        side.wait_stream(torch.cuda.current_stream())
        if t == 0:
            with torch.cuda.stream(side):
                step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for l in range(2):
            for i in range(slots):
                keys[l][i] = [torch.cat([a, b[l, i].float()]) for a, b in zip(keys[l][i], (new_k, new_v))]
                ks, vs = keys[l][i]
                js = torch.from_numpy(R.seen(len(ks) - 1, len(ks), window, sinks)).cuda()
                for y in range(hq):
                    s = ks[js, y // 2].double() @ q[l, i, y].double() / 8
                    ref = torch.softmax(s, 0) @ vs[js, y // 2].double()
                    assert (outs[l, i, y].double() - ref).abs().max() < 4e-3
    # 24 tokens and the sinks' page are what is left of each, in at most 1 + 4 pages
    free = cache.check()
    assert free >= 80 - 5 * slots
    cache.compact()
    assert cache.check() == free and int(cache.maps.table.max()) == 80 - free - 1
    cache.release(one)
    assert cache.check() == 80
    with pytest.raises(RuntimeError, match="argument is out of range"):
        cache.extend(ints([page * width + 1, 0, 0]))
        cache.check()
    with pytest.raises(RuntimeError, match="40 pages are missing"):
        cache.extend(ints([page * width] * 3))
        cache.check()


def test_pages_beyond_32_bit_offsets(cuda_device):
    """Copies, forks, compaction and writes four billion bytes and elements into the pool."""
    import torch
    from lazy_compiler_b200 import serving as S
    pages, page, h, d = 40000, 16, 8, 64
    pool = torch.zeros((14, pages, h, page, d), dtype=torch.float16, device="cuda")  # 4.6e9 elements
    last = torch.randn((14, 2, h, page, d), device="cuda").half()
    pool[:, pages - 2:] = last
    S.cache_copy(pool, ints([pages - 2]), ints([5]))
    assert torch.equal(pool[:, 5], last[:, 0]) and pool[:, 4].eq(0).all()
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[pages - 2:] = 1
    maps = S.CacheMaps(ints([[pages - 1, pages - 2], [-1, -1]]), ints([20, 0]), refs)
    new = S.cache_fork(pool, maps, ints([0, 0]))
    assert new.table.tolist() == [[pages - 1, pages - 2], [pages - 1, 0]] and torch.equal(pool[:, 0, :, :4], last[:, 0, :, :4])
    new = S.cache_compact(pool, new)
    assert new.table.tolist() == [[2, 1], [2, 0]] and torch.equal(pool[:, 1], last[:, 0]) and torch.equal(pool[:, 2], last[:, 1])
    k = torch.randn((2, 3, h, d), device="cuda").half()
    maps = S.CacheMaps(ints([[pages - 3, -1], [1, pages - 5]]), ints([3, 18]), refs)
    S.cache_write(k, k, pool[12], pool[13], maps, ints([3, 2]))
    for plane in (12, 13):
        assert torch.equal(pool[plane, pages - 3, :, :3], k[0].transpose(0, 1)) and torch.equal(pool[plane, pages - 5, :, :2], k[1, :2].transpose(0, 1))


def test_refusals_of_maps(cuda_device):
    import torch
    from lazy_compiler_b200 import runtime
    from lazy_compiler_b200 import serving as S
    pool = torch.zeros((2, 6, 2, 4, 8), device="cuda")
    maps = S.CacheMaps(ints([[0, 1], [2, -1]]), ints([6, 3]), ints([1, 1, 1, 0, 0, 0]))
    add, k = ints([1, 1]), torch.zeros((2, 1, 2, 8), device="cuda")
    small = S.CacheMaps(maps.table[:1], maps.lens[:1], maps.refs)
    refused = [
        (lambda: S.cache_extend(maps, add[:1], page_size=4), ValueError, "add: shape"),
        (lambda: S.cache_extend(maps, add.long(), page_size=4), ValueError, "add: int64"),
        (lambda: S.cache_extend(maps, add, page_size=0), runtime.LcError, "size"),
        (lambda: S.cache_extend(maps, add, page_size=4, into=small), ValueError, "into"),
        (lambda: S.cache_extend(maps._replace(lens=maps.lens[:1]), add, page_size=4), ValueError, "maps: shape"),
        (lambda: S.cache_extend(maps._replace(table=maps.table.t()), add, page_size=4), ValueError, "contiguous"),
        (lambda: S.cache_extend(maps._replace(refs=maps.refs.cpu()), add, page_size=4), ValueError, "cpu"),
        (lambda: S.cache_write(k, k, pool[0], pool[1, :5], maps, add), ValueError, "v_pages: shape"),
        (lambda: S.cache_write(k, k.half(), pool[0], pool[1], maps, add), ValueError, "v: float16"),
        (lambda: S.cache_write(k[:1], k[:1], pool[0], pool[1], maps, add), ValueError, "k: shape"),
        (lambda: S.cache_fork(pool, maps, add, into=maps), runtime.LcError, "overwrite"),
        (lambda: S.cache_fork(pool[:, :5], maps, add), ValueError, "pool"),
        (lambda: S.cache_fork(pool.transpose(3, 4), maps, add), ValueError, "contiguous"),
        (lambda: S.cache_fork(pool[:, :1].expand(-1, 6, -1, -1, -1), maps, add), ValueError, "pool: axis 1 is expanded"),
        (lambda: S.cache_write(k, k, pool[0], pool[1, :1].expand(6, -1, -1, -1), maps, add), ValueError, "v_pages: axis 0"),
        (lambda: S.cache_compact(pool[0], maps), ValueError, "pool"),
        (lambda: S.cache_trim(maps, window=0, page_size=4), runtime.LcError, "window"),
        (lambda: S.cache_release(maps, add[:1], page_size=4), ValueError, "gone: shape"),
        (lambda: S.cache_copy(pool, add, add[:1]), ValueError, "dst: shape"),
    ]
    for call, kind, text in refused:
        with pytest.raises(kind, match=text):
            call()


def test_nothing_is_written_after_a_refused_extend(cuda_device):
    """Where room was refused the newest positions are those of older tokens, some of them in pages that samples share."""
    import torch
    from lazy_compiler_b200 import serving as S
    cache = S.PagedCache(1, 6, 4, 1, 16, 3, 8, dtype=torch.float16)
    cache.extend(ints([8, 0, 12]))
    old, new = (torch.full((3, 12, 1, 16), x, dtype=torch.float16, device="cuda") for x in (1.0, 2.0))
    cache.write(0, old, old, ints([8, 0, 12]))
    cache.fork(ints([0, 0, 2]))  # 5 pages of 6 in use, 2 of them by two slots
    assert cache.check() == 1
    before = cache.pool.clone()
    one = ints([1, 1, 1])
    refused = S.cache_extend(cache.maps, one, page_size=4)  # 3 pages wanted
    assert refused.status.tolist() == [2, 1]
    S.cache_write(new, new, cache.pool[0], cache.pool[1], refused, one)
    cache.extend(one)
    cache.write(0, new[:, :1], new[:, :1], one)
    assert torch.equal(cache.pool, before)
    with pytest.raises(RuntimeError, match="2 pages are missing"):
        cache.check()
    one = ints([0, 1, 0])
    cache.extend(one)
    cache.write(0, new[:, :1], new[:, :1], one)
    assert cache.check() == 0 and int((cache.pool != before).sum()) == 2 * 16


@pytest.mark.parametrize("captured", [False, True])
def test_a_refusal_is_told_whatever_came_after_it(captured, cuda_device):
    """A loop that looks at its steps' end only: the refused step's tokens are written nowhere, and check() says so."""
    import torch
    from lazy_compiler_b200 import serving as S
    cache = S.PagedCache(1, 7, 4, 1, 16, 3, 8, dtype=torch.float16)
    side = torch.cuda.Stream()
    start = ints([8, 0, 12])
    old, new = (torch.full((3, 12, 1, 16), x, dtype=torch.float16, device="cuda") for x in (1.0, 2.0))
    add, gone = ints([0, 0, 0]), ints([0, 0, 1])

    def step():
        cache.extend(add)
        cache.trim(100)
        cache.write(0, new[:, :1], new[:, :1], add)
        cache.release(gone)
        cache.compact()

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.extend(start)
        cache.write(0, old, old, start)
        cache.fork(ints([0, 0, 2]))
        gone.zero_()
        step()
        run = step
        if captured:
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            run = graph.replay
        assert cache.check() == 2
        before, table = cache.pool.clone(), cache.maps.table.clone()
        add.copy_(ints([1, 1, 1]))  # a page each, and 2 are free
        run()
        assert torch.equal(cache.pool, before) and torch.equal(cache.maps.table, table) and cache.maps.status.tolist() == [0, 2]
        add.copy_(ints([0, 1, 0]))  # this one fits
        gone.copy_(ints([0, 0, 1]))
        run()
        assert cache.maps.lens.tolist() == [8, 9, 0]
        with pytest.raises(RuntimeError, match="1 pages are missing"):
            cache.check()
        assert cache.check() == 4


def test_a_refused_fork_is_told_too(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    cache = S.PagedCache(1, 2, 4, 1, 16, 4, 2, dtype=torch.float16)
    cache.extend(ints([3, 0, 0, 0]))
    cache.fork(ints([0, 0, 0, 0]))
    cache.fork(ints([0, -1, -1, 7]))
    cache.trim(1)
    with pytest.raises(RuntimeError, match="2 pages are missing"):
        cache.check()
    assert cache.check() == 1 and cache.maps.lens.tolist() == [3, 0, 0, 0]
    refusals = ints([0, 0])
    first = S.cache_extend(cache.maps, ints([9, 0, 0, 0]), page_size=4, refusals=refusals)
    S.cache_extend(cache.maps, ints([1, 8, 0, 0]), page_size=4, refusals=refusals)
    S.cache_fork(cache.pool, cache.maps, ints([0, 0, 0, 0]), refusals=refusals)
    assert first.status.tolist() == [-1, 1] and refusals.tolist() == [-1, 1]
    with pytest.raises(ValueError, match="refusals: shape"):
        S.cache_extend(cache.maps, ints([0, 0, 0, 0]), page_size=4, refusals=refusals[:1])


@pytest.mark.parametrize("fork_captured", [False, True])
def test_a_captured_step_goes_on_after_a_fork(fork_captured, cuda_device):
    """Beams: a fork between the replays of one captured step, or inside it, as if every step were made anew."""
    import torch
    from lazy_compiler_b200 import serving as S
    rng = np.random.default_rng(0)
    slots, h, d, page, width, pages = 4, 2, 64, 4, 12, 40
    model = R.Pages([[-1] * width for _ in range(slots)], [0] * slots, [0] * pages, page, np.zeros((2, pages, h, page, d), np.float32))
    cache = S.PagedCache(1, pages, page, h, d, slots, width, dtype=torch.float16)
    k, v = (torch.zeros((slots, 9, h, d), dtype=torch.float16, device="cuda") for _ in range(2))
    q, out = torch.randn((slots, 4, d), device="cuda").half(), torch.empty((slots, 4, d), dtype=torch.float16, device="cuda")
    parent, one = ints(list(range(slots))), ints([1] * slots)

    def tokens(most):
        new = [rng.integers(-9, 9, (slots, most, h, d)).astype(np.float32) for _ in range(2)]
        for x, y in zip((k, v), new):
            x[:, :most] = torch.from_numpy(y).cuda()
        return new

    def fork():
        cache.fork(parent, stream=side.cuda_stream)

    def step():
        if fork_captured:
            fork()
        cache.extend(one)
        cache.write(0, k[:, :1], v[:, :1], one)
        cache.decode(0, q, out=out)

    side, graph, maps = torch.cuda.Stream(), torch.cuda.CUDAGraph(), cache.maps
    add = [9, 0, 6, 0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        new = tokens(9)
        cache.extend(ints(add))
        cache.write(0, k, v, ints(add))
        model.extend(add)
        model.write(*new, add)
        for t, parents in enumerate([[0, 2, 2, 0], [0, 1, 2, 3], [3, 3, 1, 0], [1, 1, 1, 1], [0, 0, 2, -1], [2, 2, 2, 2]]):
            parent.copy_(ints(parents))
            if not fork_captured:
                fork()
            new = tokens(1)
            if t == 0:
                step()
                side.synchronize()
                with torch.cuda.graph(graph, stream=side):
                    step()
            else:
                graph.replay()
            assert model.fork(parents)[0] == 0
            status = model.extend([1] * slots)
            model.write(*new, [1] * slots)
            same(model, cache.maps, status, cache.pool)
            assert cache.maps is maps and cache.check() == status[1]
            pool = torch.from_numpy(model.pool).cuda().half()
            want = S.paged_decode(q, pool[0], pool[1], ints(model.table), ints(model.lens))
            assert torch.equal(out, want)


def test_fork_of_maps_that_the_caller_put_in(cuda_device):
    """Maps made by the functions and assigned to a cache are what its fork goes on from."""
    import torch
    from lazy_compiler_b200 import serving as S
    cache = S.PagedCache(1, 8, 4, 1, 16, 2, 4, dtype=torch.float16)
    first = cache.maps
    cache.maps = S.cache_extend(cache.maps, ints([5, 0]), page_size=4)
    cache.fork(ints([0, 0]))
    assert cache.maps is first and cache.maps.lens.tolist() == [5, 5] and cache.maps.table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1]]
    assert cache.check() == 5
