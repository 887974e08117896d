"""Serving calls with ``stream=``: what they allocate is that stream's memory, and their results are those of the current stream."""
import pytest

pytestmark = pytest.mark.gpu


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def streams_of(tensors):
    """The stream whose memory each tensor lies in."""
    import torch
    segments = [(s["address"], s["address"] + s["total_size"], s["stream"]) for s in torch.cuda.memory_snapshot()]
    found = []
    for t in tensors:
        (stream,) = [x for lo, hi, x in segments if lo <= t.data_ptr() < hi]
        found.append(stream)
    return found


def test_results_are_memory_of_the_stream_they_are_written_on(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    q, k, v = rand(2, 150, 4, 64), rand(2, 150, 2, 64), rand(2, 150, 2, 64)
    pool, maps = rand(2, 40, 2, 8, 64), S.CacheMaps(ints([[3, 9, 1, -1], [7, -1, -1, -1]]), ints([20, 5]), ints([0] * 40))
    maps.refs[ints([3, 9, 1, 7]).long()] = 1
    add, parent = ints([3, 4]), ints([1, 1])

    def calls(stream):
        """Every operation that returns new tensors; all of them work on copies of the same inputs."""
        kept = pool.clone(), pool.clone()
        old = S.CacheMaps(*(t.clone() for t in maps[:3]))
        if stream:
            torch.cuda.synchronize()  # the copies above
        new = S.cache_extend(maps, add, page_size=8, stream=stream)
        forked = S.cache_fork(kept[0], maps, parent, stream=stream)
        packed = S.cache_compact(kept[1], maps, stream=stream)
        trimmed = S.cache_trim(old, window=4, page_size=8, stream=stream)
        found = [*S.window_attention(q, k, v, window=40, sinks=2, return_lse=True, stream=stream),
                 *S.paged_decode(q[:, 0], pool[0], pool[1], maps.table, maps.lens, return_lse=True, stream=stream), *new, *forked,
                 *packed, trimmed.status]
        return found, [*trimmed[:3], *kept]

    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    made, given = calls(None)
    torch.cuda.synchronize()
    made2, given2 = calls(side.cuda_stream)
    assert torch.cuda.current_stream() == current
    assert set(streams_of(made)) == {current.cuda_stream}
    assert set(streams_of(made2)) == {side.cuda_stream}
    side.synchronize()
    for x, y in zip([*made, *given], [*made2, *given2]):
        assert torch.equal(x, y)
    S.window_attention(q, k, v, stream=0)
    with torch.cuda.stream(side):
        o = S.window_attention(q, k, v, stream=current.cuda_stream)
        assert torch.cuda.current_stream() == side
    assert streams_of([o]) == [current.cuda_stream]


def test_gradients_are_refused_and_writes_are_counted(cuda_device):
    """Inputs that require a gradient, and tensors that autograd has saved before a call wrote them."""
    import torch
    from lazy_compiler_b200 import serving as S
    half = lambda *s: torch.ones(s, dtype=torch.float16, device="cuda")  # noqa: E731
    q, k, pool = half(2, 6, 4, 64), half(2, 6, 2, 64), half(2, 9, 2, 4, 64)
    maps, one = S.CacheMaps(ints([[0, 1], [2, 3]]), ints([6, 5]), ints([1] * 4 + [0] * 5), ints([0, 5])), ints([1, 1])
    g, gp = k.clone().requires_grad_(), pool.clone().requires_grad_()
    for call, name in [
        (lambda: S.window_attention(q, k, k, out=torch.empty_like(q, requires_grad=True)), "out"),
        (lambda: S.cache_write(g[:, :1], k[:, :1], pool[0], pool[1], maps, one), "k"),
        (lambda: S.cache_write(k[:, :1], k[:, :1], pool[0], gp[1], maps, one), "v_pages"),
        (lambda: S.cache_fork(gp, maps, one), "pool"), (lambda: S.cache_compact(gp, maps), "pool"), (lambda: S.cache_copy(gp, one, one), "pool"),
    ]:
        with pytest.raises(ValueError, match=name + ": requires a gradient"):
            call()
    with torch.no_grad():
        S.window_attention(q, g, g)
        S.cache_copy(gp, ints([0]), ints([7]))
    w = torch.ones((), device="cuda", dtype=torch.float16, requires_grad=True)
    out = torch.empty_like(q)
    for saved, call in [
        (out, lambda: S.window_attention(q, k, k, out=out)), (pool, lambda: S.cache_write(k[:, :1], k[:, :1], pool[0], pool[1], maps, one)),
        (pool, lambda: S.cache_fork(pool, maps, one)), (pool, lambda: S.cache_compact(pool, maps)), (pool, lambda: S.cache_copy(pool, one, ints([8, 7]))),
    ]:
        loss = (w * saved).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = maps.lens._version
    S.cache_extend(maps, one, page_size=4, into=maps)
    assert maps.lens._version > before
    with torch.inference_mode():
        S.window_attention(q, k, k, out=torch.empty_like(q))


def test_check_tells_of_a_wait_that_ran_out(cuda_device):
    """A kernel that gave up a bounded wait (the self-test's, which nothing ever ends) is reported by check(), once,
    which waits for its own stream alone."""
    import torch
    from lazy_compiler_b200 import runtime
    from lazy_compiler_b200 import serving as S
    cache = S.PagedCache(1, 4, 4, 1, 64, 1, 2)
    assert cache.check() == 4
    runtime.call("lc_selftest_bounded_wait", 1_000_000, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(runtime.LcError, match="gave up"):
        cache.check()
    assert cache.check() == 4
    side, busy = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)
    busy.record()
    with torch.cuda.stream(side):
        runtime.call("lc_selftest_bounded_wait", 1_000_000, side.cuda_stream)
        with pytest.raises(runtime.LcError, match="gave up"):
            cache.check()
        assert cache.check() == 4
        assert not busy.query()
