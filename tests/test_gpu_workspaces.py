"""The workspaces that the library keeps for a stream, and the CUDA graphs that hold their addresses."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def is_device(address):
    from cuda.bindings import runtime as cudart
    err, attributes = cudart.cudaPointerGetAttributes(address)
    return err == cudart.cudaError_t.cudaSuccess and attributes.type == cudart.cudaMemoryType.cudaMemoryTypeDevice


def words(graph):
    """The 8-byte words of the parameters of a graph's kernels."""
    from cuda.bindings import driver, runtime as cudart
    raw = cudart.cudaGraph_t(graph.raw_cuda_graph())
    err, _, count = cudart.cudaGraphGetNodes(raw)
    err, nodes, count = cudart.cudaGraphGetNodes(raw, count)
    found = []
    for node in nodes:
        if cudart.cudaGraphNodeGetType(node)[1] != cudart.cudaGraphNodeType.cudaGraphNodeTypeKernel:
            continue
        err, params = driver.cuGraphKernelNodeGetParams(driver.CUgraphNode(int(node)))
        assert err == driver.CUresult.CUDA_SUCCESS
        at = ctypes.cast(int(params.kernelParams), ctypes.POINTER(ctypes.c_void_p))
        for k in range(64):
            err, _, size = driver.cuFuncGetParamInfo(params.func, k)
            if err != driver.CUresult.CUDA_SUCCESS:
                break
            found += (ctypes.c_uint64 * (size // 8)).from_address(at[k])
    return found


def test_a_captured_step_keeps_its_workspaces(cuda_device):
    """Larger calls on the capturing stream leave what the graph uses alive.  This is seen on the host, before the graph
    runs again; then its results are those of the same step uncaptured."""
    import torch
    from lazy_compiler_b200 import serving as S
    slots, h, d, page, width, pages = 3, 2, 128, 16, 200, 5000
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    first, one = ints([3000, 40, 0]), ints([1, 1, 1])
    k, v, q = rand(slots, 3000, h, d), rand(slots, 3000, h, d), rand(slots, 4, d)
    caches = [S.PagedCache(1, pages, page, h, d, slots, width, dtype=torch.float16) for _ in range(2)]
    outs = [torch.full((slots, 4, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]

    def step(x):
        caches[x].extend(one)
        caches[x].write(0, k[:, :1], v[:, :1], one)
        caches[x].decode(0, q, out=outs[x])

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph(keep_graph=True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for cache in caches:
            cache.extend(first)
            cache.write(0, k, v, first)
        step(0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(0)
    held = [w for w in words(graph) if is_device(w)]
    assert len(held) > 20
    many = 400  # slots of a larger decode, with more counters, and of maps with more ranks
    with torch.cuda.stream(side):
        caches[0].compact()
        big = S.PagedCache(1, 4 * pages, page, h, d, many, width, dtype=torch.float16)
        big.extend(ints([100] * many))
        big.decode(0, q.repeat(134, 1, 1)[:many])
        big.compact()
    torch.cuda.synchronize()
    assert all(is_device(w) for w in held)
    graph.replay()
    torch.cuda.synchronize()
    step(1)
    step(1)
    assert caches[0].check() == caches[1].check()
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(caches[0].maps.lens, caches[1].maps.lens) and torch.equal(caches[0].maps.refs, caches[1].maps.refs)


def test_counters_are_zero_on_a_stream_beside_a_busy_default_stream(cuda_device):
    """A stream's first call, while the default stream has work queued: nothing of it waits for that work, and its
    counters read zero although the memory they lie in held something before."""
    import torch
    from cuda.bindings import runtime as cudart
    from lazy_compiler_b200 import runtime
    from lazy_compiler_b200 import serving as S
    # 30 slots of one long and 29 short caches: the long one's parts are counted and joined by the last of its CTAs
    slots, page, h, d, n = 30, 16, 8, 128, 6000
    width = n // page
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(2 * width, h, page, d, generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn(slots, 32, d, generator=g, device="cuda").half()
    table = torch.randint(0, 2 * width, (slots, width), generator=g, device="cuda", dtype=torch.int32)
    lens = ints([n] + [100] * (slots - 1))
    x = torch.randn(1 << 22, generator=g, device="cuda")
    want = S.paged_decode(q, k, v, table, lens, return_lse=True)
    want_sum = torch.empty(1, device="cuda")
    runtime.call("lc_sum_f32", ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(want_sum.data_ptr()), x.numel(), None)
    # memory as the workspaces will find it, not zero
    dirty = [cudart.cudaMalloc(size)[1] for size in (slots * h * 4, 1 << 14, 1 << 16) for _ in range(4)]
    for at, size in zip(dirty, [slots * h * 4] * 4 + [1 << 14] * 4 + [1 << 16] * 4):
        cudart.cudaMemset(at, 0xFF, size)
    torch.cuda.synchronize()
    for at in dirty:
        cudart.cudaFree(at)
    got = [torch.full_like(w, float("nan")) for w in want] + [torch.full_like(want_sum, float("nan"))]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(2_000_000_000)
    busy.record()
    with torch.cuda.stream(side):
        for _ in range(3):
            o, lse = S.paged_decode(q, k, v, table, lens, out=got[0], return_lse=True)
        handle = ctypes.c_void_p(side.cuda_stream)
        for _ in range(3):
            runtime.call("lc_sum_f32", ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(got[2].data_ptr()), x.numel(), handle)
    side.synchronize()
    waited = busy.query()
    torch.cuda.synchronize()
    assert not waited
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and torch.equal(got[2], want_sum)
