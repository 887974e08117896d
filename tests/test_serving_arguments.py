"""What the serving operators refuse, on the host (no device work, so these run without a GPU)."""
import ctypes

import pytest
import torch

from lazy_compiler_b200 import runtime
from lazy_compiler_b200 import serving as S

P = ctypes.c_void_p(4096)
NULL = ctypes.c_void_p(0)


def strides(n):
    return (ctypes.c_int64 * n)(*[16] * n)


def window(dtype=1, q=P, k=P, o=P, batch=1, s_q=4, s_kv=4, hq=2, h=1, d=64, st=None, win=0, sinks=0, scale=1.0):
    runtime.call("lc_window_attention", dtype, q, k, P, o, NULL, NULL, NULL, batch, s_q, s_kv, hq, h, d, strides(12) if st is None else st,
                 win, sinks, scale, NULL)


def decode(dtype=1, q=P, lens=P, table=P, slots=1, width=2, pages=4, page=16, hq=2, h=1, d=64, st=None, win=0, sinks=0, scale=1.0):
    runtime.call("lc_paged_decode", dtype, q, P, P, P, NULL, table, lens, slots, width, pages, page, hq, h, d, strides(11) if st is None else st,
                 win, sinks, scale, NULL)


def fork(table_out=ctypes.c_void_p(8192), lens_out=ctypes.c_void_p(8192), refs_out=ctypes.c_void_p(8192), status=P, planes=1, heads=1,
         token=16, st=None, pool=P, page=16):
    runtime.call("lc_cache_fork", pool, planes, heads, token, strides(3) if st is None else st, P, table_out, P, lens_out, P, refs_out, P,
                 status, 4, 4, 4, page, NULL)


INVALID = [
    lambda: window(dtype=0), lambda: window(dtype=9), lambda: window(batch=-1), lambda: window(hq=3, h=2), lambda: window(d=0),
    lambda: window(h=0), lambda: window(q=NULL), lambda: window(k=NULL), lambda: window(o=NULL), lambda: window(st=NULL), lambda: window(win=-1),
    lambda: window(sinks=-1), lambda: window(scale=0.0), lambda: window(scale=float("nan")), lambda: window(scale=float("inf")),
    lambda: decode(dtype=0), lambda: decode(slots=-1), lambda: decode(page=0), lambda: decode(hq=3, h=2), lambda: decode(lens=NULL),
    lambda: decode(table=NULL), lambda: decode(q=NULL), lambda: decode(st=NULL), lambda: decode(win=-2), lambda: decode(scale=-1.0),
    lambda: fork(table_out=P), lambda: fork(lens_out=P), lambda: fork(refs_out=P), lambda: fork(status=NULL), lambda: fork(planes=-1),
    lambda: fork(heads=0), lambda: fork(token=0), lambda: fork(st=NULL), lambda: fork(pool=NULL), lambda: fork(page=0),
    lambda: runtime.call("lc_cache_extend", P, P, P, P, P, P, NULL, P, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_extend", P, P, P, P, P, P, P, NULL, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_extend", P, P, P, P, P, P, P, P, -4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_write", P, P, NULL, P, P, P, P, 1, 1, 1, 1, 16, 1, 16, strides(12), NULL),
    lambda: runtime.call("lc_cache_write", P, P, P, P, P, P, P, 1, 1, 1, 1, 16, 0, 16, strides(12), NULL),
    lambda: runtime.call("lc_cache_release", P, P, P, NULL, 0, 0, P, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_release", P, P, P, NULL, 8, -1, P, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_release", P, NULL, P, P, 0, 0, P, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_compact", P, 1, 1, 16, strides(3), P, P, P, P, NULL, P, P, 4, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_copy", P, 1, 1, 16, strides(3), P, P, -1, 4, 16, NULL),
    lambda: runtime.call("lc_cache_copy", P, 1, 1, 16, strides(3), NULL, P, 1, 4, 16, NULL),
]


@pytest.mark.parametrize("case", range(len(INVALID)))
def test_invalid_arguments(case):
    with pytest.raises(runtime.LcError) as err:
        INVALID[case]()
    assert err.value.status == -1 and err.value.message


UNSUPPORTED = [
    lambda: window(d=264), lambda: window(batch=1 << 17), lambda: window(s_q=1 << 31), lambda: decode(d=257), lambda: decode(width=1 << 30),
    lambda: decode(slots=1 << 21), lambda: fork(token=1 << 20),
    lambda: runtime.call("lc_cache_fork", P, 1, 1, 16, strides(3), P, P, P, P, P, P, P, P, 8193, 4, 4, 16, NULL),
    lambda: runtime.call("lc_cache_extend", P, P, P, P, P, P, P, P, 1 << 24, 4, 4, 16, NULL),
]


@pytest.mark.parametrize("case", range(len(UNSUPPORTED)))
def test_unsupported_sizes(case):
    with pytest.raises(runtime.LcError) as err:
        UNSUPPORTED[case]()
    assert err.value.status == -5 and err.value.message


def test_elements_off_their_alignment():
    with pytest.raises(runtime.LcError) as err:
        window(q=ctypes.c_void_p(4097))
    assert err.value.status == -2


def test_nothing_to_do_is_no_error():
    window(batch=0, q=NULL)
    window(s_q=0, q=NULL)
    decode(slots=0, q=NULL)
    runtime.call("lc_cache_copy", NULL, 0, 1, 16, strides(3), NULL, NULL, 0, 0, 16, NULL)
    runtime.call("lc_cache_write", NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, 1, 1, 1, 16, 1, 16, strides(12), NULL)


def test_tensors_off_the_device_or_of_another_type():
    q = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="float32 is not"):
        S.window_attention(q, q, q)
    q = q.half()
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.window_attention(q, q, q)
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.paged_decode(q[0], q, q, torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    maps = S.CacheMaps(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.cache_extend(maps, maps.lens, page_size=16)
    with pytest.raises(ValueError, match="at least 1"):
        S.PagedCache(0, 1, 1, 1, 1, 1, 1)


def test_limits_of_the_counts():
    """A table whose entries, or a scale whose product with log2 e, would leave 32 bits."""
    for call, status in [
        (lambda: runtime.call("lc_cache_extend", P, P, P, P, P, P, P, P, 1 << 12, 1 << 19, 4, 16, NULL), -5),
        (lambda: runtime.call("lc_cache_release", P, P, P, P, 0, 0, P, 1 << 20, 1 << 11, 4, 16, NULL), -5),
        (lambda: window(scale=2.5e38), -1), (lambda: decode(scale=2.5e38), -1),
    ]:
        with pytest.raises(runtime.LcError) as err:
            call()
        assert err.value.status == status


def test_numbers_in_the_refusals():
    """The extension's messages hold sizes: with a libstdc++ of its own in the module, writing one faulted."""
    from lazy_compiler_b200 import _serving
    with pytest.raises(ValueError, match="expected 11 arguments, got 1"):
        _serving.window_attention(1)
    with pytest.raises(TypeError):
        _serving.bind(*[1.5] * 8)


def test_what_requires_a_gradient():
    """Nothing has a gradient, and no one that is asked for is dropped without a word."""
    q, k = torch.zeros(1, 4, 2, 64, dtype=torch.half), torch.zeros(1, 4, 2, 64, dtype=torch.half)
    table, lens, refs = (torch.zeros(n, dtype=torch.int32) for n in ((1, 2), 1, 4))
    g, pages = (torch.zeros(s, dtype=torch.half, requires_grad=True) for s in ((1, 4, 2, 64), (4, 2, 16, 64)))
    for call, name in [
        (lambda: S.window_attention(g, k, k), "q"), (lambda: S.window_attention(q, g, k), "k"), (lambda: S.window_attention(q, k, g), "v"),
        (lambda: S.paged_decode(g[0], pages.detach(), pages.detach(), table, lens), "q"),
        (lambda: S.paged_decode(q[0], pages, pages.detach(), table, lens), "k_pages"),
        (lambda: S.paged_decode(q[0], pages.detach(), pages, table, lens), "v_pages"),
    ]:
        with pytest.raises(ValueError, match=name + ": requires a gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA devices only"):
            call()


@pytest.mark.parametrize("heads,row_bytes,status", [(1 << 16, 1 << 12, -5), ((1 << 16) - 1, 1 << 12, 0), (1 << 16, (1 << 12) - 1, 0)])
def test_write_counts_that_leave_32_bits(heads, row_bytes, status):
    """Eight tokens of 2^28 bytes: their pieces are counted in an int.  (No slots: what fits launches nothing.)"""
    write = lambda slots: runtime.call("lc_cache_write", P, P, P, P, P, P, P, slots, 1, 1, 1, 16, heads, row_bytes, strides(12), NULL)  # noqa: E731
    if not status:
        write(0)
        return
    with pytest.raises(runtime.LcError) as err:
        write(0)
    assert err.value.status == status
