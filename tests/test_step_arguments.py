"""What the operators around the serving attention refuse, on the host (no device work, so these run without a GPU)."""
import ctypes
import math

import pytest
import torch

from lazy_compiler_b200 import _serving, runtime
from lazy_compiler_b200 import serving as S

P = ctypes.c_void_p(4096)
NULL = ctypes.c_void_p(0)


def strides(n):
    return (ctypes.c_int64 * n)(*[16] * n)


def rotate(dtype=1, x=P, out=P, positions=P, turns=P, batch=1, tokens=2, heads=3, d=64, rot=64, magnitude=1.0, st=None):
    runtime.call("lc_rotate", dtype, x, out, positions, turns, batch, tokens, heads, d, rot, 0, magnitude, strides(8) if st is None else st, NULL)


def append(dtype=1, q=P, k=P, v=P, out=P, kp=P, vp=P, table=P, lens=P, add=P, turns=P, slots=1, most=2, width=4, pages=8, page=16, hq=2,
           h=1, d=64, rot=64, magnitude=1.0, st=None):
    runtime.call("lc_cache_append", dtype, q, k, v, out, kp, vp, table, lens, add, NULL, turns, slots, most, width, pages, page, hq, h, d,
                 rot, 0, magnitude, 1, strides(18) if st is None else st, NULL)


def prefixes(table=P, lens=P, leader=P, shared=P, order=P, slots=4, width=4, pages=8, page=16):
    runtime.call("lc_cache_prefixes", table, lens, leader, shared, order, slots, width, pages, page, NULL)


def sample(dtype=0, logits=P, uniform=P, token=P, rows=2, vocab=10):
    runtime.call("lc_sample", dtype, logits, uniform, NULL, NULL, NULL, NULL, 1.0, 0, 1.0, 0.0, token, NULL, rows, vocab, 16, NULL)


def shared(dtype=1, q=P, o=P, table=P, lens=P, leader=P, prefix=P, order=P, slots=1, width=2, pages=4, page=16, hq=2, h=1, d=64, st=None, win=0,
           sinks=0, scale=1.0):
    runtime.call("lc_shared_decode", dtype, q, P, P, o, NULL, table, lens, leader, prefix, order, slots, width, pages, page, hq, h, d,
                 strides(11) if st is None else st, win, sinks, scale, NULL)


INVALID = [
    lambda: shared(dtype=0), lambda: shared(q=NULL), lambda: shared(o=NULL), lambda: shared(table=NULL), lambda: shared(lens=NULL),
    lambda: shared(leader=NULL), lambda: shared(prefix=NULL), lambda: shared(order=NULL), lambda: shared(slots=-1), lambda: shared(page=0),
    lambda: shared(hq=3, h=2), lambda: shared(st=NULL), lambda: shared(win=-1), lambda: shared(sinks=-1), lambda: shared(scale=math.nan),
    lambda: rotate(dtype=3), lambda: rotate(d=0), lambda: rotate(rot=3), lambda: rotate(rot=66), lambda: rotate(rot=-2), lambda: rotate(turns=NULL),
    lambda: rotate(magnitude=0.0), lambda: rotate(magnitude=math.nan), lambda: rotate(magnitude=math.inf), lambda: rotate(batch=-1),
    lambda: rotate(tokens=-1), lambda: rotate(heads=-1), lambda: rotate(st=NULL), lambda: rotate(x=NULL), lambda: rotate(out=NULL),
    lambda: rotate(positions=NULL),
    lambda: append(dtype=7), lambda: append(rot=65), lambda: append(turns=NULL), lambda: append(slots=-1), lambda: append(most=-1),
    lambda: append(page=0), lambda: append(h=0), lambda: append(hq=-1), lambda: append(st=NULL), lambda: append(k=NULL), lambda: append(q=NULL),
    lambda: append(out=NULL), lambda: append(kp=NULL), lambda: append(vp=NULL), lambda: append(table=NULL), lambda: append(lens=NULL),
    lambda: append(add=NULL), lambda: append(width=-1), lambda: append(pages=-1),
    lambda: prefixes(table=NULL), lambda: prefixes(lens=NULL), lambda: prefixes(leader=NULL), lambda: prefixes(shared=NULL),
    lambda: prefixes(order=NULL), lambda: prefixes(page=0), lambda: prefixes(slots=-1), lambda: prefixes(width=-1),
    lambda: sample(dtype=5), lambda: sample(rows=-1), lambda: sample(vocab=0), lambda: sample(logits=NULL), lambda: sample(uniform=NULL),
    lambda: sample(token=NULL),
]


@pytest.mark.parametrize("case", range(len(INVALID)))
def test_invalid_arguments(case):
    with pytest.raises(runtime.LcError) as err:
        INVALID[case]()
    assert err.value.status == -1 and err.value.message


UNSUPPORTED = [
    lambda: rotate(d=1026, rot=2), lambda: rotate(heads=1 << 20), lambda: rotate(batch=1 << 31), lambda: rotate(tokens=1 << 30),
    lambda: append(slots=1 << 21), lambda: append(most=1 << 31), lambda: append(width=1 << 25), lambda: append(hq=1 << 20),
    lambda: append(page=1 << 21), lambda: prefixes(slots=8193), lambda: prefixes(width=1 << 30), lambda: sample(rows=1 << 25),
    lambda: sample(vocab=(1 << 24) + 1), lambda: shared(slots=8193), lambda: shared(d=257), lambda: shared(width=1 << 30),
    lambda: rotate(heads=1 << 62), lambda: append(hq=1 << 62), lambda: append(h=1 << 61),
]


@pytest.mark.parametrize("case", range(len(UNSUPPORTED)))
def test_unsupported_sizes(case):
    with pytest.raises(runtime.LcError) as err:
        UNSUPPORTED[case]()
    assert err.value.status == -5 and err.value.message


@pytest.mark.parametrize("call", [lambda: rotate(x=ctypes.c_void_p(4097)), lambda: rotate(dtype=0, out=ctypes.c_void_p(4098)),
                                  lambda: append(v=ctypes.c_void_p(4097)), lambda: append(dtype=0, kp=ctypes.c_void_p(4098)),
                                  lambda: sample(logits=ctypes.c_void_p(4098))])
def test_elements_off_their_alignment(call):
    with pytest.raises(runtime.LcError) as err:
        call()
    assert err.value.status == -2


def test_nothing_to_do_is_no_error():
    rotate(batch=0, x=NULL)
    rotate(heads=0, x=NULL)
    append(slots=0, k=NULL)
    append(most=0, k=NULL)
    prefixes(slots=0, lens=NULL)
    sample(rows=0, logits=NULL)
    shared(slots=0, q=NULL)


def test_rotary():
    """The frequencies' formulas, and what is no rotation."""
    i = torch.arange(0, 64, 2, dtype=torch.float64)
    f = 10000.0 ** (-i / 64)
    plain = S.Rotary(64, device="cpu")
    assert torch.allclose(plain.frequencies, f, rtol=1e-15) and plain.magnitude == 1
    assert torch.allclose(plain.turns.double() * 2.0 ** -64 * 2 * math.pi, f, rtol=1e-15)
    assert torch.allclose(S.Rotary(64, scaling="linear", factor=4, device="cpu").frequencies, f / 4, rtol=1e-15)
    base = S.Rotary(64, scaling="base", factor=4, device="cpu").frequencies
    assert torch.allclose(base, (10000.0 * 4 ** (64 / 62)) ** (-i / 64), rtol=1e-14)
    assert abs(float(base[-1] / f[-1]) - 0.25) < 1e-12 and base[0] == f[0]  # the slowest pair is interpolated, the fastest stays
    bands = S.Rotary(64, scaling="bands", factor=16, trained=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(bands.frequencies[turns >= 32], f[turns >= 32])
    assert torch.allclose(bands.frequencies[turns <= 1], f[turns <= 1] / 16, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    share = (turns[between] - 1) / 31
    assert torch.allclose(bands.frequencies[between], f[between] * (share + (1 - share) / 16), rtol=1e-14)
    assert abs(bands.magnitude - (1 + 0.1 * math.log(16))) < 1e-15
    assert S.Rotary(64, scaling="bands", factor=16, trained=4096, magnitude=1.0, device="cpu").magnitude == 1
    own = S.Rotary(4, frequencies=[7.0, -0.5], device="cpu")  # over a turn a position: the whole turns are left out
    assert abs(float(own.turns[0]) * 2.0 ** -64 - (7 / (2 * math.pi) - 1)) < 1e-15 and float(own.turns[1]) < 0
    for call in (lambda: S.Rotary(3), lambda: S.Rotary(-2), lambda: S.Rotary(4, scaling="other"), lambda: S.Rotary(4, factor=2.0),
                 lambda: S.Rotary(4, base=0.0), lambda: S.Rotary(4, scaling="bands", factor=2.0), lambda: S.Rotary(2, scaling="base", factor=2.0),
                 lambda: S.Rotary(4, scaling="linear", factor=0.0), lambda: S.Rotary(4, frequencies=[1.0]),
                 lambda: S.Rotary(4, frequencies=[1.0, math.inf]), lambda: S.Rotary(4, magnitude=0.0), lambda: S.Rotary(4, base=math.nan),
                 lambda: S.Rotary(4, frequencies=[1.0, 1.0], scaling="linear", factor=2.0)):
        with pytest.raises(ValueError):
            call()


def test_tensors_off_the_device_or_of_another_type():
    x, positions, rotary = torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, dtype=torch.int32), S.Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.rotate(x, positions, rotary)
    with pytest.raises(ValueError, match="float64 is not"):
        S.rotate(x.double(), positions, rotary)
    maps = S.CacheMaps(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    pages = torch.zeros(4, 3, 16, 64)
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.cache_append(None, x, x, pages, pages, maps, maps.lens, rotary)
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.cache_prefixes(maps, page_size=16)
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.sample(x[0, 0], torch.zeros(3))
    with pytest.raises(ValueError, match="int32 is not"):
        S.sample(positions, torch.zeros(1))
    q, ints = x[0].half(), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA devices only"):
        S.shared_decode(q, pages.half(), pages.half(), maps.table, maps.lens, S.CachePrefixes(ints, ints, ints))
    with pytest.raises(ValueError, match="expected 9 arguments, got 1"):
        _serving.sample(1)


def test_what_requires_a_gradient():
    x, positions, rotary = torch.zeros(1, 2, 3, 64, requires_grad=True), torch.zeros(1, 2, dtype=torch.int32), S.Rotary(64, device="cpu")
    for call, name in [(lambda: S.rotate(x, positions, rotary), "x"), (lambda: S.sample(x[0, 0], torch.zeros(3)), "logits")]:
        with pytest.raises(ValueError, match=name + ": requires a gradient"):
            call()
