"""Sampling against the definition in 64 bits: the tokens are equal, whole numbers that they are."""
import numpy as np
import pytest
import torch

import step_ref as R
from lazy_compiler_b200 import serving as S

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def check(logits, u, temperature, top_k, top_p, min_p, **call):
    """Rows of logits against the definition; each of the four a list or a number.

    The logarithm: f32's rounding of it and of the share's (2^-23 of its size), and the weights' 2^-42, summed up."""
    rows = logits.shape[0]
    f = lambda v, t: torch.tensor(v, dtype=t, device="cuda") if isinstance(v, list) else v  # noqa: E731
    args = dict(temperature=f(temperature, torch.float32), top_k=f(top_k, torch.int32), top_p=f(top_p, torch.float32), min_p=f(min_p, torch.float32))
    token, logprob = S.sample(logits, f(u, torch.float32), **args, return_logprob=True, **call)
    at = lambda v, i: float(np.float32(v[i] if isinstance(v, list) else v))  # noqa: E731
    x = logits.double().cpu().numpy()
    for i in range(rows):
        k = top_k[i] if isinstance(top_k, list) else top_k
        want, share = R.sample(x[i], at(u, i), at(temperature, i), k, at(top_p, i), at(min_p, i))
        assert int(token[i]) == want, (i, int(token[i]), want)
        got = float(logprob[i])
        assert got == share or abs(got - share) <= 2.0 ** -22 * max(1.0, abs(share)), (i, got, share)
    return token


def peaked(rows, vocab, seed, dtype="f32", bulk=1.5, base=-2.0, likely=100):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * bulk + base
    n = min(vocab, likely)
    for i in range(rows):
        at = torch.randperm(vocab, generator=g)[:n]
        x[i, at] = 14 - (1 + 2.5 * torch.rand((), generator=g)) * torch.log(torch.arange(1, n + 1).float())
    return x.to(TYPES[dtype]).cuda()


def uniforms(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)).tolist()


ASKS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 0.99, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.05),
        (0.9, 1000, 0.8, 0.01), (1.0, 1, 1.0, 0.0), (0.0, 50, 0.9, 0.1), (0.2, 0, 0.5, 0.0)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 2047, 2049, 4097, 32000, 50257, 151643])
def test_asks(dtype, vocab):
    rows = 2 * len(ASKS)
    t, k, p, m = (list(x) for x in zip(*(ASKS * 2)))
    check(peaked(rows, vocab, vocab, dtype), uniforms(rows, vocab), t, k, p, m)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3000, 65537])
def test_flat_rows(dtype, vocab):
    """No likely head: what is kept fills no list."""
    t, k, p, m = (list(x) for x in zip(*ASKS, (1.0, vocab // 2, 1.0, 0.0), (1.0, vocab - 1, 0.9, 0.0), (2.0, 5000, 0.7, 1e-4)))
    check(peaked(len(t), vocab, 1, dtype, bulk=1.0, likely=0), uniforms(len(t), 2), t, k, p, m)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(20, 2100), (20, 32000), (3, 151643), (300, 20011)])
def test_many_likeliest(dtype, rows, vocab):
    """Top-k around what a list holds, alone and with what comes behind it; rows of one CTA to eight."""
    k = [255, 256, 257, 511, 512, 513, 1023, 1025, 1500, 1999, 2040, 2047, 2048, 2049, 2090, 5000, vocab - 1]
    t, p, m = [1.0, 1.3, 0.7, 5.0], [0.9, 1.0, 0.99, 0.5, 0.999], [0.0, 0.0, 1e-3]
    ask = [[v[i % len(v)] for i in range(rows)] for v in (t, k, p, m)]
    if rows == 3:
        ask[1] = [1500, 2040, 700]
    check(peaked(rows, vocab, 23, dtype), uniforms(rows, 24), *ask)


@pytest.mark.parametrize("vocab", [5, 2048, 2500, 40000])
def test_equal_logits(vocab):
    """Ties go by index: all equal, two values, and a tie where the list or the cut ends."""
    x = torch.zeros(7, vocab, device="cuda")
    x[1] = -3.5
    x[2, ::2] = 1.0
    x[3, vocab // 2:] = 2.0
    x[4, :3] = 5.0
    x[5] = torch.arange(vocab, device="cuda").float() % 3
    x[6, 1::2] = -0.0
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.61, 0.0), (1.0, vocab // 2 + 1, 1.0, 0.0), (0.5, vocab // 3 + 1, 0.77, 0.0),
                       (1.0, 0, 1.0, 1.0), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0)]:
        for seed in (3, 4):
            check(x, uniforms(7, seed), t, k, p, m)


@pytest.mark.parametrize("vocab", [9, 2049, 30001])
def test_masked_and_infinite(vocab):
    """Rows of which a mask leaves some, one or nothing; the type's lowest value as a mask; NaN; infinities."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(9, vocab, generator=g).cuda()
    allowed = torch.randperm(vocab, generator=g)[:5].cuda()
    inf = float("inf")
    x[0, :] = -inf
    x[1, :] = float("nan")
    x[2, torch.arange(vocab, device="cuda") != allowed[0]] = -inf
    keep = x[3, allowed].clone()
    x[3, :] = -inf
    x[3, allowed] = keep
    x[4, :] = torch.finfo(torch.float32).min
    x[5, :] = torch.finfo(torch.float32).min
    x[5, allowed] = keep
    x[6, allowed] = float("nan")
    x[7, allowed[:2]] = inf
    x[8, 0], x[8, 1] = inf, -inf
    for t, k, p, m in ASKS + [(1.0, 3, 1.0, 0.0), (1.0, 4, 0.5, 0.0), (1e-6, 0, 1.0, 0.0), (1.0, 8, 1.0, 0.0)]:
        token = check(x, uniforms(9, 6), t, k, p, m)
        assert token[:3].tolist() == [-1, -1, int(allowed[0])]


def test_borders():
    """u at its ends and outside, p and min_p of 0 and below, over 1, NaN; temperatures at f32's ends."""
    x = peaked(1, 5000, 7).expand(12, -1)
    last = 1 - 2.0 ** -24
    u = [0.0, last, 1.0, 2.0, -1.0, float("nan"), 0.3, 0.3, 0.3, 0.3, 0.3, 0.3]
    check(x, u, 1.0, 0, 1.0, 0.0)
    check(x, u, 1.0, 100, 1.0, 0.0)
    check(x, u, 1.0, 0, 0.9, 0.0)
    nan, inf = float("nan"), float("inf")
    one = x[:1].expand(9, -1)
    some = uniforms(9, 8)
    check(one, some, 1.0, 0, [0.0, -1.0, 1e-30, 1.0, 2.0, nan, 0.999999, 1e-7, 0.5], 0.0)
    check(one, some, 1.0, 0, 1.0, [0.0, -1.0, 1.0, 2.0, nan, 1e-30, 0.5, 0.999999, 1e-3])
    check(one, some, [1e-45, 1e-38, 1e-3, inf, 3e38, nan, -1.0, 100.0, 5e-2], 0, 1.0, 0.0)
    check(one, some, [1e-45, 1e-38, 1e-3, inf, 3e38, nan, -1.0, 100.0, 5e-2], 60, 0.9, 1e-3)
    check(one, some, 1.0, [-5, 0, 1, 2, 4999, 5000, 2 ** 31 - 1, 2048, 2047], 1.0, 0.0)


def test_large_values():
    """Logits of 1e30, of 1e4 with a small spread, and of f16's size."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(4, 3001, generator=g)
    x[0] *= 1e30
    x[1] = x[1] + 1e4
    x[2] = x[2] * 1e-20
    x[3] = -x[3].abs() * 1e4
    for t, k, p, m in ASKS:
        check(x.cuda(), uniforms(4, 10), t, k, p, m)
    check((x[1:2] * 6).half().cuda().expand(3, -1), uniforms(3, 11), 1.0, 0, 0.9, 0.0)


@pytest.mark.parametrize("dtype,shift,stride", [("f32", 1, 5003), ("f32", 3, 5000), ("bf16", 1, 5001), ("f16", 5, 5007), ("bf16", 0, 8192)])
def test_rows_off_their_alignment(dtype, shift, stride):
    """Rows that begin anywhere, with infinities beside them."""
    rows, vocab = 10, 4999
    t, k, p, m = (list(x) for x in zip(*ASKS))
    flat = torch.full((rows * stride + 64,), float("inf"), dtype=TYPES[dtype], device="cuda")
    view = flat[shift:].as_strided((rows, vocab), (stride, 1))
    view.copy_(peaked(rows, vocab, 12, dtype))
    check(view, uniforms(rows, 13), t, k, p, m)


def test_a_vocabulary_of_a_million():
    t, k, p, m = (list(x) for x in zip(*ASKS))
    check(peaked(len(t), 1000003, 18, "bf16"), uniforms(len(t), 19), t, k, p, m)


def test_refusals():
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    for name, wrong in (("temperature", u[:2]), ("temperature", u.double()), ("top_k", u), ("top_p", u.half()), ("min_p", u.cpu()),
                        ("top_p", torch.zeros(6, device="cuda")[::2]), ("out", torch.zeros(3, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError, match=name):
            S.sample(x, u, **{name: wrong})
    for call in (lambda: S.sample(x, u[:2]), lambda: S.sample(x[0], u), lambda: S.sample(x.T, u[:1].expand(10)), lambda: S.sample(x.double(), u)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        S.sample(x, u, top_k=1.5)


def test_streams_at_once():
    x, u = peaked(40, 30011, 20, "bf16"), torch.tensor(uniforms(40, 21), device="cuda")
    want = S.sample(x, u, top_p=0.95)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = [S.sample(x, u, top_p=0.95, stream=s.cuda_stream) for s in streams * 5]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_a_row_depends_on_itself_alone():
    """The same rows alone, in a batch of others and in another order: other splits of the rows over CTAs."""
    rows, vocab = 300, 20011
    x = peaked(20, vocab, 14, "bf16").repeat(15, 1)
    u = torch.tensor(uniforms(20, 15) * 15, device="cuda")
    ask = dict(temperature=0.9, top_p=0.97, return_logprob=True)
    token, logprob = S.sample(x, u, **ask)
    for i in (0, 7, 19):
        one, one_logprob = S.sample(x[i:i + 1], u[i:i + 1], **ask)
        assert bool((token[i::20] == one).all()) and bool((logprob[i::20] == one_logprob).all())
    assert rows == len(token)


def test_shares():
    """Frequencies over a grid of u are the weights' shares, to the grid's step."""
    x, n = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]], device="cuda"), 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    token = S.sample(x.expand(n, -1), u)
    share = torch.softmax(x[0].double(), 0)
    assert bool((torch.bincount(token, minlength=5).double() / n - share).abs().max() <= 1.0 / n)


def test_given_outputs_streams_and_graphs():
    x, u = peaked(6, 3333, 16, "f16"), torch.tensor(uniforms(6, 17), device="cuda")
    want = check(x, u.tolist(), 1.0, 0, 0.9, 0.0)
    out, side, graph = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    assert S.sample(x, u, top_p=0.9, out=out) is out and torch.equal(out, want)
    torch.cuda.synchronize()
    other = S.sample(x, u, top_p=0.9, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(other, want)
    with torch.cuda.graph(graph, stream=side):
        S.sample(x, u, top_p=0.9, out=out)
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.flip(0))
    assert S.sample(x[:0], u[:0]).shape == (0,)
