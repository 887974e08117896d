"""Prompt attention with a sliding window and sinks, and paged single-token attention, against 64-bit plain forms.

The tolerances are the ones derived in serving_ref.check_attention.
"""
import math

import numpy as np
import pytest

import serving_ref as R

pytestmark = pytest.mark.gpu

DTYPES = ["f16", "bf16"]


def torch_dtype(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def normal(shape, dtype, seed, spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(torch_dtype(dtype))


def f64(t):
    return t.double().cpu().numpy()


def ints(values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prompt(dtype, b, s_q, s_kv, hq, h, d, window, sinks, q_lens=None, kv_lens=None, scale=None, spread=1.0, seed=0, poison=False):
    """Runs one case and checks it; with `poison`, what no row of a sequence sees is NaN or infinite."""
    import torch
    from lazy_compiler_b200 import serving as S
    from lazy_compiler_b200 import runtime
    q, k, v = (normal(shape, dtype, seed + i, spread if i < 2 else 1.0)
               for i, shape in enumerate([(b, s_q, hq, d), (b, s_kv, h, d), (b, s_kv, h, d)]))
    nq, nkv = q_lens or [s_q] * b, kv_lens or [s_kv] * b
    ref = R.window_attention(f64(q), f64(k), f64(v), scale or 1 / math.sqrt(d), window, sinks, nq, nkv)
    if poison:
        for x in range(b):
            k[x, nkv[x]:] = float("nan")
            v[x, nkv[x]:] = float("inf")
            q[x, nq[x]:] = float("nan")
            gone = np.ones(nkv[x], bool)
            for i in range(nq[x]):
                gone[R.seen(nkv[x] - nq[x] + i, nkv[x], window, sinks)] = False
            gone = torch.from_numpy(gone).cuda()
            k[x, :nkv[x]][gone] = float("inf")
            v[x, :nkv[x]][gone] = float("nan")
    o, lse = S.window_attention(q, k, v, window=window, sinks=sinks, scale=scale, q_lens=ints(q_lens) if q_lens else None,
                                kv_lens=ints(kv_lens) if kv_lens else None, return_lse=True)
    runtime.call("lc_device_status", None)
    R.check_attention(f64(o), f64(lse), ref, dtype)
    return q, k, v, o, lse


# (batch, s_q, s_kv, q_heads, kv_heads, d, window, sinks)
PROMPTS = [
    (1, 1, 1, 1, 1, 64, 0, 0), (1, 1, 1, 1, 1, 128, 1, 0), (1, 1, 300, 8, 2, 128, 64, 4), (2, 19, 19, 8, 2, 64, 8, 2),
    (1, 128, 128, 1, 1, 128, 0, 0), (1, 129, 129, 2, 1, 128, 0, 0), (1, 257, 257, 4, 4, 64, 128, 0),
    (2, 200, 333, 4, 1, 128, 100, 7), (1, 300, 300, 3, 1, 128, 17, 40), (1, 150, 420, 5, 1, 64, 200, 130),
    (1, 90, 700, 7, 7, 128, 129, 1), (1, 64, 1000, 6, 2, 96, 300, 260), (1, 70, 70, 2, 2, 80, 16, 3), (1, 33, 65, 2, 1, 40, 0, 0),
    (1, 20, 50, 2, 1, 256, 24, 2), (1, 9, 30, 2, 2, 17, 6, 1), (1, 40, 40, 16, 1, 128, 12, 2), (1, 30, 90, 24, 1, 64, 0, 0),
    (1, 520, 520, 2, 2, 128, 1, 0), (1, 300, 900, 2, 1, 64, 2, 1), (1, 400, 400, 1, 1, 8, 64, 4),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", PROMPTS)
def test_prompt(case, dtype, cuda_device):
    prompt(dtype, *case, seed=sum(case))


# The same edges with enough rows that they are not taken one by one.
MANY_ROWS = [
    (1, 129, 129, 16, 4, 128, 9, 0), (2, 200, 333, 8, 2, 128, 100, 7), (1, 300, 300, 12, 4, 128, 17, 40), (1, 150, 420, 10, 2, 64, 20, 130),
    (1, 520, 520, 8, 8, 128, 1, 0), (1, 500, 900, 8, 1, 64, 2, 1), (1, 400, 400, 2, 1, 8, 64, 4), (1, 140, 140, 32, 2, 128, 12, 2),
    (1, 130, 165, 48, 1, 64, 30, 3), (1, 257, 700, 7, 7, 96, 65, 64), (1, 257, 700, 6, 2, 128, 63, 63), (1, 70, 400, 100, 1, 64, 24, 5),
    (1, 130, 700, 6, 2, 128, 300, 65), (1, 65, 1200, 20, 4, 64, 600, 300),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", MANY_ROWS)
def test_prompt_many_rows(case, dtype, cuda_device):
    prompt(dtype, *case, seed=sum(case))


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_few_rows_of_many_keys(dtype, cuda_device):
    """The keys of a few rows are cut over the SMs and joined."""
    prompt(dtype, 1, 3, 5000, 4, 1, 128, 0, 0, seed=20)
    prompt(dtype, 2, 5, 3000, 4, 2, 64, 2500, 9, q_lens=[5, 2], kv_lens=[2900, 1500], seed=21, poison=True)
    prompt(dtype, 1, 130, 2000, 3, 1, 96, 1100, 200, seed=22)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_joined_rows_keep_infinite_values_to_themselves(d, cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    q, k, v, clean, lse = prompt("f16", 1, 6, 4000, 4, 2, d, 0, 0, seed=23)
    v[0, 3997, 1, 3] = float("inf")  # seen by the last three queries
    o, lse2 = S.window_attention(q, k, v, return_lse=True)
    assert torch.equal(o[:, :, :2], clean[:, :, :2]) and torch.equal(lse, lse2)
    assert torch.isposinf(o[0, 3:, 2:, 3]).all()
    u = R.U["f16"]
    near = (o[0, :3, 2:].float() - clean[0, :3, 2:].float()).abs() <= 4 * u * (1 + clean[0, :3, 2:].float().abs())
    assert near.all() and torch.isfinite(o[0, 3:, 2:, 4:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 24])
def test_prompt_ragged_and_empty_rows(d, dtype, cuda_device):
    """Lengths of zero, more queries than keys (the first rows see nothing), padded rows."""
    prompt(dtype, 7, 200, 310, 4, 2, d, 50, 3, q_lens=[200, 0, 150, 1, 200, 37, 130], kv_lens=[310, 100, 0, 1, 90, 37, 129], seed=5)
    prompt(dtype, 3, 140, 60, 2, 2, d, 0, 0, seed=6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 17])
@pytest.mark.parametrize("window,sinks", [(40, 3), (0, 0)])
def test_prompt_does_not_see_what_is_masked(window, sinks, d, dtype, cuda_device):
    prompt(dtype, 3, 100, 400, 4, 2, d, window, sinks, q_lens=[100, 60, 3], kv_lens=[400, 250, 131], seed=7, poison=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_keeps_infinite_values_to_the_rows_that_see_them(d, dtype, cuda_device):
    """A key with an infinite value changes the rows that see it and no other."""
    import torch
    from lazy_compiler_b200 import serving as S
    q, k, v, clean, clean_lse = prompt(dtype, 1, 300, 300, 4, 2, d, 64, 2, seed=8)
    k[0, 100, 1] = float("nan")
    v[0, 40, 0] = float("inf")
    v[0, 150, 1, 5] = -float("inf")
    v[0, 290, 0, 3] = float("nan")
    o, lse = S.window_attention(q, k, v, window=64, sinks=2, return_lse=True)
    i = torch.arange(300, device="cuda")
    sees = lambda j: (i >= j) & (i < j + 64)  # noqa: E731
    hit = torch.zeros(300, 4, dtype=torch.bool, device="cuda")
    hit[:, :2] = (sees(40) | sees(290))[:, None]
    hit[:, 2:] = (sees(100) | sees(150))[:, None]
    # rows that see nothing special: as before, up to the rounding of another path's sums
    u = R.U[dtype]
    far = (o[0].float() - clean[0].float()).abs()[~hit]
    assert torch.isfinite(far).all() and (far <= 4 * u * (1 + clean[0].float().abs()[~hit])).all()
    assert torch.isnan(o[0, :, 2:][sees(100)]).all() and torch.isnan(lse[0, 2:][:, sees(100)]).all()
    only40 = sees(40) & ~sees(290)
    assert torch.isposinf(o[0, :, :2][only40]).all()
    only150 = sees(150) & ~sees(100)
    assert torch.isneginf(o[0, :, 2:, 5][only150]).all() and torch.isfinite(o[0, :, 2:, :5][only150]).all()
    assert torch.isnan(o[0, :, :2, 3][sees(290)]).all() and torch.isfinite(o[0, :, :2, 4][sees(290) & ~sees(40)]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_large_scores_and_scale(dtype, cuda_device):
    prompt(dtype, 1, 260, 260, 2, 1, 128, 90, 4, spread=3.0, seed=9)
    prompt(dtype, 1, 260, 260, 2, 1, 64, 0, 0, scale=0.7, seed=10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 96])
def test_prompt_layouts(d, dtype, cuda_device):
    """Heads outside tokens, slices of a fused projection, an output inside a larger one, odd offsets."""
    import torch
    from lazy_compiler_b200 import serving as S
    b, s, hq, h = 2, 170, 4, 2
    fused = normal((b, s, (hq + 2 * h) * d), dtype, 11)
    q, k, v = (x.view(b, s, -1, d) for x in fused.split([hq * d, h * d, h * d], -1))
    ref = R.window_attention(f64(q), f64(k), f64(v), 1 / math.sqrt(d), 60, 5, [s] * b, [s] * b)
    wide = torch.full((b, s, hq, d + 8), 7.0, dtype=q.dtype, device="cuda")
    o, lse = S.window_attention(q, k, v, window=60, sinks=5, out=wide[..., :d], return_lse=True)
    assert o.data_ptr() == wide.data_ptr() and (wide[..., d:] == 7).all()
    R.check_attention(f64(o), f64(lse), ref, dtype)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    o2, lse2 = S.window_attention(*turned, window=60, sinks=5, return_lse=True)
    R.check_attention(f64(o2), f64(lse2), ref, dtype)
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape) for x in (q, k, v)]
    for x, y in zip(odd, (q, k, v)):
        x.copy_(y)
    o3, lse3 = S.window_attention(*odd, window=60, sinks=5, return_lse=True)
    R.check_attention(f64(o3), f64(lse3), ref, dtype)


def test_prompt_one_key_head_for_a_batch_by_broadcasting(cuda_device):
    """Keys and values shared by the batch with a stride of zero."""
    from lazy_compiler_b200 import serving as S
    q, k, v = normal((3, 140, 4, 128), "f16", 1), normal((1, 140, 2, 128), "f16", 2), normal((1, 140, 2, 128), "f16", 3)
    k, v = k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)
    ref = R.window_attention(f64(q), f64(k), f64(v), 128 ** -0.5, 33, 2, [140] * 3, [140] * 3)
    o, lse = S.window_attention(q, k, v, window=33, sinks=2, return_lse=True)
    R.check_attention(f64(o), f64(lse), ref, "f16")


def test_prompt_without_keys_or_queries(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    q = normal((2, 5, 4, 128), "f16", 0)
    none = torch.empty((2, 0, 2, 128), dtype=torch.float16, device="cuda")
    o, lse = S.window_attention(q, none, none, return_lse=True)
    assert (o == 0).all() and torch.isneginf(lse).all()
    o = S.window_attention(q[:, :0], none, none)
    assert o.shape == (2, 0, 4, 128)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_repeats_and_long_rows(d, cuda_device):
    """Many items per CTA, several sequences; twice the same bits; a sample of rows against 64 bits."""
    import torch
    from lazy_compiler_b200 import serving as S
    from lazy_compiler_b200 import runtime
    b, s, hq, h, window, sinks = 2, 5000, 16, 4, 700, 9
    q, k, v = normal((b, s, hq, d), "bf16", 1), normal((b, s, h, d), "bf16", 2), normal((b, s, h, d), "bf16", 3)
    lens = ints([4999, 3111])
    o, lse = S.window_attention(q, k, v, window=window, sinks=sinks, q_lens=lens, kv_lens=lens, return_lse=True)
    o2, lse2 = S.window_attention(q, k, v, window=window, sinks=sinks, q_lens=lens, kv_lens=lens, return_lse=True)
    runtime.call("lc_device_status", None)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    rng = np.random.default_rng(0)
    got = ([], [], [], [], [])
    for x, n in enumerate((4999, 3111)):
        for i in sorted(set(rng.integers(0, n, 40)) | {0, 1, 699, 700, 708, 709, n - 1}):
            js = torch.from_numpy(R.seen(i, n, window, sinks)).cuda()
            for y in rng.integers(0, hq, 3):
                z = y // (hq // h)
                r = R.attend(f64(q[x, i, y]), f64(k[x, js, z]), f64(v[x, js, z]), d ** -0.5)
                for lst, item in zip(got, (*r, f64(o[x, i, y]), float(lse[x, y, i]))):
                    lst.append(item)
    ref_o, ref_lse, size, o_rows, lse_rows = (np.array(g) for g in got)
    R.check_attention(o_rows, lse_rows, (ref_o, ref_lse, size), "bf16")
    assert (o[1, 3111:] == 0).all() and torch.isneginf(lse[1, :, 3111:]).all()


# ---------------------------------------------------------------- one token

def cache(dtype, lens, page, h, d, spare, seed, order="hnd", spread=1.0):
    """(k_pages, v_pages, table): scattered pages; `order` nhd keeps a page's tokens outside its heads."""
    import torch
    rng = np.random.default_rng(seed)
    held = [-(-n // page) for n in lens]
    pages, width = sum(held) + spare, max(held + [1])
    ids = rng.permutation(pages)
    table, at = np.full((len(lens), width), -1), 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    shape = (2, pages, h, page, d) if order == "hnd" else (2, pages, page, h, d)
    pool = normal(shape, dtype, seed)
    pool[0] *= spread
    if order == "nhd":
        pool = pool.transpose(2, 3)
    return pool[0], pool[1], table


def decode(dtype, lens, page, hq, h, d, window, sinks, seed=0, order="hnd", poison=True, spread=1.0, scale=None, edit=None):
    import torch
    from lazy_compiler_b200 import serving as S
    from lazy_compiler_b200 import runtime
    k, v, table = cache(dtype, lens, page, h, d, 3, seed, order, spread)
    q = normal((len(lens), hq, d), dtype, seed + 1, spread)
    lens = list(lens)
    if edit:
        edit(table, lens)
    ref = R.paged_decode(f64(q), f64(k), f64(v), table, lens, scale or d ** -0.5, window, sinks)
    if poison:
        used = np.zeros((k.shape[0], page), bool)
        for i, n in enumerate(lens):
            n = min(max(n, 0), table.shape[1] * page)
            for j in R.seen(n - 1, n, window, sinks):
                if 0 <= table[i, j // page] < k.shape[0]:
                    used[table[i, j // page], j % page] = True
        gone = torch.from_numpy(~used).cuda()[:, None, :, None]
        k.masked_fill_(gone, float("nan"))
        v.masked_fill_(gone, float("inf"))
    o, lse = S.paged_decode(q, k, v, ints(table), ints(lens), window=window, sinks=sinks, scale=scale, return_lse=True)
    runtime.call("lc_device_status", None)
    R.check_attention(f64(o), f64(lse), ref, dtype)
    again, lse2 = S.paged_decode(q, k, v, ints(table), ints(lens), window=window, sinks=sinks, scale=scale, return_lse=True)
    assert torch.equal(o, again) and torch.equal(lse, lse2)


# (lens, page, q_heads, kv_heads, d, window, sinks)
TOKENS = [
    ([1], 16, 1, 1, 64, 0, 0), ([0, 1, 2], 16, 8, 2, 128, 0, 0), ([301], 16, 8, 2, 64, 64, 4), ([33, 0, 500, 17], 16, 32, 8, 128, 0, 0),
    ([1000], 64, 64, 8, 128, 0, 0), ([257, 256, 255], 32, 5, 1, 128, 100, 3), ([77, 400], 1, 4, 4, 64, 0, 0), ([90, 300], 5, 6, 2, 96, 50, 7),
    ([1200, 3, 64], 24, 7, 1, 128, 0, 0), ([640, 129], 128, 16, 1, 64, 33, 200), ([300], 16, 24, 1, 128, 0, 0), ([200, 90], 8, 40, 1, 64, 17, 1),
    ([150, 40], 16, 4, 2, 256, 0, 0), ([150, 40], 16, 4, 2, 192, 60, 2), ([55, 14], 16, 4, 2, 17, 20, 1), ([70], 16, 2, 2, 8, 0, 0), ([4097, 31], 16, 3, 3, 128, 1, 0),
    ([5000], 16, 8, 1, 128, 0, 0), ([2000] * 5 + [9], 32, 4, 4, 128, 1999, 1), ([48], 16, 1, 1, 128, 1, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", TOKENS)
def test_token(case, dtype, cuda_device):
    decode(dtype, *case, seed=sum(case[0]))


# The same edges with enough slots that they are not taken row by row.
MANY_TOKENS = [
    ([0, 1, 2, 15, 16, 17] * 20, 16, 8, 2, 128, 0, 0), ([1] * 200, 16, 4, 1, 64, 0, 0), ([301, 2, 40] * 12, 16, 8, 2, 64, 64, 4),
    ([90, 30] * 10, 5, 12, 4, 96, 50, 7), ([64, 129] * 8, 128, 16, 1, 64, 33, 200), ([40, 14] * 16, 16, 24, 1, 128, 20, 1),
    ([70] * 40, 16, 8, 8, 8, 0, 0), ([48, 97] * 30, 16, 4, 4, 128, 1, 1), ([25] * 12, 8, 32, 2, 192, 0, 0), ([20000], 32, 5, 1, 128, 0, 0),
    ([9000, 11], 64, 20, 1, 64, 8000, 30), ([6000], 16, 4, 2, 256, 0, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(MANY_TOKENS)))
def test_token_more(case, dtype, cuda_device):
    decode(dtype, *MANY_TOKENS[case], seed=case)


def test_token_joined_rows_keep_infinite_values_to_themselves(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    k, v, table = cache("f16", [9000], 16, 2, 128, 1, 24)
    q = normal((1, 4, 128), "f16", 25)
    clean = S.paged_decode(q, k, v, ints(table), ints([9000]))
    v[table[0, 300], 1, 2, 7] = float("inf")
    o = S.paged_decode(q, k, v, ints(table), ints([9000]))
    keep = torch.arange(128, device="cuda") != 7
    assert torch.equal(o[:, :2], clean[:, :2]) and torch.isposinf(o[:, 2:, 7]).all() and torch.equal(o[:, 2:][..., keep], clean[:, 2:][..., keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_many_slots(dtype, cuda_device):
    rng = np.random.default_rng(3)
    decode(dtype, rng.integers(0, 90, 300).tolist(), 16, 4, 2, 64, 0, 0, seed=4)
    decode(dtype, rng.integers(0, 300, 1100).tolist(), 16, 1, 1, 64, 40, 2, seed=5)


@pytest.mark.parametrize("slots, most, d", [(1, 130, 64), (2, 64, 128), (150, 130, 64), (151, 128, 128), (297, 65, 128), (40, 1000, 96)])
def test_token_many_short_caches(slots, most, d, cuda_device):
    """Runs that begin and end at, just behind and just before the ends of segments of a few tiles."""
    lens = [(i * 37) % (most + 1) for i in range(slots)]
    decode("bf16", lens, 16, 6, 3, d, 0, 0, seed=slots)
    decode("f16", [most] * slots, 16, 6, 3, d, 0, 0, seed=slots + 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_layouts_and_scores(dtype, cuda_device):
    decode(dtype, [100, 333], 16, 8, 2, 128, 0, 0, seed=6, order="nhd")
    decode(dtype, [100, 333], 7, 8, 2, 64, 70, 5, seed=7, order="nhd")
    decode(dtype, [700, 333], 16, 8, 2, 128, 0, 0, seed=8, spread=3.0)
    decode(dtype, [700, 333], 16, 8, 2, 128, 0, 0, seed=9, scale=0.7)


def test_token_absent_pages_and_lengths_out_of_range(cuda_device):
    """Entries of -1 or beyond the pool are not visible; lengths are cut at the table, or at zero."""
    def edit(table, lens):
        table[0, 2] = -1
        table[1, 0] = 10 ** 6
        table[2, :] = -1
        lens[1] = 10 ** 8
        lens[3] = -5
    decode("f16", [100, 90, 40, 20], 16, 8, 2, 128, 0, 0, seed=10, edit=edit)
    decode("f16", [100, 90, 40, 20], 16, 8, 2, 128, 30, 20, seed=10, edit=edit)


def test_token_odd_offsets_and_strides(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    lens = [90, 41]
    k, v, table = cache("bf16", lens, 16, 2, 64, 1, 12)
    q = normal((2, 8, 64), "bf16", 13)
    ref = R.paged_decode(f64(q), f64(k), f64(v), table, lens, 0.125, 0, 0)
    odd = []
    for x in (q, k, v):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        y.copy_(x)
        odd.append(y)
    out = torch.zeros((2, 8, 65), dtype=q.dtype, device="cuda")
    wide = torch.full((2, table.shape[1] + 3), 99, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = ints(table)
    o, lse = S.paged_decode(*odd, wide[:, :table.shape[1]], ints(lens), out=out[..., :64], return_lse=True)
    R.check_attention(f64(o), f64(lse), ref, "bf16")
    assert (out[..., 64] == 0).all()


def test_token_infinite_values_reach_their_heads_alone(cuda_device):
    import torch
    from lazy_compiler_b200 import serving as S
    k, v, table = cache("f16", [200], 16, 2, 128, 1, 14)
    q = normal((1, 8, 128), "f16", 15)
    clean = S.paged_decode(q, k, v, ints(table), ints([200]))
    v[table[0, 3], 1, 2, 7] = float("inf")
    o = S.paged_decode(q, k, v, ints(table), ints([200]))
    assert torch.equal(o[:, :4], clean[:, :4]) and torch.isposinf(o[:, 4:, 7]).all()
    keep = torch.arange(128, device="cuda") != 7
    assert torch.equal(o[:, 4:][..., keep], clean[:, 4:][..., keep])


def test_token_matches_the_prompt_form(cuda_device):
    """The last position of a prompt, once from contiguous keys and once from pages."""
    from lazy_compiler_b200 import serving as S
    n, page = 700, 16
    k, v, table = cache("bf16", [n], page, 2, 128, 2, 16)
    flat = [x[ints(table[0]).long()].permute(0, 2, 1, 3).reshape(1, -1, 2, 128)[:, :n] for x in (k, v)]
    q = normal((1, 8, 128), "bf16", 17)
    a = S.paged_decode(q, k, v, ints(table), ints([n]), window=300, sinks=4)
    b = S.window_attention(q[:, None], *flat, window=300, sinks=4)[:, 0]
    assert ((a.float() - b.float()).abs() <= 2 * R.U["bf16"] * (1 + b.float().abs())).all()


def test_streams_and_graph_capture(cuda_device):
    """On a side stream, and captured: the lengths and tables are read when the graph runs."""
    import torch
    from lazy_compiler_b200 import serving as S
    k, v, table = cache("f16", [900, 50], 16, 2, 128, 1, 18)
    q, table, lens = normal((2, 8, 128), "f16", 19), ints(table), ints([900, 50])
    want = S.paged_decode(q, k, v, table, lens)
    other = torch.full_like(want, float("nan"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.paged_decode(q, k, v, table, lens, out=other)
    side.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        S.paged_decode(q, k, v, table, lens, out=other)
    lens.copy_(ints([333, 0]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(other, S.paged_decode(q, k, v, table, ints([333, 0])))


def test_offsets_beyond_32_bits(cuda_device):
    """Sequences four billion elements into their buffers: pages at the end of a long pool, a batch far apart."""
    import torch
    from lazy_compiler_b200 import serving as S
    pages, page, h, d = 270000, 16, 8, 128  # 4.4e9 elements a plane
    k = torch.zeros((pages, h, page, d), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    table = np.array([[pages - 1, pages - 40, pages - 7], [3, pages - 2, 0]])
    for x, seed in ((k, 26), (v, 27)):
        x[torch.from_numpy(table.ravel()).cuda()] = normal((6, h, page, d), "f16", seed)
    q, lens = normal((2, 8, d), "f16", 28), [45, 33]
    small = [x[torch.from_numpy(table.ravel()).cuda()] for x in (k, v)]
    ref = R.paged_decode(f64(q), f64(small[0]), f64(small[1]), np.arange(6).reshape(2, 3), lens, d ** -0.5, 0, 0)
    for repeat in (1, 40):  # row by row, and by tiles
        o, lse = S.paged_decode(q.repeat(repeat, 1, 1), k, v, ints(table).repeat(repeat, 1), ints(lens).repeat(repeat), return_lse=True)
        for r in (0, repeat - 1):
            R.check_attention(f64(o[2 * r:2 * r + 2]), f64(lse[2 * r:2 * r + 2]), ref, "f16")
    far = (1 << 32) + 64
    flat = k.view(-1)
    qs, ks, vs, outs = (flat[i * 10 ** 7:].as_strided((2, 200, n, d), (far, n * d, d, 1)) for i, n in enumerate((4, 2, 2, 4)))
    for i, x in enumerate((qs, ks, vs)):
        x.copy_(normal(x.shape, "f16", 30 + i))
    ref = R.window_attention(f64(qs), f64(ks), f64(vs), d ** -0.5, 150, 3, [200] * 2, [200] * 2)
    o, lse = S.window_attention(qs, ks, vs, window=150, sinks=3, out=outs, return_lse=True)
    R.check_attention(f64(o), f64(lse), ref, "f16")
    o, lse = S.window_attention(qs[:, :, :, :125], ks[:, :, :, :125], vs[:, :, :, :125], window=150, sinks=3, scale=d ** -0.5, return_lse=True)
    ref = R.window_attention(f64(qs[..., :125]), f64(ks[..., :125]), f64(vs[..., :125]), d ** -0.5, 150, 3, [200] * 2, [200] * 2)
    R.check_attention(f64(o), f64(lse), ref, "f16")


def test_refusals_of_tensors(cuda_device):
    """What does not fit is refused before anything is launched."""
    import torch
    from lazy_compiler_b200 import runtime
    from lazy_compiler_b200 import serving as S
    q, k = normal((2, 5, 4, 64), "f16", 0), normal((2, 7, 2, 64), "f16", 1)
    pages, table, lens = normal((6, 2, 16, 64), "f16", 2), ints([[0, 1], [2, 3]]), ints([20, 9])
    qt = q[:, 0]
    refused = [
        (lambda: S.window_attention(q, k, k[:, :6]), ValueError, "v: shape"),
        (lambda: S.window_attention(q, k, k.bfloat16()), ValueError, "v: bfloat16"),
        (lambda: S.window_attention(q.float(), k, k), ValueError, "q: float32"),
        (lambda: S.window_attention(q, k.cpu(), k), ValueError, "k: float16 on cpu"),
        (lambda: S.window_attention(q[0], k, k), ValueError, "3 axes"),
        (lambda: S.window_attention(q.transpose(2, 3), k.transpose(2, 3), k.transpose(2, 3)), ValueError, "k: shape"),
        (lambda: S.window_attention(k.mT, k.mT, k.mT), ValueError, "q: the last axis must be contiguous"),
        (lambda: S.window_attention(q, k, k, q_lens=lens.long()), ValueError, "q_lens: int64"),
        (lambda: S.window_attention(q, k, k, kv_lens=lens[:1]), ValueError, "kv_lens: shape"),
        (lambda: S.window_attention(q, k, k, out=q[:, :4]), ValueError, "out: shape"),
        (lambda: S.window_attention(q, k, k, out=q[:1].expand(2, -1, -1, -1)), ValueError, "out: axis 0 is expanded"),
        (lambda: S.paged_decode(qt, pages, pages, table, lens, out=qt[:, :1].expand(-1, 4, -1)), ValueError, "out: axis 1"),
        (lambda: S.window_attention(q, k, k, window=1.5), TypeError, "integer"),
        (lambda: S.window_attention(q, k, k, window=-1), runtime.LcError, "negative"),
        (lambda: S.window_attention(q[:, :, :3], k, k), runtime.LcError, "3 query heads over 2"),
        (lambda: S.window_attention(q, k, k, scale=0.0), runtime.LcError, "scale"),
        (lambda: S.window_attention(None, k, k), ValueError, "q: expected a tensor"),
        (lambda: S.paged_decode(qt, pages, pages[:5], table, lens), ValueError, "v_pages: shape"),
        (lambda: S.paged_decode(qt, pages, pages, table[:1], lens), ValueError, "table: shape"),
        (lambda: S.paged_decode(qt, pages, pages, table.long(), lens), ValueError, "table: int64"),
        (lambda: S.paged_decode(qt, pages, pages, table, lens[::2]), ValueError, "lens: shape"),
        (lambda: S.paged_decode(qt[:1], pages, pages, table, lens), ValueError, "table: shape"),
        (lambda: S.paged_decode(normal((2, 4, 264), "f16", 3), *[normal((6, 2, 16, 264), "f16", 4)] * 2, table, lens), runtime.LcError, "over 256"),
    ]
    for call, kind, text in refused:
        with pytest.raises(kind, match=text):
            call()
    o, lse = S.window_attention(q, k, k, return_lse=1)
    assert o.shape == q.shape and lse.shape == (2, 4, 5)


# ---------------------------------------------------------------- a sink that outweighs a long tail

def sink_rows(dtype, shape, axis, d, gap, seed):
    """Keys and values: key 0 along `axis` scores `gap` over all others for a query of ones, and its value is zero."""
    import torch
    k = torch.zeros(shape, dtype=torch_dtype(dtype), device="cuda")
    k.select(axis, 0).fill_(gap / d ** 0.5)
    v = normal(shape, dtype, seed).abs() + 0.5
    v.select(axis, 0).zero_()
    return k, v


def check_tail(o, lse, ref, dtype, keys, weight):
    """As check_attention, and what a weight may be off by beside its relative error: `weight` of the row's largest
    one for each key (f16 only; the values are below 8)."""
    extra = keys * weight * 8 if dtype == "f16" else 0.0
    far = np.abs(o - ref[0]) - extra
    R.check_attention(np.where(far <= 0, ref[0], ref[0] + np.sign(o - ref[0]) * far), lse, ref, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [8.0, 12.0, 18.0])
@pytest.mark.parametrize("lens,heads", [([700] * 64, 8), ([6000] + [100] * 29, 8), ([100003], 2)])
def test_token_tail_under_a_sink(lens, heads, gap, dtype, cuda_device):
    """Whole segments, segments joined by a CTA, and by the second kernel.  Two 16-bit parts end at 2^-25, the largest
    weight is 2^14: 2^-39 of it a key."""
    import torch
    from lazy_compiler_b200 import serving as S
    d, page = 64, 16
    width = -(-max(lens) // page)
    k, v = sink_rows(dtype, (heads, width * page, d), 1, d, gap, 40)
    k_pages, v_pages = (x.view(heads, width, page, d).transpose(0, 1).contiguous() for x in (k, v))
    q = torch.ones((len(lens), 2 * heads, d), dtype=k.dtype, device="cuda")
    table = torch.arange(width, dtype=torch.int32, device="cuda").repeat(len(lens), 1)
    o, lse = S.paged_decode(q, k_pages, v_pages, table, ints(lens), return_lse=True)
    for x in {0, len(lens) - 1}:
        n = lens[x]
        ref = [np.array(a) for a in zip(*(R.attend(f64(q[x, y]), f64(k[y // 2, :n]), f64(v[y // 2, :n]), d ** -0.5) for y in range(2 * heads)))]
        check_tail(f64(o[x]), f64(lse[x]), ref, dtype, n, 2.0 ** -39)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [8.0, 12.0, 18.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s_q,s_kv,heads,window", [(3000, 3000, 16, 0), (3000, 3000, 16, 2000), (9, 40000, 2, 0), (260, 30000, 2, 0)])
def test_prompt_tail_under_a_sink(s_q, s_kv, heads, window, d, gap, dtype, cuda_device):
    """Whole items, and runs of them joined with and without the deep form.  One 16-bit part ends at 2^-25, the largest
    weight is 2^7 or more: 2^-32 of it a key."""
    import torch
    from lazy_compiler_b200 import serving as S
    k, v = sink_rows(dtype, (1, s_kv, heads, d), 1, d, gap, 41)
    q = torch.ones((1, s_q, 2 * heads, d), dtype=k.dtype, device="cuda")
    o, lse = S.window_attention(q, k, v, window=window, sinks=1, return_lse=True)
    for i in (s_q - 1, s_q // 2, 0):
        js = torch.from_numpy(R.seen(s_kv - s_q + i, s_kv, window, 1)).cuda()
        ys = (0, heads, 2 * heads - 1)
        ref = [np.array(a) for a in zip(*(R.attend(f64(q[0, i, y]), f64(k[0, js, y // 2]), f64(v[0, js, y // 2]), d ** -0.5) for y in ys))]
        check_tail(f64(o[0, i, list(ys)]), f64(lse[0, list(ys), i]), ref, dtype, len(js), 2.0 ** -32)


# ---------------------------------------------------------------- values near f32's largest number

@pytest.mark.parametrize("case", [(1, 3, 20, 4, 2, 64, 0, 0), (1, 200, 200, 8, 2, 128, 60, 2), (1, 150, 420, 10, 2, 64, 0, 0), (1, 9, 5000, 4, 2, 128, 0, 0),
                                  (1, 20, 50, 2, 1, 256, 24, 2), (1, 130, 2000, 3, 1, 96, 1100, 200)])
def test_prompt_values_whose_sums_leave_f32(case, cuda_device):
    """A mean of bf16 values is in their range, whatever their sum is; beside them, ordinary columns."""
    from lazy_compiler_b200 import serving as S
    b, s_q, s_kv, hq, h, d, window, sinks = case
    q, k, v = normal((b, s_q, hq, d), "bf16", 50), normal((b, s_kv, h, d), "bf16", 51), normal((b, s_kv, h, d), "bf16", 52)
    v[..., :d // 2] = v[..., :d // 2].sign() * 3e38
    v[..., 1] = 3.3e38
    ref = R.window_attention(f64(q), f64(k), f64(v), d ** -0.5, window, sinks, [s_q] * b, [s_kv] * b)
    o, lse = S.window_attention(q, k, v, window=window, sinks=sinks, return_lse=True)
    R.check_attention(f64(o), f64(lse), ref, "bf16")


@pytest.mark.parametrize("case", [([30, 7], 16, 4, 2, 64), ([700] * 64, 16, 8, 2, 128), ([9000], 16, 4, 2, 64), ([3000] + [40] * 59, 16, 32, 8, 128),
                                  ([150, 40], 16, 4, 2, 256), ([90], 16, 2, 2, 17)])
def test_token_values_whose_sums_leave_f32(case, cuda_device):
    from lazy_compiler_b200 import serving as S
    lens, page, hq, h, d = case
    k, v, table = cache("bf16", lens, page, h, d, 2, 53)
    q = normal((len(lens), hq, d), "bf16", 54)
    v[..., :d // 2] = v[..., :d // 2].sign() * 3e38
    v[..., 1] = 3.3e38
    ref = R.paged_decode(f64(q), f64(k), f64(v), table, lens, d ** -0.5, 0, 0)
    o, lse = S.paged_decode(q, k, v, ints(table), ints(lens), return_lse=True)
    R.check_attention(f64(o), f64(lse), ref, "bf16")


def test_large_values_take_no_other_path(cuda_device):
    """Rows of values near f32's largest number are those of the same values 2^60 smaller, bit by bit."""
    import torch
    from lazy_compiler_b200 import serving as S
    q, k = normal((2, 300, 8, 128), "bf16", 55), normal((2, 300, 2, 128), "bf16", 56)
    v = normal((2, 300, 2, 128), "bf16", 57).clamp(-3.9, 3.9)
    small = S.window_attention(q, k, v * 2.0 ** 66, window=90, sinks=3)
    assert torch.equal(S.window_attention(q, k, v * 2.0 ** 126, window=90, sinks=3), small * 2.0 ** 60)
    pages = [x[:, :288].reshape(2 * 18, 16, 2, 128).transpose(1, 2).contiguous() for x in (k, v)]
    table, lens = torch.arange(36, dtype=torch.int32, device="cuda").view(2, 18), ints([288, 203])
    small = S.paged_decode(q[:, 0], pages[0], pages[1] * 2.0 ** 66, table, lens)
    assert torch.equal(S.paged_decode(q[:, 0], pages[0], pages[1] * 2.0 ** 126, table, lens), small * 2.0 ** 60)
