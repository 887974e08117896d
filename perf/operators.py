"""The serving operators' measured cases: prompt attention with a sliding window and always-visible first
tokens, attention of one new token over a paged key-value cache, and the cache's page operations.

Each case runs either in its plain form (``own`` false: elementary torch operations in 32 bits) or through
``lazy_compiler_b200.serving`` (``own`` true).  Five kinds of case:

* ``window``  attention of a prompt (or a chunk of one) over its keys;
* ``decode``  one new token of every sequence over its pages;
* ``append``  pages for new tokens are taken and their keys and values written;
* ``fork``    sequences continue others (samples of one prompt, beams), sharing their full pages;
* ``compact`` pages in use move to the lowest numbers, the tables follow.

Query ``i`` of a sequence with ``n_q`` queries and ``n_kv`` keys has position ``p = n_kv - n_q + i`` and sees
key ``j`` when ``j <= p`` and (``window == 0`` or ``j > p - window`` or ``j < sinks``).  A row that sees
nothing has output 0 and log-sum-exp -inf.  A cache pool is ``[planes, pages, kv_heads, page_size, head_dim]``
(a plane is the keys or the values of one layer); a sequence's table row lists its pages in order.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one short request of a small model: launch latency is all there is
        {"name": "window_short", "kind": "window", "batch": 1, "s_q": 19, "s_kv": 19, "ragged": False,
         "q_heads": 8, "kv_heads": 2, "dim": 64, "window": 8, "sinks": 2, "dtype": "f16"},
        # ragged prompts, the next chunk of each over what came before
        {"name": "window_chunk", "kind": "window", "batch": 4, "s_q": 777, "s_kv": 4001, "ragged": True,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4, "dtype": "bf16"},
        # one long document, read in one go
        {"name": "window_long", "kind": "window", "batch": 1, "s_q": 32768, "s_kv": 32768, "ragged": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 4096, "sinks": 16, "dtype": "f16"},
        # one chat, a short cache, a window with sinks
        {"name": "decode_one", "kind": "decode", "batch": 1, "max_len": 301, "min_len": 301, "page": 16,
         "q_heads": 8, "kv_heads": 2, "dim": 64, "window": 64, "sinks": 4, "dtype": "f16"},
        # a full serving batch of very different lengths
        {"name": "decode_batch", "kind": "decode", "batch": 64, "max_len": 8192, "min_len": 1, "page": 16,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # two very long contexts: few rows, the cache's length has to be split
        {"name": "decode_long", "kind": "decode", "batch": 2, "max_len": 131072, "min_len": 100003, "page": 64,
         "q_heads": 64, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "f16"},
        # every sequence of a batch gets one token
        {"name": "append_token", "kind": "append", "batch": 64, "add": 1, "max_len": 2000, "min_len": 0, "page": 16,
         "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # ragged prompts enter the cache
        {"name": "append_prompt", "kind": "append", "batch": 16, "add": 8191, "max_len": 500, "min_len": 0, "page": 32,
         "kv_heads": 8, "dim": 128, "dtype": "f16"},
        # four beams reorder
        {"name": "fork_beams", "kind": "fork", "batch": 4, "parents": 2, "layers": 4, "max_len": 777, "min_len": 777,
         "page": 16, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # eight samples of each prompt, all layers' pages
        {"name": "fork_samples", "kind": "fork", "batch": 256, "parents": 32, "layers": 16, "max_len": 2047,
         "min_len": 16, "page": 16, "kv_heads": 4, "dim": 128, "dtype": "f16"},
        # a small cache after a few requests have left
        {"name": "compact_small", "kind": "compact", "batch": 8, "layers": 2, "max_len": 300, "min_len": 1, "page": 16,
         "kv_heads": 2, "dim": 64, "used": 0.5, "dtype": "f16"},
        # a large cache, two thirds in use and scattered
        {"name": "compact_large", "kind": "compact", "batch": 96, "layers": 4, "max_len": 2048, "min_len": 1, "page": 16,
         "kv_heads": 8, "dim": 128, "used": 0.66, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["window", "decode", "append", "fork", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([64, 64, 96, 128, 128])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    case = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    if kind == "window":
        batch = _log(rng, 1, 8)
        s_q = _log(rng, 1, 16384 // batch)
        s_kv = s_q if rng.random() < 0.5 else s_q + _log(rng, 1, 16384 // batch)
        window = rng.choice([0, _log(rng, 4, 4000), _log(rng, 64, 4000)])
        if window == 0 and s_kv > 4096:
            window = 4000
        return dict(case, batch=batch, s_q=s_q, s_kv=s_kv, ragged=rng.random() < 0.5, q_heads=kv_heads * group,
                    window=window, sinks=rng.choice([0, 1, 4, _log(rng, 1, 130)]))
    if kind == "decode":
        batch = _log(rng, 1, 128)
        max_len = _log(rng, 1, 262144 // batch)
        return dict(case, batch=batch, max_len=max_len, min_len=rng.choice([0, 1, max_len]), page=page,
                    q_heads=kv_heads * group, window=rng.choice([0, 0, _log(rng, 16, 8192)]),
                    sinks=rng.choice([0, 4, _log(rng, 1, 100)]))
    if kind == "append":
        batch = _log(rng, 1, 128)
        return dict(case, batch=batch, add=_log(rng, 1, 65536 // batch), max_len=_log(rng, 1, 4096), min_len=0, page=page)
    batch = _log(rng, 2, 128)
    case = dict(case, batch=batch, layers=_log(rng, 1, 8), max_len=_log(rng, 1, 32768 // batch), min_len=1, page=page)
    if kind == "fork":
        return dict(case, parents=rng.randint(1, batch))
    return dict(case, used=round(rng.uniform(0.3, 0.9), 2))


# ---------------------------------------------------------------- inputs

def _spread(n, lo, hi):
    """n whole numbers spread evenly over lo..hi, the largest among them."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _lens(case):
    """Cached tokens of each sequence, a fork's parents (their order comes from the seed)."""
    return _spread(case.get("parents", case["batch"]), min(case["min_len"], case["max_len"]), case["max_len"])


def _adds(case):
    """New tokens of each sequence."""
    return [1] * case["batch"] if case["add"] == 1 else _spread(case["batch"], max(1, case["add"] // 4), case["add"])


def _window_lens(case):
    """(queries, keys) of each sequence of a window case."""
    if not case["ragged"]:
        return [(case["s_q"], case["s_kv"])] * case["batch"]
    q = _spread(case["batch"], max(1, case["s_q"] // 3), case["s_q"])
    return [(n, case["s_kv"] - (case["s_q"] - n) - (n % 5 if case["s_kv"] > 2 * case["s_q"] else 0)) for n in q]


def _ceil(a, b):
    return -(-a // b)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _tables(lens, page, pages, width, gen):
    """Tables over randomly scattered pages, and how often each page is used (once, or never)."""
    ids = torch.randperm(pages, generator=gen).tolist()
    table, at = [], 0
    for n in lens:
        held = _ceil(n, page)
        table.append(ids[at:at + held] + [-1] * (width - held))
        at += held
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[torch.tensor(ids[:at], dtype=torch.int64)] = 1
    return _int32(table).reshape(len(lens), width), refs.to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator().manual_seed(int(seed))
    cuda = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    h, d, batch = case["kv_heads"], case["dim"], case["batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=cuda, device=DEVICE, dtype=dtype)

    state = {"case": case}
    if case["kind"] == "window":
        state["q"] = normal(batch, case["s_q"], case["q_heads"], d)
        state["k"] = normal(batch, case["s_kv"], h, d)
        state["v"] = normal(batch, case["s_kv"], h, d)
        state["q_lens"] = state["kv_lens"] = None
        if case["ragged"]:
            lens = _shuffled(_window_lens(case), gen)
            state["q_lens"], state["kv_lens"] = _int32([n for n, _ in lens]), _int32([n for _, n in lens])
        return state

    page = case["page"]
    lens = _shuffled(_lens(case), gen)
    adds = _shuffled(_adds(case), gen) if case["kind"] == "append" else [0] * batch
    if case["kind"] == "fork":  # only the parents' slots hold something before
        lens = lens + [0] * (batch - case["parents"])
    width = max(1, _ceil(max(lens) + max(adds), page))
    held = sum(_ceil(n, page) for n in lens)
    pages = held + sum(_ceil(a, page) for a in adds) + max(4, held // 8)
    if case["kind"] == "fork":
        pages = held + batch + 4
    if case["kind"] == "compact":
        pages = max(held + 1, int(held / case["used"]))
    table, refs = _tables(lens, page, pages, width, gen)
    planes = 2 * case.get("layers", 1)
    state.update(pool=normal(planes, pages, h, page, d), table=table, lens=_int32(lens), refs=refs)
    if case["kind"] == "decode":
        state["q"] = normal(batch, case["q_heads"], d)
    if case["kind"] == "append":
        state["add"] = _int32(adds)
        state["k"] = normal(batch, max(adds), h, d)
        state["v"] = normal(batch, max(adds), h, d)
    if case["kind"] == "fork":
        # every parent goes on in its own slot; the other slots take the parents in turn, in the seed's order
        n = case["parents"]
        state["parent"] = _int32(list(range(n)) + _shuffled([i % n for i in range(batch - n)], gen))
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from lazy_compiler_b200 import serving as S

    case, kind = state["case"], state["case"]["kind"]
    if kind == "window":
        return S.window_attention(state["q"], state["k"], state["v"], window=case["window"], sinks=case["sinks"],
                                  q_lens=state["q_lens"], kv_lens=state["kv_lens"], return_lse=True)
    pool = state["pool"]
    if kind == "decode":
        return S.paged_decode(state["q"], pool[0], pool[1], state["table"], state["lens"], window=case["window"],
                              sinks=case["sinks"], return_lse=True)
    maps = S.CacheMaps(state["table"], state["lens"], state["refs"])
    if kind == "append":
        new = S.cache_extend(maps, state["add"], page_size=case["page"])
        S.cache_write(state["k"], state["v"], pool[0], pool[1], new, state["add"])
    elif kind == "fork":
        new = S.cache_fork(pool, maps, state["parent"])
    else:
        new = S.cache_compact(pool, maps)
    return [new.table, new.lens, new.refs, new.status, pool]


def _run_plain(state):
    case = state["case"]
    return {"window": _plain_window, "decode": _plain_decode, "append": _plain_append, "fork": _plain_fork,
            "compact": _plain_compact}[case["kind"]](state, case)


def _softmax_parts(s):
    """exp(s - max), its sum and the log-sum-exp over the last axis; rows of -inf alone give sum 0."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    return e, z, (m + torch.log(z)).squeeze(-1)


def _plain_window(state, case):
    """Blocks of queries against the span of keys that any of them sees, and the sinks before it."""
    q, k, v = state["q"], state["k"], state["v"]
    b, s_q, hq, d = q.shape
    s_kv, h = k.shape[1], k.shape[2]
    window, sinks = case["window"] or s_kv + s_q, min(case["sinks"], s_kv)
    dev = q.device
    n_q = state["q_lens"].long() if state["q_lens"] is not None else torch.full((b,), s_q, device=dev)
    n_kv = state["kv_lens"].long() if state["kv_lens"] is not None else torch.full((b,), s_kv, device=dev)
    t = min(s_q, 512)
    blocks = _ceil(s_q, t)
    span = min(s_kv, window + t)
    row = torch.arange(blocks * t, device=dev).view(blocks, t)
    pos = (n_kv - n_q).view(b, 1, 1) + row  # [b, blocks, t]
    first = (pos[:, :, 0] - window + 1).clamp(min=0).minimum(torch.full((), s_kv - span, device=dev))
    key = torch.cat([first.view(b, blocks, 1) + torch.arange(span, device=dev),
                     torch.arange(sinks, device=dev).expand(b, blocks, sinks)], -1)  # [b, blocks, span + sinks]
    fresh = torch.ones_like(key, dtype=torch.bool)
    fresh[:, :, span:] = key[:, :, span:] < first.view(b, blocks, 1)  # a sink inside the span counts once
    p, j = pos.view(b, blocks, t, 1), key.view(b, blocks, 1, -1)
    sees = (j <= p) & ((j > p - window) | (j < sinks)) & (j < n_kv.view(b, 1, 1, 1)) & fresh.view(b, blocks, 1, -1)
    sees &= (row < n_q.view(b, 1, 1)).view(b, blocks, t, 1)
    which = torch.arange(b, device=dev).view(b, 1, 1)
    kk = k[which, key].float().permute(0, 1, 3, 4, 2)  # [b, blocks, h, d, keys]
    vv = v[which, key].float().permute(0, 1, 3, 2, 4)
    qq = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, blocks * t - s_q)).float() / math.sqrt(d)
    qq = qq.view(b, blocks, t, h, hq // h, d).permute(0, 1, 3, 4, 2, 5).reshape(b, blocks, h, -1, d)
    s = torch.matmul(qq, kk).view(b, blocks, h, hq // h, t, -1)
    s = s.masked_fill_(~sees.view(b, blocks, 1, 1, t, -1), -math.inf)
    e, z, lse = _softmax_parts(s)
    o = torch.matmul(e.view(b, blocks, h, (hq // h) * t, -1), vv).view(b, blocks, h, hq // h, t, d)
    o = o / torch.where(z == 0, torch.ones_like(z), z)
    o = o.permute(0, 1, 4, 2, 3, 5).reshape(b, blocks * t, hq, d)[:, :s_q]
    lse = lse.permute(0, 2, 3, 1, 4).reshape(b, hq, blocks * t)[:, :, :s_q]
    return o.to(q.dtype), lse.contiguous()


def _plain_decode(state, case):
    q, pool, table, n = state["q"], state["pool"], state["table"].long(), state["lens"].long()
    b, hq, d = q.shape
    h, page = pool.shape[2], pool.shape[3]
    keys = table.shape[1] * page
    window = case["window"] or keys + 1
    at = table.clamp(min=0)
    k = pool[0][at].float().permute(0, 2, 4, 1, 3).reshape(b, h, d, keys)
    v = pool[1][at].float().permute(0, 2, 1, 3, 4).reshape(b, h, keys, d)
    j, p = torch.arange(keys, device=q.device), (n - 1).view(b, 1)
    sees = (j <= p) & ((j > p - window) | (j < case["sinks"]))
    s = torch.matmul(q.float().view(b, h, hq // h, d) / math.sqrt(d), k)
    s = s.masked_fill(~sees.view(b, 1, 1, keys), -math.inf)
    e, z, lse = _softmax_parts(s)
    v = v.masked_fill(~sees.view(b, 1, keys, 1), 0)
    o = torch.matmul(e, v) / torch.where(z == 0, torch.ones_like(z), z)
    return o.view(b, hq, d).to(q.dtype), lse.view(b, hq)


def _plain_extend(table, lens, refs, add, page):
    """The tables, lengths and use counts with pages for `add` more tokens, the lowest free pages in slot order."""
    width = table.shape[1]
    held, want = (lens + page - 1) // page, (lens + add + page - 1) // page
    before = torch.cumsum(want - held, 0) - (want - held)
    total, free = (want - held).sum(), (refs == 0).sum()
    fits = (total <= free) & (want <= width).all()
    ids = torch.argsort((refs != 0).to(torch.int32), stable=True)  # the free ones first, ascending
    j = torch.arange(width, device=table.device)
    fresh = (j >= held.view(-1, 1)) & (j < want.view(-1, 1)) & fits
    pick = (before.view(-1, 1) + j - held.view(-1, 1)).clamp(0, refs.numel() - 1)
    table = torch.where(fresh, ids[pick].to(torch.int32), table)
    lens = torch.where(fits, lens + add, lens)
    refs = refs.clone()
    refs[ids] += ((torch.arange(refs.numel(), device=refs.device) < total) & fits).to(torch.int32)
    code = torch.where((want <= width).all(), (total - free).clamp(min=0), torch.full_like(total, -1))
    status = torch.stack([code, (refs == 0).sum()]).to(torch.int32)
    return table, lens, refs, status


def _plain_append(state, case):
    pool, add, page = state["pool"], state["add"], case["page"]
    table, lens, refs, status = _plain_extend(state["table"], state["lens"], state["refs"], add, page)
    t = torch.arange(state["k"].shape[1], device=add.device)
    pos = ((lens - add).view(-1, 1) + t).long()
    real = t < add.view(-1, 1)
    at = torch.gather(table, 1, (pos // page).clamp(max=table.shape[1] - 1)).long()
    where, off = at[real], (pos % page)[real]
    pool[0][where, :, off] = state["k"][real]
    pool[1][where, :, off] = state["v"][real]
    return [table, lens, refs, status, pool]


def _plain_fork(state, case):
    pool, page, parent = state["pool"], case["page"], state["parent"].long()
    table, lens, refs = state["table"], state["lens"], state["refs"]
    slots, width = table.shape
    dev = table.device
    alive = parent >= 0
    src = parent.clamp(min=0)
    new_lens = torch.where(alive, lens[src], torch.zeros_like(lens))
    new = torch.where(alive.view(-1, 1), table[src], torch.full_like(table, -1))
    partial = new_lens % page
    last = (new_lens // page).clamp(max=width - 1).long()
    slot = torch.arange(slots, device=dev)
    lowest = torch.full((slots,), slots, device=dev).scatter_reduce(0, src, torch.where(alive, slot, slots), "amin")
    copies = alive & (partial > 0) & (lowest[src] != slot)  # these take a page of their own
    old = torch.gather(new, 1, last.view(-1, 1)).view(-1).clamp(min=0).long()
    j = torch.arange(width, device=dev)
    shared = (new >= 0) & ~(copies.view(-1, 1) & (j == last.view(-1, 1)))
    counts = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=dev)
    counts.scatter_add_(0, torch.where(shared, new.long(), refs.numel()).view(-1), torch.ones_like(new).view(-1))
    counts = counts[:-1]
    ids = torch.argsort((counts != 0).to(torch.int32), stable=True)
    order = torch.cumsum(copies.long(), 0) - 1
    total, free = copies.sum(), (counts == 0).sum()
    fits = total <= free
    fresh = ids[order.clamp(min=0)]
    takes = copies & fits
    new = torch.where(takes.view(-1, 1) & (j == last.view(-1, 1)), fresh.view(-1, 1).to(torch.int32), new)
    counts = counts + torch.zeros_like(counts).scatter_add_(0, fresh, takes.to(torch.int32))
    new, new_lens, counts = (torch.where(fits, x, y) for x, y in ((new, table), (new_lens, lens), (counts, refs)))
    status = torch.stack([(total - free).clamp(min=0), (counts == 0).sum()]).to(torch.int32)
    to, fro, n = fresh[takes], old[takes], partial[takes]
    held = torch.arange(page, device=dev) < n.view(-1, 1)  # only the tokens held are copied
    pool[:, to] = torch.where(held.view(1, -1, 1, page, 1), pool[:, fro], pool[:, to])
    return [new, new_lens, counts, status, pool]


def _plain_compact(state, case):
    pool, table, lens, refs = state["pool"], state["table"], state["lens"], state["refs"]
    pages = refs.numel()
    live = refs > 0
    used = live.sum()
    i = torch.arange(pages, device=refs.device)
    hole, mover = ~live & (i < used), live & (i >= used)
    holes, movers = i[hole], i[mover]  # as many of one as of the other, both ascending
    to = i.clone()
    to[movers] = holes
    new = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    counts = torch.where(i < used, refs, torch.zeros_like(refs))
    counts[holes] = refs[movers]
    status = torch.stack([torch.zeros_like(used), pages - used]).to(torch.int32)
    pool[:, holes] = pool[:, movers]
    return [new, lens, counts, status, pool]


# ---------------------------------------------------------------- the work of one pass

def work(case):
    h, d, size = case["kv_heads"], case["dim"], 2
    if case["kind"] == "window":
        pairs = queries = keys = 0
        for n_q, n_kv in _window_lens(case):
            pos = torch.arange(n_kv - n_q, n_kv)
            seen = torch.clamp(pos + 1, min=0)
            if case["window"]:
                sinks = torch.clamp(pos - case["window"] + 1, min=0, max=case["sinks"])
                seen = torch.clamp(seen, max=case["window"]) + sinks
            pairs += int(seen.sum())
            queries += n_q
            keys += (min(n_kv, n_q + case["window"] + case["sinks"]) if case["window"] else n_kv)
        rows = case["batch"] * case["s_q"]  # every row is written, also the empty ones
        return {"bytes": size * d * (case["q_heads"] * (queries + rows) + 2 * h * keys) + 4 * case["q_heads"] * rows,
                "flops": 4 * d * case["q_heads"] * pairs}
    lens, page = _lens(case), case["page"]
    if case["kind"] == "decode":
        seen = sum((min(n, case["window"] + case["sinks"]) if case["window"] else n) for n in lens)
        q = case["batch"] * case["q_heads"]
        return {"bytes": size * d * (2 * h * seen + 2 * q) + 4 * q + 4 * _ceil(seen, page), "flops": 4 * d * case["q_heads"] * seen}
    if case["kind"] == "append":
        tokens = sum(_adds(case))
        held = sum(_ceil(n + case["add"], page) for n in lens)
        return {"bytes": 2 * size * 2 * h * d * tokens + 4 * 3 * held, "flops": 0}
    token = size * 2 * case["layers"] * h * d  # of all planes
    if case["kind"] == "fork":
        mean = sum(n % page for n in lens) / len(lens)
        held = sum(_ceil(n, page) for n in lens) / len(lens)
        return {"bytes": 2 * token * mean * (case["batch"] - case["parents"]) + 4 * 3 * held * case["batch"], "flops": 0}
    held = sum(_ceil(n, page) for n in lens)
    pages = max(held + 1, int(held / case["used"]))
    moved = held * (pages - held) / pages  # pages in use above the number in use, scattered evenly
    return {"bytes": 2 * token * page * moved + 4 * (2 * pages + 2 * held), "flops": 0}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definition in 64 bits, sequence by sequence."""
    if case["kind"] not in ("window", "decode"):
        return _exact_pages(case, prepare(case, seed))
    state = prepare(case, seed)
    q, scale = state["q"], 1.0 / math.sqrt(case["dim"])
    group, limit = case["q_heads"] // case["kv_heads"], 1 << 26
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if case["kind"] == "decode":
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        for i, n in enumerate(state["lens"].tolist()):
            if n == 0:
                continue
            ids = state["table"][i, :_ceil(n, case["page"])].long()
            lo = max(0, n - case["window"]) if case["window"] else 0
            seen = torch.cat([torch.arange(min(lo, case["sinks"])), torch.arange(lo, n)]).to(q.device)
            for head in range(case["kv_heads"]):
                k, v = (state["pool"][x][ids, head].reshape(-1, case["dim"])[seen].double() for x in (0, 1))
                rows = slice(head * group, (head + 1) * group)
                s = q[i, rows].double() @ k.T * scale
                lse[i, rows] = torch.logsumexp(s, -1)
                out[i, rows] = torch.exp(s - lse[i, rows, None]) @ v
        return out, lse
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, dtype=torch.float64, device=q.device)
    n_q = state["q_lens"].tolist() if case["ragged"] else [case["s_q"]] * case["batch"]
    n_kv = state["kv_lens"].tolist() if case["ragged"] else [case["s_kv"]] * case["batch"]
    for i in range(case["batch"]):
        for head in range(case["kv_heads"]):
            k, v = (state[x][i, :n_kv[i], head].double() for x in "kv")
            rows = slice(head * group, (head + 1) * group)
            step = max(1, limit // (group * max(1, n_kv[i])))
            for a in range(0, n_q[i], step):
                e = min(n_q[i], a + step)
                pos = torch.arange(a, e, device=q.device) + n_kv[i] - n_q[i]
                keep = torch.arange(n_kv[i], device=q.device)[None, :] <= pos[:, None]
                if case["window"]:
                    past = torch.arange(n_kv[i], device=q.device)[None, :] <= pos[:, None] - case["window"]
                    past[:, :case["sinks"]] = False
                    keep &= ~past
                s = torch.einsum("qgd,kd->gqk", q[i, a:e, rows].double(), k) * scale
                s.masked_fill_(~keep, -math.inf)
                part = torch.logsumexp(s, -1)
                lse[i, rows, a:e] = part
                w = torch.exp(s - part[..., None]).masked_fill_(~keep, 0.0)
                out[i, a:e, rows] = torch.einsum("gqk,kd->qgd", w, v)
    return out, lse


def _exact_pages(case, state):
    """The page operations one page at a time, on lists."""
    page, pool = case["page"], state["pool"].double()
    table, lens, refs = state["table"].tolist(), state["lens"].tolist(), state["refs"].tolist()
    if case["kind"] == "append":
        free = iter([i for i, n in enumerate(refs) if n == 0])
        for i, add in enumerate(state["add"].tolist()):
            start, lens[i] = lens[i], lens[i] + add
            for at in range(_ceil(start, page), _ceil(lens[i], page)):
                table[i][at] = next(free)
                refs[table[i][at]] = 1
            for at in range(start // page, _ceil(lens[i], page)):
                lo, hi = max(start, at * page), min(lens[i], (at + 1) * page)
                for plane, new in enumerate((state["k"], state["v"])):
                    pool[plane, table[i][at], :, lo - at * page:hi - at * page] = new[i, lo - start:hi - start].transpose(0, 1).double()
    elif case["kind"] == "fork":
        old, old_lens, kept, moves = [list(row) for row in table], list(lens), set(), []
        refs = [0] * len(refs)
        for i, p in enumerate(state["parent"].tolist()):
            lens[i], table[i] = old_lens[p], list(old[p])
            whole = lens[i] // page
            for at in table[i][:whole]:
                refs[at] += 1
            if lens[i] % page:
                if p in kept:
                    moves.append((i, whole))
                else:
                    refs[table[i][whole]] += 1
                kept.add(p)
        free = iter([i for i, n in enumerate(refs) if n == 0])
        for i, at in moves:
            to, fro, n = next(free), table[i][at], lens[i] % page
            pool[:, to, :, :n] = pool[:, fro, :, :n]
            table[i][at], refs[to] = to, 1
    else:
        used = sum(n > 0 for n in refs)
        holes = iter([i for i in range(used) if refs[i] == 0])
        to = {i: next(holes) for i in range(used, len(refs)) if refs[i] > 0}
        for fro, hole in to.items():
            pool[:, hole], refs[hole], refs[fro] = pool[:, fro], refs[fro], 0
        table = [[to.get(at, at) for at in row] for row in table]
    return [torch.tensor(x) for x in (table, lens, refs, [0, refs.count(0)])] + [pool]
