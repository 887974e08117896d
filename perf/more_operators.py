"""Measured cases of the operators around the serving attention: positions, the cache's writes, shared prefixes and the
drawing of tokens.

Each case runs either in its plain form (``own`` false: elementary torch operations, 32 bits or 64) or through
``lazy_compiler_b200.serving`` (``own`` true).  Five kinds of case:

* ``rotate``    positions enter queries and keys as rotations of pairs of a head's elements;
* ``append``    new tokens' keys, rotated, and values go to their pages, the rotated queries come back;
* ``prefixes``  which slots of a cache begin with the same pages, and how far;
* ``shared``    one new token of every sequence over its pages, a shared prefix read once for all that share it;
* ``sample``    a token of each row of logits: temperature, top-k, top-p and min-p, from given random numbers.

A head's first ``rot`` elements are pairs, ``(i, i + rot / 2)`` or interleaved ``(2 i, 2 i + 1)``; pair ``i`` at
position ``p`` turns by the angle ``p f_i``, ``f_i = base ** (-2 i / rot)`` or scaled for contexts longer than trained:
``linear`` f / factor; ``base`` base * factor ** (rot / (rot - 2)); ``bands`` f (g + (1 - g) / factor) with the ramp
g = (turns over the trained context - 1) / 31 in 0..1, and the rotated pairs times 1 + 0.1 ln factor.

The weights of a row of logits are w_i = exp((x_i - max) / T).  Kept are the ``top_k`` largest, of these the shortest
run from the largest on that holds ``top_p`` of their sum, of these those with w_i >= min_p; equal logits are taken in
index order.  The token is the first index at which the running sum of what is kept passes u times its total.
``T = 0`` takes the largest; ``top_k = 0``, ``top_p = 1`` and ``min_p = 0`` leave all.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
DEVICE = "cuda"


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one token of each of 64 sequences, queries and keys together: the call is all there is
        {"name": "rotate_token", "kind": "rotate", "batch": 64, "tokens": 1, "heads": 40, "dim": 128, "rot": 128,
         "interleaved": False, "scaling": "none", "factor": 1.0, "start": 5000, "dtype": "bf16"},
        # chunks of four long documents, a context eight times as long as trained
        {"name": "rotate_prompt", "kind": "rotate", "batch": 4, "tokens": 8191, "heads": 40, "dim": 128, "rot": 128,
         "interleaved": False, "scaling": "bands", "factor": 8.0, "start": 1000000, "dtype": "bf16"},
        # every sequence of a batch gets one token
        {"name": "append_token", "kind": "append", "batch": 64, "add": 1, "max_len": 2000, "page": 16, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "dtype": "bf16"},
        # ragged prompts enter the cache, a quarter of each head rotated
        {"name": "append_prompt", "kind": "append", "batch": 16, "add": 4095, "max_len": 500, "page": 32, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 32, "interleaved": True, "scaling": "linear", "factor": 4.0, "dtype": "f16"},
        # two prompts with four samples each
        {"name": "prefixes_small", "kind": "prefixes", "prompts": 2, "samples": 4, "prefix": 300, "suffix": 64, "page": 16},
        # a large batch of samples of long prompts
        {"name": "prefixes_large", "kind": "prefixes", "prompts": 8, "samples": 32, "prefix": 32000, "suffix": 1000, "page": 16},
        # four samples of one short prompt, a small model: latency
        {"name": "shared_beams", "kind": "shared", "prompts": 1, "samples": 4, "prefix": 301, "suffix": 40, "page": 16,
         "q_heads": 8, "kv_heads": 2, "dim": 64, "window": 0, "sinks": 0, "dtype": "f16"},
        # eight samples of each of eight prompts
        {"name": "shared_samples", "kind": "shared", "prompts": 8, "samples": 8, "prefix": 8000, "suffix": 600, "page": 16,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "bf16"},
        # sixty-four questions to one long document
        {"name": "shared_document", "kind": "shared", "prompts": 1, "samples": 64, "prefix": 100003, "suffix": 300, "page": 64,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "f16"},
        # one chat's next token
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 32000, "mode": "mixed", "dtype": "f16"},
        # a serving batch whose requests ask for different things
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 50257, "mode": "mixed", "dtype": "bf16"},
        # a large batch, logits in 32 bits, nucleus sampling for all
        {"name": "sample_large", "kind": "sample", "rows": 256, "vocab": 151643, "mode": "nucleus", "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "prefixes", "shared", "shared", "sample", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 1000, 151643), "dtype": rng.choice(["f16", "bf16", "f32"]),
                "mode": rng.choice(["mixed", "mixed", "nucleus", "all", "greedy", "top_k"])}
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind == "prefixes":
        prompts = _log(rng, 2, 32)
        samples = _log(rng, 2, 256 // prompts)
        return {"kind": kind, "prompts": prompts, "samples": samples, "prefix": _log(rng, 8 * page, 4096 * page // max(4, samples)),
                "suffix": _log(rng, 1, 1000), "page": page}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([64, 64, 96, 128, 128])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "shared":
        prompts = _log(rng, 1, 16)
        samples = _log(rng, 1, 64 // min(4, prompts))
        suffix = _log(rng, 1, 1500)
        most = 64 * 100003 * 32 // (prompts * samples * q_heads)
        return {"kind": kind, "prompts": prompts, "samples": samples, "prefix": _log(rng, 1, max(1, min(65536 // prompts, most) - suffix)),
                "suffix": suffix, "page": page, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "window": rng.choice([0, 0, 0, _log(rng, 16, 8192)]), "sinks": rng.choice([0, 4, _log(rng, 1, 100)]), "dtype": dtype}
    scaling = rng.choice(["none", "none", "linear", "base", "bands"])
    case = {"kind": kind, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
            "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 10.0, 32.0]), "dtype": dtype}
    batch = _log(rng, 1, 128)
    if kind == "rotate":
        heads = rng.choice([1, 3, 8, 10, 32, 40])
        return dict(case, batch=batch, tokens=_log(rng, 1, max(1, 30000 // batch)), heads=heads,
                    start=_log(rng, 1, 4000000), dtype=rng.choice(["f16", "bf16", "f32"]))
    return dict(case, batch=batch, add=_log(rng, 1, max(1, 50000 // batch)), max_len=_log(rng, 1, 4096), page=page,
                q_heads=min(q_heads, 32), kv_heads=kv_heads if q_heads <= 32 else 4)


# ---------------------------------------------------------------- inputs

def _spread(n, lo, hi):
    """n whole numbers spread evenly over lo..hi, the largest among them."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _adds(case):
    """New tokens of each sequence."""
    return [1] * case["batch"] if case["add"] == 1 else _spread(case["batch"], max(1, case["add"] // 4), case["add"])


def _prefixes(case):
    """Tokens of each prompt."""
    return _spread(case["prompts"], max(1, case["prefix"] // 2), case["prefix"])


def _suffixes(case):
    """Tokens of each sample behind its prompt."""
    return _spread(case["prompts"] * case["samples"], 1, case["suffix"])


def _ceil(a, b):
    return -(-a // b)


def _int32(values):
    return torch.as_tensor(values, dtype=torch.int32).to(DEVICE)


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _base(case):
    return 500000.0 if case["scaling"] == "base" else 10000.0


TRAINED = 8192  # tokens of the context that the scaled cases stand for


def _positions_handle(case):
    """The frequencies that a program computes once."""
    if not own:
        return _frequencies(case)
    from lazy_compiler_b200 import serving as S

    return S.Rotary(case["rot"], _base(case), interleaved=case["interleaved"], scaling=case["scaling"], factor=case["factor"],
                    trained=TRAINED, device=DEVICE)


def _frequencies(case):
    rot, factor, i = case["rot"], case["factor"], torch.arange(case["rot"] // 2, dtype=torch.float64)
    base = _base(case) * (factor ** (rot / (rot - 2)) if case["scaling"] == "base" else 1.0)
    f, magnitude = base ** (-2 * i / rot), 1.0
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "bands":
        g = ((TRAINED * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, magnitude = f * (g + (1 - g) / factor), 1 + 0.1 * math.log(factor)
    return f.to(DEVICE), magnitude


def prepare(case, seed):
    gen = torch.Generator().manual_seed(int(seed))
    cuda = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, state = DTYPES[case.get("dtype", "f16")], {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=cuda, device=DEVICE, dtype=dtype)

    if case["kind"] == "sample":
        return dict(state, **_logits(case, gen, cuda))

    if case["kind"] == "rotate":
        # queries and keys as they lie in the projection's output, the values behind them
        b, t, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
        state["x"] = normal(b, t, h + _ceil(h, 4), d)[:, :, :h]
        start = torch.randint(0, case["start"], (b, 1), generator=gen, dtype=torch.int32)
        state["positions"] = (start + torch.arange(t, dtype=torch.int32)).to(DEVICE)
        state["rotary"] = _positions_handle(case)
        return state

    page = case["page"]
    if case["kind"] == "append":
        b, h, hq, d = case["batch"], case["kv_heads"], case["q_heads"], case["dim"]
        adds = _shuffled(_adds(case), gen)
        lens = _shuffled(_spread(b, 0, case["max_len"]), gen)
        lens = [n + a for n, a in zip(lens, adds)]  # as they are when room has been made
        held = [_ceil(n, page) for n in lens]
        pages = sum(lens) // page + b  # as many for every seed
        pages, width = pages + max(4, pages // 8), _ceil(case["max_len"] + case["add"], page)
        ids = torch.randperm(pages, generator=gen, dtype=torch.int64).to(torch.int32)
        table, at = torch.full((b, width), -1, dtype=torch.int32), 0
        for i, n in enumerate(held):
            table[i, :n] = ids[at:at + n]
            at += n
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[ids[:at].long()] = 1
        qkv = normal(b, max(adds), hq + 2 * h, d)  # one projection's output
        state.update(q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + h], v=qkv[:, :, hq + h:], pool=normal(2, pages, h, page, d),
                     table=table.to(DEVICE), lens=_int32(lens), refs=refs.to(DEVICE), add=_int32(adds))
        state["rotary"] = _positions_handle(case)
        return state

    # samples of prompts: each shares the full pages of its prompt and has pages of its own behind them
    n, prompts = case["prompts"] * case["samples"], _prefixes(case)
    if case["kind"] == "prefixes":
        prompts = [p - int(torch.randint(0, p // 2 + 1, (1,), generator=gen)) for p in prompts]
    which = _shuffled([i % case["prompts"] for i in range(n)], gen)
    lens = [prompts[w] + s for w, s in zip(which, _shuffled(_suffixes(case), gen))]
    full = [p // page for p in prompts]
    held = [_ceil(x, page) for x in lens]
    pages = sum(full) + sum(h - full[w] for h, w in zip(held, which))
    pages, width = pages + max(4, pages // 8), _ceil(case["prefix"] + case["suffix"], page)
    ids = torch.randperm(pages, generator=gen, dtype=torch.int64).to(torch.int32)
    shared, at = [], 0
    for f in full:
        shared.append(ids[at:at + f])
        at += f
    table = torch.full((n, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for i, w in enumerate(which):
        table[i, :full[w]] = shared[w]
        table[i, full[w]:held[i]] = ids[at:at + held[i] - full[w]]
        at += held[i] - full[w]
    refs.index_add_(0, table[table >= 0].long(), torch.ones(int((table >= 0).sum()), dtype=torch.int32))
    state.update(table=table.to(DEVICE), lens=_int32(lens), refs=refs.to(DEVICE))
    if case["kind"] == "shared":
        state["q"] = normal(n, case["q_heads"], case["dim"])
        state["pool"] = normal(2, pages, case["kv_heads"], page, case["dim"])
        # what the program keeps between two forks
        lowest = {}
        for i, w in enumerate(which):
            lowest.setdefault(w, i)
        alone = [full[w] == 0 or case["samples"] == 1 for w in which]
        leader = [i if alone[i] else lowest[w] for i, w in enumerate(which)]
        tokens = [0 if alone[i] else full[w] * page for i, w in enumerate(which)]
        state["prefixes"] = [_int32(leader), _int32(tokens), _int32(sorted(range(n), key=lambda i: (leader[i], i)))]
    return state


def _logits(case, gen, cuda):
    """Logits with a head of some likely tokens over a bulk of unlikely ones, rows of different sharpness, and what each
    request asks for."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=cuda, device=DEVICE) * 1.5 - 2
    likely = min(vocab, 200)
    first = torch.randint(0, vocab, (rows, 1), generator=gen).to(DEVICE)
    at = torch.randperm(vocab, generator=gen).to(DEVICE)[(first + torch.arange(likely, device=DEVICE)) % vocab]
    sharp = torch.rand(rows, 1, generator=cuda, device=DEVICE) * 2.5 + 1.0
    head = 14 - sharp * torch.log(torch.arange(1, likely + 1, device=DEVICE, dtype=torch.float32))
    x.scatter_(1, at, head + torch.randn(rows, likely, generator=cuda, device=DEVICE) * 0.5)

    def pick(values, ints=False):
        chosen = [values[i] for i in torch.randint(0, len(values), (rows,), generator=gen).tolist()]
        return torch.tensor(chosen, dtype=torch.int32 if ints else torch.float32, device=DEVICE)

    mode = case["mode"]
    asks = {"mixed": ([0.0, 0.6, 0.8, 1.0, 1.3], [0, 0, 20, 50, 1000], [1.0, 0.8, 0.9, 0.95], [0.0, 0.0, 0.02, 0.1]),
            "nucleus": ([0.7, 1.0], [0], [0.8, 0.9, 0.95, 0.99], [0.0]), "all": ([0.8, 1.0], [0], [1.0], [0.0]),
            "greedy": ([0.0], [0], [1.0], [0.0]), "top_k": ([0.7, 1.0], [1, 20, 50, 100], [1.0], [0.0])}[mode]
    return {"logits": x.to(DTYPES[case["dtype"]]), "uniform": torch.rand(rows, generator=cuda, device=DEVICE),
            "temperature": pick(asks[0]), "top_k": pick(asks[1], True), "top_p": pick(asks[2]), "min_p": pick(asks[3])}


# ---------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from lazy_compiler_b200 import serving as S

    case, kind = state["case"], state["case"]["kind"]
    if kind == "rotate":
        return S.rotate(state["x"], state["positions"], state["rotary"])
    if kind == "sample":
        return S.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                        top_p=state["top_p"], min_p=state["min_p"], return_logprob=True)
    maps = S.CacheMaps(state["table"], state["lens"], state["refs"])
    if kind == "prefixes":
        return list(S.cache_prefixes(maps, page_size=case["page"]))
    pool = state["pool"]
    if kind == "append":
        q = S.cache_append(state["q"], state["k"], state["v"], pool[0], pool[1], maps, state["add"], state["rotary"])
        return [q, pool]
    return S.shared_decode(state["q"], pool[0], pool[1], state["table"], state["lens"], S.CachePrefixes(*state["prefixes"]),
                           window=case["window"], sinks=case["sinks"], return_lse=True)


def _run_plain(state):
    case = state["case"]
    return {"rotate": _plain_rotate, "append": _plain_append, "prefixes": _plain_prefixes, "shared": _plain_shared,
            "sample": _plain_sample}[case["kind"]](state, case)


def _rotated(x, positions, rotary, interleaved):
    """x [..., heads, d] at positions [...], in 32 bits, the angles in 64."""
    f, magnitude = rotary
    rot = 2 * f.numel()
    angle = positions.double()[..., None, None] * f
    cos, sin = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    y = x.float()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _plain_rotate(state, case):
    return _rotated(state["x"], state["positions"], state["rotary"], case["interleaved"])


def _plain_append(state, case):
    pool, add, page, table = state["pool"], state["add"], case["page"], state["table"]
    t = torch.arange(state["k"].shape[1], device=add.device)
    pos = ((state["lens"] - add).view(-1, 1) + t).long()
    real = t < add.view(-1, 1)
    q, k = (_rotated(state[x], pos, state["rotary"], case["interleaved"]) for x in "qk")
    at = torch.gather(table, 1, (pos // page).clamp(max=table.shape[1] - 1)).long()
    where, off = at[real], (pos % page)[real]
    pool[0][where, :, off] = k[real]
    pool[1][where, :, off] = state["v"][real]
    return [torch.where(real[..., None, None], q, torch.zeros_like(q)), pool]


def _plain_prefixes(state, case):
    table, page = state["table"], case["page"]
    slots, width = table.shape
    slot, j = torch.arange(slots, device=table.device), torch.arange(width, device=table.device)
    full = state["lens"].clamp(max=width * page) // page
    real = (full > 0) & (table[:, 0] >= 0)
    same = (table[:, :1] == table[:, 0]) & real & real.view(-1, 1) | (slot == slot.view(-1, 1))
    leader = torch.where(same, slot, slots).amin(1)
    alike = (table == table[leader]) & (j < torch.minimum(full, full[leader]).view(-1, 1))
    common = torch.cumprod(alike.to(torch.int32), 1).sum(1).to(torch.int32)
    least = torch.full((slots,), width, dtype=torch.int32, device=table.device).scatter_reduce(0, leader, common, "amin")
    members = torch.zeros_like(least).scatter_add(0, leader, torch.ones_like(least))
    shared = torch.where(members[leader] > 1, least[leader] * page, torch.zeros_like(least))
    order = torch.argsort(leader, stable=True)
    return [leader.to(torch.int32), shared.to(torch.int32), order.to(torch.int32)]


def _plain_shared(state, case):
    q, pool, table = state["q"], state["pool"], state["table"].long()
    n, hq, d = q.shape
    h, page = pool.shape[2], pool.shape[3]
    keys = table.shape[1] * page
    window = case["window"] or keys + 1
    j = torch.arange(keys, device=q.device)
    out, lse = torch.empty_like(q), torch.empty((n, hq), device=q.device)
    for i in range(n):
        at = table[i].clamp(min=0)
        k = pool[0][at].float().permute(1, 3, 0, 2).reshape(h, d, keys)
        v = pool[1][at].float().permute(1, 0, 2, 3).reshape(h, keys, d)
        p = state["lens"][i] - 1
        sees = (j <= p) & ((j > p - window) | (j < case["sinks"]))
        s = torch.matmul(q[i].float().view(h, hq // h, d) / math.sqrt(d), k).masked_fill(~sees, -math.inf)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        e = torch.exp(s - m)
        z = e.sum(-1, keepdim=True)
        o = torch.matmul(e, v.masked_fill(~sees.view(keys, 1), 0)) / torch.where(z == 0, torch.ones_like(z), z)
        out[i] = o.view(hq, d).to(q.dtype)
        lse[i] = (m + torch.log(z)).view(hq)
    return out, lse


def _plain_sample(state, case):
    x, u = state["logits"].double(), state["uniform"].double().view(-1, 1)
    t, k, p, m = (state[name].view(-1, 1) for name in ("temperature", "top_k", "top_p", "min_p"))
    vocab = x.shape[1]
    down, index = torch.sort(x, dim=1, descending=True, stable=True)
    weights = torch.exp((down - down[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)).double())
    rank = torch.arange(vocab, device=x.device)
    k = torch.where(t > 0, torch.where(k > 0, k, vocab), 1)
    weights = torch.where(rank < k, weights, torch.zeros_like(weights))
    run = torch.cumsum(weights, 1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], 1)
    keep = (before < p.double() * run[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= weights >= m.double()
    weights = torch.where(keep, weights, torch.zeros_like(weights))
    weights = torch.zeros_like(weights).scatter_(1, index, weights)
    run = torch.cumsum(weights, 1)
    token = (run <= u * run[:, -1:]).sum(1, keepdim=True).clamp(max=vocab - 1)
    logprob = torch.log(torch.gather(weights, 1, token) / run[:, -1:])
    return token.view(-1).to(torch.int32), logprob.view(-1).float()


# ---------------------------------------------------------------- the work of one pass

def work(case):
    kind, size = case["kind"], 4 if case.get("dtype") == "f32" else 2
    if kind == "sample":
        return {"bytes": case["rows"] * (size * case["vocab"] + 4 * 7), "flops": 0}
    if kind == "rotate":
        rows = case["batch"] * case["tokens"]
        return {"bytes": rows * (2 * size * case["heads"] * case["dim"] + 4), "flops": 3 * rows * case["heads"] * case["rot"]}
    page = case["page"]
    if kind == "append":
        tokens, d = sum(_adds(case)), case["dim"]
        rows = case["batch"] * max(_adds(case))  # of the rotated queries: every one is written
        held = sum(_ceil(a, page) for a in _adds(case))
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": size * d * (tokens * (heads + 2 * case["kv_heads"]) + rows * case["q_heads"]) + 4 * held,
                "flops": 3 * tokens * (case["q_heads"] + case["kv_heads"]) * case["rot"]}
    prompts, n = _prefixes(case), case["prompts"] * case["samples"]
    full = [p // page for p in prompts]
    if kind == "prefixes":
        # three quarters of the longest prompts, as far as their samples agree
        return {"bytes": 4 * (sum(full) * 3 // 4 * case["samples"] + 4 * n), "flops": 0}
    window, sinks = case["window"], case["sinks"]
    mean = sum(prompts) / len(prompts)
    seen = sum(min(mean + s, window + sinks) if window else mean + s for s in _suffixes(case))
    if window:  # what a window leaves of the prefixes: between one sample's share and the whole
        once = sum(min(p, window + sinks) for p in prompts) + sum(min(s, window) for s in _suffixes(case))
    else:
        once = sum(prompts) + sum(_suffixes(case)) + sum((p % page) * (case["samples"] - 1) for p in prompts)
    q = n * case["q_heads"]
    return {"bytes": size * case["dim"] * (2 * case["kv_heads"] * once + 2 * q) + 4 * q + 4 * _ceil(int(seen), page),
            "flops": 4 * case["dim"] * case["q_heads"] * seen}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions in 64 bits, one sequence, token or row at a time."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    return {"rotate": _exact_rotate, "append": _exact_append, "prefixes": _exact_prefixes, "shared": _exact_shared,
            "sample": _exact_sample}[case["kind"]](case, state)


def _exact_turn(case, x, positions):
    """x [n, heads, d] at positions [n]: pairs as complex numbers."""
    x = x.double()
    rot, half = case["rot"], case["rot"] // 2
    first = [2 * i if case["interleaved"] else i for i in range(half)]
    second = [i + 1 if case["interleaved"] else i + half for i in first]
    f, magnitude = _frequencies(case)
    z = torch.complex(x[..., first], x[..., second])
    z = z * torch.polar(torch.full_like(f, magnitude).expand(len(positions), half), positions.double()[:, None] * f)[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_rotate(case, state):
    return torch.stack([_exact_turn(case, x.clone(), p) for x, p in zip(state["x"], state["positions"])])


def _exact_append(case, state):
    pool, page = state["pool"].double(), case["page"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    for i, (n, add) in enumerate(zip(state["lens"].tolist(), state["add"].tolist())):
        pos = torch.arange(n - add, n, device=DEVICE)
        out[i, :add] = _exact_turn(case, state["q"][i, :add].clone(), pos)
        k, v = _exact_turn(case, state["k"][i, :add].clone(), pos), state["v"][i, :add].double()
        for at in range((n - add) // page, _ceil(n, page)):
            lo, hi, to = max(n - add, at * page), min(n, (at + 1) * page), int(state["table"][i, at])
            for plane, new in enumerate((k, v)):
                pool[plane, to, :, lo - at * page:hi - at * page] = new[lo - n + add:hi - n + add].transpose(0, 1)
    return [out, pool]


def _exact_prefixes(case, state):
    table, lens, page = state["table"].tolist(), state["lens"].tolist(), case["page"]
    groups, leader, shared = {}, list(range(len(lens))), [0] * len(lens)
    for i, row in enumerate(table):
        if lens[i] >= page:
            groups.setdefault(row[0], []).append(i)
    for members in groups.values():
        if len(members) > 1:
            rows, n = [table[i] for i in members], 0
            while n < min(lens[i] // page for i in members) and all(row[n] == rows[0][n] for row in rows):
                n += 1
            for i in members:
                leader[i], shared[i] = members[0], n * page
    order = sorted(range(len(lens)), key=lambda i: (leader[i], i))
    return [torch.tensor(x, dtype=torch.int32) for x in (leader, shared, order)]


def _exact_shared(case, state):
    q, page, scale = state["q"], case["page"], 1.0 / math.sqrt(case["dim"])
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for i, n in enumerate(state["lens"].tolist()):
        ids = state["table"][i, :_ceil(n, page)].long()
        lo = max(0, n - case["window"]) if case["window"] else 0
        seen = torch.cat([torch.arange(min(lo, case["sinks"])), torch.arange(lo, n)]).to(q.device)
        for head in range(case["kv_heads"]):
            k, v = (state["pool"][x][ids, head].reshape(-1, case["dim"])[seen].double() for x in (0, 1))
            rows = slice(head * group, (head + 1) * group)
            s = q[i, rows].double() @ k.T * scale
            lse[i, rows] = torch.logsumexp(s, -1)
            out[i, rows] = torch.exp(s - lse[i, rows, None]) @ v
    return out, lse


def _exact_sample(case, state):
    tokens, logprobs = [], []
    asks = [state[x].tolist() for x in ("uniform", "temperature", "top_k", "top_p", "min_p")]
    for x, u, t, k, p, m in zip(state["logits"].double().cpu().numpy(), *asks):
        order = (-x).argsort(kind="stable")
        if t == 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        if k:
            order = order[:k]
        w = torch.from_numpy(x[order] - x[order[0]]).div(t).exp()
        run = w.cumsum(0)
        n = 1 + int((run[:-1] < p * run[-1]).sum()) if p < 1 else len(order)
        n = min(n, int((w >= m).sum()))
        kept, by_index = w[:n], torch.from_numpy(order[:n].copy()).argsort()
        run = kept[by_index].cumsum(0)
        at = min(int((run <= u * run[-1]).sum()), n - 1)
        tokens.append(int(order[int(by_index[at])]))
        logprobs.append(float(torch.log(kept[by_index[at]] / run[-1])))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)
