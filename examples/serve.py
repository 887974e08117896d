"""Answers a few prompts with a small random-weight transformer, on the library's serving operators.

    python examples/serve.py [--layers 2 --steps 64 --samples 3 --window 128 --sinks 4 --temperature 0.8 --top-p 0.95]

The prompts, of different lengths, turned to their positions, run through windowed prompt attention while their keys and
values enter a paged cache; every prompt is forked into samples that share its pages; each step of all samples is one
replayed CUDA graph (projections with ``lc_gemm``, norms with ``lc_rmsnorm_f32``, pages taken, keys turned and written
with their values, attention of the one new token with the samples' common prefixes, pages behind the window given back,
the next token drawn); at the end some requests leave and the cache is compacted.
The last step's logits are then compared with those of the whole sequences run as prompts again.
"""
from __future__ import annotations

import argparse
import ctypes
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from lazy_compiler_b200 import runtime  # noqa: E402
from lazy_compiler_b200 import serving as S  # noqa: E402


def P(t):
    return ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class Model:
    """Attention layers only: x += Wo attend(norm(x) Wq, norm(x) Wk, norm(x) Wv)."""

    def __init__(self, layers: int, width: int = 512, q_heads: int = 8, kv_heads: int = 2, dim: int = 64, vocab: int = 1024):
        g = torch.Generator(device="cuda").manual_seed(0)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda") / s[0] ** 0.5  # noqa: E731
        self.q_heads, self.kv_heads, self.dim, self.width, self.vocab = q_heads, kv_heads, dim, width, vocab
        self.embed = rand(vocab, width) * vocab ** 0.5
        self.qkv = [rand(width, (q_heads + 2 * kv_heads) * dim).half() for _ in range(layers)]
        self.out = [rand(q_heads * dim, width).half() for _ in range(layers)]
        self.head = rand(width, vocab).half()
        self.norm, self.count = torch.ones(width, device="cuda"), torch.tensor([float(width)], device="cuda")
        self.eps = torch.tensor([1e-6], device="cuda")

    def normed(self, x):
        """RMS norm of the rows, as the GEMMs take them."""
        y = torch.empty_like(x)
        runtime.call("lc_rmsnorm_f32", P(self.count), P(self.eps), P(x), P(self.norm), P(y), x.numel() // self.width, self.width, stream())
        return y.half()

    def product(self, a, w):
        """a[..., k] w[k, n] in f16 with f32 sums."""
        k, n = w.shape
        c = torch.empty((*a.shape[:-1], n), dtype=torch.float16, device="cuda")
        runtime.call("lc_gemm", runtime.LC_F16, runtime.LC_F16, 0, 0, P(a), P(w), P(c), a.numel() // k, n, k, stream())
        return c

    def run(self, tokens, attend):
        """Logits of every token; ``attend(layer, q, k, v)`` is the attention, [..., heads, dim] each."""
        x = self.embed[tokens]
        cuts = [self.q_heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim]
        for layer, (qkv, out) in enumerate(zip(self.qkv, self.out)):
            q, k, v = (t.unflatten(-1, (-1, self.dim)) for t in self.product(self.normed(x), qkv).split(cuts, -1))
            x = x + self.product(attend(layer, q, k, v).flatten(-2), out).float()
        return self.product(self.normed(x), self.head)


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, default in (("layers", 2), ("steps", 64), ("samples", 3), ("window", 128), ("sinks", 4)):
        ap.add_argument(f"--{name}", type=int, default=default)
    for name, default in (("temperature", 0.8), ("top-p", 0.95)):
        ap.add_argument(f"--{name}", type=float, default=default)
    a = ap.parse_args(argv)
    if a.layers < 1 or a.samples < 1 or a.steps < 1:
        ap.error("--layers, --samples and --steps are at least 1")
    model = Model(a.layers)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lengths, page = [37, 300, 5], 16
    slots, most = len(lengths) * a.samples, max(lengths)
    cache = S.PagedCache(a.layers, slots * ((most + a.steps) // page + 2), page, model.kv_heads, model.dim, slots,
                         (most + a.steps) // page + 2, dtype=torch.float16)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.zeros((slots, most + a.steps + 1), dtype=torch.long, device="cuda")
    tokens[:len(lengths), :most] = torch.randint(0, model.vocab, (len(lengths), most), generator=g, device="cuda")

    rotary = S.Rotary(model.dim)
    uniform = torch.rand((slots, most + a.steps + 1), generator=g, device="cuda")
    positions = torch.arange(most + a.steps + 1, dtype=torch.int32, device="cuda").expand(slots, -1)

    # the prompts, padded to one batch; slots without a prompt have length 0
    lens = ints(lengths + [0] * (slots - len(lengths)))
    cache.extend(lens)

    def turned(x):
        return S.rotate(x, positions[:, :x.shape[1]], rotary)

    def prompt_attention(layer, q, k, v):
        q, k = turned(q), turned(k)
        cache.write(layer, k, v, lens)
        return S.window_attention(q, k, v, window=a.window, sinks=a.sinks, q_lens=lens, kv_lens=lens)

    logits = model.run(tokens[:, :most], prompt_attention)
    # samples of each prompt: their full pages are shared
    cache.fork(ints([s % len(lengths) for s in range(slots)]))
    parent = torch.arange(slots, device="cuda") % len(lengths)
    tokens, at = tokens[parent], lens[parent].long()
    first = logits[parent].gather(1, (at - 1).view(-1, 1, 1).expand(-1, 1, model.vocab)).squeeze(1)
    # each sample begins with another of the likeliest tokens
    rank = torch.arange(slots, device="cuda") // len(lengths)
    now = first.topk(a.samples).indices.gather(1, rank.view(-1, 1)).squeeze(1)
    one = ints([1] * slots)
    step_logits = torch.empty((slots, model.vocab), dtype=torch.float16, device="cuda")
    prefixes = cache.prefixes()

    def token_attention(layer, q, k, v):
        q = cache.append(layer, q[:, None], k[:, None], v[:, None], one, rotary)[:, 0]
        return cache.shared_decode(layer, q, prefixes, window=a.window, sinks=a.sinks)

    def step():
        tokens.scatter_(1, at.view(-1, 1), now.view(-1, 1))
        cache.extend(one)
        if a.window:
            cache.prefixes(into=prefixes)  # trimming takes pages from them
        step_logits.copy_(model.run(now, token_attention))
        if a.window:
            cache.trim(a.window, a.sinks)
        u = uniform.gather(1, at.view(-1, 1)).view(-1)
        now.copy_(S.sample(step_logits, u, temperature=a.temperature, top_p=a.top_p))
        at.add_(1)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # once uncaptured: the library's workspaces of this stream
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    with torch.cuda.stream(side):
        begin.record()
        for _ in range(a.steps - 1):
            graph.replay()
        end.record()
    torch.cuda.synchronize()
    free = cache.check()
    print(f"{slots} sequences, {a.steps - 1} steps: {begin.elapsed_time(end) / max(1, a.steps - 1) * 1e3:.1f} us a step, "
          f"{cache.pool.shape[1] - free} pages in use")

    # the same sequences as prompts
    whole = at.int()
    full = model.run(tokens[:, :int(at.max())], lambda layer, q, k, v: S.window_attention(
        turned(q), turned(k), v, window=a.window, sinks=a.sinks, q_lens=whole, kv_lens=whole))
    ref = full.gather(1, (at - 1).view(-1, 1, 1).expand(-1, 1, model.vocab)).squeeze(1).float()
    off = float((step_logits.float() - ref).norm() / ref.norm())
    print(f"last logits against the whole sequences run as prompts: {off:.1e} relative")

    # every second request leaves
    cache.release(ints([i % 2 for i in range(slots)]))
    cache.compact()
    free = cache.check()
    used = cache.pool.shape[1] - free
    print(f"{used} pages in use after every second sequence left, the highest is {int(cache.maps.table.max())}")
    assert int(cache.maps.table.max()) == used - 1
    runtime.call("lc_device_status", stream())
    return off


if __name__ == "__main__":
    main()
