"""Plain 64-bit forms of the serving operators: attention row by row, and the page operations on lists."""
import numpy as np

# unit roundoff of the storage types
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def seen(p, n_kv, window, sinks):
    """The keys that position p sees among n_kv."""
    j = np.arange(max(0, min(p + 1, n_kv)))
    return j if window == 0 else j[(j > p - window) | (j < sinks)]


def attend(q, k, v, scale):
    """(o, lse, mean |v| under the weights) of one row; q[d], k, v[n, d] float64."""
    if len(k) == 0:
        return np.zeros_like(q), -np.inf, np.zeros_like(q)
    s = k @ q * scale
    m = s.max()
    w = np.exp(s - m)
    total = w.sum()
    return w @ v / total, m + np.log(total), w @ np.abs(v) / total


def window_attention(q, k, v, scale, window, sinks, q_lens, kv_lens):
    b, s_q, hq, d = q.shape
    h = k.shape[2]
    o, size = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full((b, hq, s_q), -np.inf)
    for x in range(b):
        for i in range(q_lens[x]):
            js = seen(kv_lens[x] - q_lens[x] + i, kv_lens[x], window, sinks)
            for y in range(hq):
                z = y // (hq // h)
                o[x, i, y], lse[x, y, i], size[x, i, y] = attend(q[x, i, y], k[x, js, z], v[x, js, z], scale)
    return o, lse, size


def paged_decode(q, k_pages, v_pages, table, lens, scale, window, sinks):
    slots, hq, d = q.shape
    pages, h, page, _ = k_pages.shape
    o, size, lse = np.zeros(q.shape), np.zeros(q.shape), np.full((slots, hq), -np.inf)
    for x in range(slots):
        n = min(max(int(lens[x]), 0), table.shape[1] * page)
        js = seen(n - 1, n, window, sinks)
        js = js[[0 <= table[x, j // page] < pages for j in js]] if len(js) else js
        at, r = table[x, js // page], js % page
        for y in range(hq):
            z = y // (hq // h)
            o[x, y], lse[x, y], size[x, y] = attend(q[x, y], k_pages[at, z, r], v_pages[at, z, r], scale)
    return o, lse, size


def check_attention(got, lse, ref, dtype):
    """Output rounding (u |o|), the weights' rounding to the storage type before the second product (u sum w |v|), the
    f32 scores and exponentials (1e-4 of sum w |v|: a score of size 20 is off by some 2e-6 absolute, an exponential by
    at most 7.5e-5), and the smallest number of the type.  The log-sum-exp: the same exponentials, averaged, and f32."""
    o, ref_lse, size = ref
    u = U[dtype]
    tol = u * np.abs(o) + (1.01 * u + 1e-4) * size + 2.0 ** -24
    bad = ~(np.abs(got - o) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], o[bad][:5], tol[bad][:5])
    empty = np.isneginf(ref_lse)
    assert (np.isneginf(lse) == empty).all()
    off = np.abs(lse[~empty] - ref_lse[~empty])
    assert (off <= 1e-4 + 4e-6 * np.abs(ref_lse[~empty])).all(), off.max()


class Pages:
    """A cache's maps and pool as plain lists and an array."""

    def __init__(self, table, lens, refs, page, pool=None):
        self.table, self.lens, self.refs = [list(map(int, r)) for r in table], list(map(int, lens)), list(map(int, refs))
        self.page, self.pool = page, pool

    def held(self, n):
        return -(-n // self.page)

    def free(self):
        return [i for i, n in enumerate(self.refs) if n == 0]

    def status(self, code=0):
        return [code, len(self.free())]

    def extend(self, add):
        width = len(self.table[0]) if self.table else 0
        want = [self.held(n + a) for n, a in zip(self.lens, add)]
        if any(a < 0 for a in add) or any(w > width for w in want):
            return self.status(-1)
        need = sum(w - self.held(n) for w, n in zip(want, self.lens))
        free = self.free()
        if need > len(free):
            return self.status(need - len(free))
        for i, a in enumerate(add):
            for j in range(self.held(self.lens[i]), want[i]):
                self.table[i][j] = free.pop(0)
                self.refs[self.table[i][j]] = 1
            self.lens[i] += a
        return self.status()

    def write(self, k, v, add, planes=(0, 1)):
        for i, a in enumerate(add):
            for t in range(a):
                j = self.lens[i] - a + t
                at = self.table[i][j // self.page]
                self.pool[planes[0], at, :, j % self.page] = k[i, t]
                self.pool[planes[1], at, :, j % self.page] = v[i, t]

    def fork(self, parent):
        if any(p < -1 or p >= len(self.lens) for p in parent):
            return self.status(-1)
        table, lens = [list(r) for r in self.table], list(self.lens)
        new, new_lens, refs, kept, moves = [], [], [0] * len(self.refs), set(), []
        for i, p in enumerate(parent):
            row = list(table[p]) if p >= 0 else [-1] * len(table[i])
            n = lens[p] if p >= 0 else 0
            own = n // self.page if n % self.page and p in kept else None
            if p >= 0 and n % self.page:
                kept.add(p)
            for j, at in enumerate(row):
                if j != own and at >= 0:
                    refs[at] += 1
            if own is not None:
                moves.append((i, own, n % self.page))
            new.append(row)
            new_lens.append(n)
        free = [i for i, n in enumerate(refs) if n == 0]
        if len(moves) > len(free):
            return self.status(len(moves) - len(free))
        self.table, self.lens, self.refs = new, new_lens, refs
        for i, j, n in moves:
            to, at = free.pop(0), new[i][j]
            if self.pool is not None:
                self.pool[:, to, :, :n] = self.pool[:, at, :, :n]
            new[i][j], refs[to] = to, 1
        return self.status()

    def release(self, gone):
        for i, g in enumerate(gone):
            if g:
                for j in range(self.held(self.lens[i])):
                    if self.table[i][j] >= 0:
                        self.refs[self.table[i][j]] -= 1
                    self.table[i][j] = -1
                self.lens[i] = 0
        return self.status()

    def trim(self, window, sinks):
        for i, n in enumerate(self.lens):
            for j in range(self.held(n)):
                tokens = range(j * self.page, (j + 1) * self.page)
                if all(t <= n - window and t >= sinks for t in tokens):
                    if self.table[i][j] >= 0:
                        self.refs[self.table[i][j]] -= 1
                    self.table[i][j] = -1
        return self.status()

    def compact(self):
        used = sum(n > 0 for n in self.refs)
        holes = [i for i in range(used) if self.refs[i] == 0]
        movers = [i for i in range(used, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(movers, holes))
        for at, hole in to.items():
            if self.pool is not None:
                self.pool[:, hole] = self.pool[:, at]
            self.refs[hole], self.refs[at] = self.refs[at], 0
        self.table = [[to.get(at, at) for at in row] for row in self.table]
        return self.status()
