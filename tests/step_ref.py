"""Plain 64-bit forms of the operators around the serving attention: rotations, shared prefixes and sampling."""
from fractions import Fraction

import numpy as np

# 2 pi to 50 digits
TURN = Fraction("6.2831853071795864769252867665590057683943387987502")


def frequencies(dim, base=10000.0):
    return base ** (-np.arange(0, dim, 2, dtype=np.float64) / max(1, dim))


def cos_sin(positions, f):
    """Of positions [n] times frequencies [m], the angle reduced exactly."""
    cos, sin = np.zeros((len(positions), len(f))), np.zeros((len(positions), len(f)))
    turns = [Fraction(float(x)) / TURN for x in f]
    for i, p in enumerate(positions):
        for j, t in enumerate(turns):
            angle = float((int(p) * t + Fraction(1, 2)) % 1 - Fraction(1, 2)) * float(TURN)
            cos[i, j], sin[i, j] = np.cos(angle), np.sin(angle)
    return cos, sin


def rotate(x, positions, f, interleaved, magnitude=1.0):
    """x[n, heads, d] float64 at positions[n]; the turned heads, and |a| + |b| of each element's pair times the magnitude
    (0 behind the pairs)."""
    rot = 2 * len(f)
    cos, sin = cos_sin(positions, f)
    first = np.arange(0, rot, 2) if interleaved else np.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    out, size = x.copy(), np.zeros_like(x)
    a, b = x[:, :, first], x[:, :, second]
    c, s = cos[:, None] * magnitude, sin[:, None] * magnitude
    out[:, :, first], out[:, :, second] = a * c - b * s, a * s + b * c
    size[:, :, first] = size[:, :, second] = (np.abs(a) + np.abs(b)) * magnitude
    return out, size


def prefixes(table, lens, pages, page_size):
    table = np.asarray(table)
    slots, width = table.shape
    full = [min(max(int(n), 0), width * page_size) // page_size for n in lens]
    groups, leader, shared = {}, list(range(slots)), [0] * slots
    for i in range(slots):
        if full[i] and 0 <= table[i, 0] < pages:
            groups.setdefault(int(table[i, 0]), []).append(i)
    for members in groups.values():
        n = 0
        while n < min(full[i] for i in members) and len({int(table[i, n]) for i in members}) == 1:
            n += 1
        for i in members:
            leader[i] = members[0]
            shared[i] = n * page_size if len(members) > 1 else 0
    return leader, shared, sorted(range(slots), key=lambda i: (leader[i], i))


def sample(x, u, temperature, top_k, top_p, min_p):
    """(token, log of its share) of one row; x float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, -np.inf
    if not temperature > 0:
        return int(order[0]), 0.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / float(temperature)))
    run = np.cumsum(w)
    n = len(order)
    if top_p < 1:
        n = 1 + int((run[:-1] < float(top_p) * run[-1]).sum())
    if min_p > 0:
        n = min(n, int((w >= min(float(min_p), 1.0)).sum()))
    kept = np.sort(order[:n])
    weight = dict(zip(order[:n].tolist(), w[:n].tolist()))
    w = np.array([weight[i] for i in kept.tolist()])
    run = np.cumsum(w)
    u = 0.0 if not u > 0 else float(u)
    at = min(int((run <= u * run[-1]).sum()), int(np.nonzero(w)[0][-1]))
    return int(kept[at]), float(np.log(w[at] / run[-1]))
