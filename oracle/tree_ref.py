"""Trees of drafted tokens and scores against a vocabulary, restated in numpy in 64 bits."""
from __future__ import annotations

import numpy as np


def ancestors(parent):
    """Of every node the numbers of its ancestors and itself, from the top."""
    found = []
    for i, up in enumerate(parent):
        found.append((found[up] if 0 <= up < i else []) + [i])
    return found


def rotate(x, position, cos, sin):
    """x [n][heads][dim], the first 2 half channels turned in pairs (i, i + half) by the tables' row `position`."""
    half = cos.shape[1]
    c, s = (np.asarray(t, np.float64)[position][:, None] for t in (cos, sin))
    y = x.astype(np.float64).copy()
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def attention(q, keys, values, parent, length, scale, lost=()):
    """q [n][heads][dim]; keys, values [length + n][kv heads][dim]; `lost`: positions that nobody sees. Returns the output and sum p |v| [n][heads][dim]."""
    n, heads, dim = q.shape
    group = heads // keys.shape[1]
    out, mass = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    for i, seen in enumerate(ancestors(parent)):
        at = [p for p in list(range(length)) + [length + j for j in seen] if p not in lost] if len(lost) else np.r_[0:length, length + np.array(seen)]
        if not len(at):
            continue
        for h in range(heads):
            k, v = keys[at, h // group].astype(np.float64), values[at, h // group].astype(np.float64)
            z = k @ q[i, h].astype(np.float64) * scale
            with np.errstate(invalid="ignore"):
                w = np.exp(z - z.max())
                w /= w.sum()
                out[i, h], mass[i, h] = w @ v, w @ np.abs(v)
    return out, mass


def accept(parent, token, pick):
    """(path, what follows it)."""
    if not len(parent):
        return [], -1
    path = [0]
    while True:
        fits = [i for i, up in enumerate(parent) if 0 <= up < i and up == path[-1] and token[i] == pick[path[-1]]]
        if not fits:
            return path, int(pick[path[-1]])
        path.append(fits[0])


def _mix(x):
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x7feb352d)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0x846ca68b)
    return x ^ (x >> np.uint32(16))


def noise(seed, rows, vocab):
    """g of every row and token: -log(-log(1 - v)), v in f32."""
    with np.errstate(over="ignore"):
        at = np.arange(vocab, dtype=np.uint32)[None] + np.uint32(0x9e3779b9) * (np.arange(rows, dtype=np.uint32)[:, None] + np.uint32(1))
    h = _mix(np.uint32(seed) ^ _mix(at))
    v = np.minimum((h.astype(np.float32) + np.float32(0.5)) * np.float32(2.0 ** -32), np.float32(1 - 2.0 ** -24)).astype(np.float64)
    return -np.log(-np.log1p(-v))


def logits(hidden, weight, bias=None, cap=0.0):
    """z [rows][vocab] and sum |x w| (what the products' errors go by)."""
    x, w = hidden.astype(np.float64), weight.astype(np.float64)
    z = x @ w.T
    if bias is not None:
        z = z + np.asarray(bias, np.float64)
    if cap:
        z = np.where(np.isneginf(z), z, cap * np.tanh(z / cap))   # what a bias leaves out stays out
    return z, np.abs(x) @ np.abs(w).T


def lse(z):
    m = z.max(-1, keepdims=True)
    return (m + np.log(np.exp(z - m).sum(-1, keepdims=True)))[:, 0]
