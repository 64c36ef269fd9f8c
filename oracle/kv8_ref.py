"""The 8-bit paged cache and its attention in 64 bits (numpy): norms and rotation of queries and keys, blocks of whole numbers with a scale, their
byte order, softmax attention over what the cache stands for."""
from __future__ import annotations

import numpy as np

BLOCK = 16
MIN_SCALE = 2.0 ** -60


def to_bf16(x):
    """The nearest bf16 (ties to even), as f32; infinities and NaN stay."""
    x = np.asarray(x, np.float32)
    bits = x.view(np.uint32)
    out = ((bits + 0x7FFF + ((bits >> 16) & 1)) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isfinite(x), out, x)


def norm_rotate(x, gain, eps, cos, sin, neighbours=False):
    """x [rows][heads][dim]; cos, sin [rows][pairs] (or None): the angle of every pair of every row."""
    x = np.asarray(x, np.float64).copy()
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gain, np.float64)
    if cos is not None and cos.shape[1]:
        n = cos.shape[1]
        a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if neighbours else (slice(0, n), slice(n, 2 * n))
        c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
        p, q = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = p * c - q * s, q * c + p * s
    return x


def quantise(block):
    """[16][heads][dim] (bf16 values) -> whole numbers, scales [heads] (f32; NaN where a value is not finite)."""
    block = np.asarray(block, np.float32)
    top = np.abs(block).max((0, 2))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        scale = np.maximum(top / np.float32(127), np.float32(MIN_SCALE)).astype(np.float32)
        scale[~np.isfinite(top)] = np.nan
        q = np.rint(block / scale[None, :, None])
    return np.where(np.isfinite(q), q, 0).astype(np.int64), scale


def pack(kq, vq, ks, vs):
    """One page: whole numbers [16][heads][dim], scales [heads] -> bytes [heads][32 dim + 16]."""
    _, heads, dim = kq.shape
    out = np.zeros((heads, 32 * dim + 16), np.uint8)
    t, d = np.arange(BLOCK)[:, None], np.arange(dim)[None]
    out[:, d // 32 * 512 + t % 8 * 64 + d % 32 // 8 * 16 + t // 8 * 8 + d % 8] = kq.transpose(1, 0, 2) + 128
    out[:, 16 * dim + d // 32 * 512 + d % 8 * 64 + t % 8 // 2 * 16 + d % 32 // 8 * 4 + t // 8 * 2 + t % 2] = vq.transpose(1, 0, 2) + 128
    out[:, 32 * dim:32 * dim + 8] = np.stack([ks, vs], 1).astype(np.float32).view(np.uint8)
    return out


class Sequence:
    """What a slot has been given: keys and values [tokens][heads][dim], bf16 values."""

    def __init__(self, heads, dim):
        self.k = self.v = np.zeros((0, heads, dim), np.float32)

    def append(self, start, k, v):
        assert start <= len(self.k)
        self.k, self.v = np.concatenate([self.k[:start], k]), np.concatenate([self.v[:start], v])

    def page(self, block):
        rows = slice(block * BLOCK, block * BLOCK + BLOCK)
        (kq, ks), (vq, vs) = quantise(self.k[rows]), quantise(self.v[rows])
        return pack(kq, vq, ks, vs)

    def held(self):
        """What the cache stands for: keys and values in 64 bits."""
        out = []
        for x in (self.k, self.v):
            x = x.astype(np.float64)
            for b in range(len(x) // BLOCK):
                rows = slice(b * BLOCK, b * BLOCK + BLOCK)
                q, s = quantise(x[rows])
                x[rows] = q * s.astype(np.float64)[None, :, None]
            out.append(x)
        return out

    def value_scales(self):
        """[tokens][heads]: the scale of a token's block; of the block that is not complete the power of two that brings its largest value to [1, 2)."""
        out = np.ones(self.v.shape[:2])
        for b in range((len(self.v) + BLOCK - 1) // BLOCK):
            rows = slice(b * BLOCK, b * BLOCK + BLOCK)
            top = np.abs(self.v[rows].astype(np.float64)).max((0, 2))
            out[rows] = quantise(self.v[rows])[1] if b < len(self.v) // BLOCK else 2.0 ** np.maximum(np.floor(np.log2(np.maximum(top, MIN_SCALE))), -60)
        return out


def attention(q, k, v, begin, end, scale, v_scale):
    """One row: q [heads][dim], k and v [tokens][kv heads][dim], v_scale [tokens][kv heads] -> (out [heads][dim], sum of p |v| per channel, what the
    weights p v_scale would move the output by if each were off by as much as the largest of them, and what the values would, off by their scale
    each). begin >= end: zeros."""
    heads, dim = q.shape
    group = heads // k.shape[1]
    out, size, unit = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros((heads, dim))
    if end <= begin:
        return out, size, unit
    for h in range(heads):
        kk, vv, vs = (x[begin:end, h // group] for x in (k, v, v_scale))
        s = kk @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], size[h] = p @ vv, p @ np.abs(vv)
        unit[h] = (p * vs).max() * (np.abs(vv) / vs[:, None]).sum(0) + p @ vs
    return out, size, unit
