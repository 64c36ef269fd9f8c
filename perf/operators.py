"""Attention over a paged cache held in 8 bits, and what stands in front of it: the norms of queries and keys per head with their
rotation, the append to the cache, the step of single tokens, and prompts.

The cache. A page holds 16 tokens; of every kv head it has one block of 32 dim + 16 bytes: 16 dim bytes of keys, 16 dim bytes of values, the
keys' scale and the values' (f32), 8 bytes of nothing. A byte u stands for (u - 128) scale, with scale = max(largest |x| of the block / 127,
2^-60) and u - 128 = x / scale rounded to the nearest whole number, ties to even. Byte order inside a block:
    keys    [dim / 32][token % 8][dim % 32 / 8][token / 8][dim % 8]
    values  [dim / 32][dim % 8][token % 8 / 2][dim % 32 / 8][token / 8][token % 2]
Tokens of a block that is not complete yet are bf16 rows in open[slot][block % 2][kv head][key, value][token % 16][dim].

Where `own` is false, `run` computes the operators with elementary torch operations; where it is true, with the framework's. `exact` computes
them in 64 bits."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
BLOCK = 16


def listed():
    return [
        # Norms and rotation of the queries and keys of one generated token in f32, as the f32 path has its rows.
        dict(name="rotate-one", op="rotate", dtype="f32", rows=1, heads=32, kv_heads=8, dim=128, axes=1),
        # A prompt of images and text: positions in time, height and width.
        dict(name="rotate-images", op="rotate", dtype="bf16", rows=9001, heads=32, kv_heads=8, dim=128, axes=3),
        # One user's next token goes into the cache and completes a block.
        dict(name="append-one", op="append", batch=1, start=1503, new=1, heads=32, kv_heads=8, dim=128, axes=1),
        # A server's full batch: the next token of 64 sequences of unequal lengths.
        dict(name="append-batch", op="append", batch=64, start=2000, new=1, heads=32, kv_heads=8, dim=128, axes=1),
        # Ragged prompts with pictures in them, a chunk of each.
        dict(name="append-prompts", op="append", batch=6, start=512, new=2777, heads=16, kv_heads=4, dim=128, axes=3),
        # One user in the middle of a chat.
        dict(name="attend-one", op="attend", batch=1, low=1500, high=1500, heads=32, kv_heads=8, dim=128, window=0),
        # A server's batch with 512 to 8192 cached tokens each.
        dict(name="attend-batch", op="attend", batch=64, low=512, high=8192, heads=32, kv_heads=8, dim=128, window=0),
        # Two readers of whole books.
        dict(name="attend-long", op="attend", batch=2, low=100003, high=131072, heads=32, kv_heads=8, dim=128, window=0),
        # Heads of 64 without groups and a sliding window.
        dict(name="attend-window", op="attend", batch=12, low=301, high=5000, heads=12, kv_heads=12, dim=64, window=1024),
        # One long prompt at once.
        dict(name="prompt-long", op="prompt", batch=1, start=0, low=8192, high=8192, heads=32, kv_heads=8, dim=128, window=0),
        # Ragged prompts of a batch, small heads.
        dict(name="prompt-ragged", op="prompt", batch=7, start=0, low=91, high=1777, heads=12, kv_heads=12, dim=64, window=0),
        # A chunk of a prompt behind a long context.
        dict(name="prompt-chunk", op="prompt", batch=1, start=32768, low=500, high=500, heads=32, kv_heads=8, dim=128, window=0),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "append", "attend", "attend", "attend", "prompt", "prompt"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 4, 128), (8, 2, 128), (8, 8, 128), (8, 1, 128), (12, 12, 64), (14, 2, 64), (12, 4, 128)])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim)
    if op == "rotate":
        return dict(case, dtype=rng.choice(["f32", "bf16"]), rows=_log_uniform(rng, 1, 9001), axes=rng.choice([1, 2, 3]))
    if op == "append":
        case["axes"] = rng.choice([1, 1, 3])
        if rng.random() < 0.6:
            return dict(case, batch=_log_uniform(rng, 1, 96), start=_log_uniform(rng, 1, 4000), new=1)
        batch = _log_uniform(rng, 1, 6)
        return dict(case, batch=batch, start=BLOCK * rng.randint(0, 60), new=_log_uniform(rng, 3, 12000 // batch))
    if op == "attend":
        batch = _log_uniform(rng, 1, 64)
        low, high = sorted((_log_uniform(rng, 1, 200000 // batch), _log_uniform(rng, 1, 200000 // batch)))
        return dict(case, batch=batch, low=low, high=high, window=rng.choice([0, 0, 0, 512, 1000]))
    batch = _log_uniform(rng, 1, 6)
    low, high = sorted((_log_uniform(rng, 2, 5000 // batch), _log_uniform(rng, 2, 5000 // batch)))
    return dict(case, batch=batch, start=rng.choice([0, 0, rng.randint(1, 2000)]), low=low, high=high, window=rng.choice([0, 0, 777]))


def _spread(n, low, high):
    """n whole numbers over the range, unequal, the largest one among them."""
    if n == 1:
        return [high]
    at = [(i * 37) % n for i in range(n)]
    return [low + (high - low) * a // (n - 1) for a in at] if math.gcd(37, n) == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def _chunks(case):
    """(first position, tokens) of every sequence's new tokens."""
    b = case["batch"]
    if case["op"] == "append" and case["new"] == 1:
        return [(max(0, case["start"] - 7 * i), 1) for i in range(b)]
    if case["op"] == "append":   # a scheduler cuts prompts at the edges of blocks, their ends are ragged
        return [(BLOCK * (case["start"] // BLOCK + i % 3), n) for i, n in enumerate(_spread(b, max(1, case["new"] // 3), case["new"]))]
    return [(case["start"], n) for n in _spread(b, case["low"], case["high"])]


def _lengths(case):
    """Tokens that the cache holds of every sequence when the attention runs."""
    if case["op"] == "attend":
        return _spread(case["batch"], case["low"], case["high"])
    return [s + n for s, n in _chunks(case)]


def _visible(case):
    """Sum over the query rows of the keys that they see."""
    w = case["window"] or 1 << 60
    if case["op"] == "attend":
        return sum(min(n, w) for n in _lengths(case))
    return sum(min(i + 1, w) for s, n in _chunks(case) for i in range(s, s + n))


def work(case):
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotate":
        size = case["rows"] * (h + g) * d
        return {"bytes": 2 * size * (4 if case["dtype"] == "f32" else 2), "flops": 8 * size}
    if case["op"] == "append":   # rows in, queries out, the tokens' own bytes into the cache; what the blocks that they touch hold comes back as bf16
        rows = sum(n for _, n in _chunks(case))
        touched = sum(s + n - s // BLOCK * BLOCK for s, n in _chunks(case))
        return {"bytes": rows * ((2 * h + 2 * g) * d * 2 + 2 * g * d) + 4 * touched * g * d, "flops": 8 * rows * (h + 2 * g) * d}
    if case["op"] == "attend":
        keys, rows = _visible(case), case["batch"]
    else:
        w = case["window"] or 1 << 60
        keys, rows = sum(s + n - max(0, s + 1 - w) for s, n in _chunks(case)), sum(n for _, n in _chunks(case))
    return {"bytes": keys * g * 2 * d + 4 * rows * h * d, "flops": 4 * _visible(case) * h * d}


# ---- the cache ----------------------------------------------------------------------------------------------------------------
def pack(kq, vq, ks, vs):
    """Whole numbers [pages][kv heads][16][dim] in -127 .. 127 and scales [pages][kv heads] -> blocks [pages][kv heads][32 dim + 16]."""
    p, h, _, d = kq.shape
    k = (kq + 128).to(torch.uint8).view(p, h, 2, 8, d // 32, 4, 8).permute(0, 1, 4, 3, 5, 2, 6).reshape(p, h, 16 * d)
    v = (vq + 128).to(torch.uint8).view(p, h, 2, 4, 2, d // 32, 4, 8).permute(0, 1, 5, 7, 3, 6, 2, 4).reshape(p, h, 16 * d)
    s = torch.stack([ks, vs, torch.zeros_like(ks), torch.zeros_like(ks)], -1).float().contiguous().view(torch.uint8)
    return torch.cat([k, v, s], -1).contiguous()


def unpack(blocks, d):
    """The values that blocks [..., 32 dim + 16] stand for: keys and values [..., 16, dim] in f32."""
    lead = blocks.shape[:-1]
    n = len(lead)
    s = blocks[..., 32 * d:32 * d + 8].contiguous().view(torch.float32)
    at = list(range(n))
    k = blocks[..., :16 * d].reshape(*lead, d // 32, 8, 4, 2, 8).permute(*at, n + 3, n + 1, n, n + 2, n + 4).reshape(*lead, 16, d)
    v = blocks[..., 16 * d:32 * d].reshape(*lead, d // 32, 8, 4, 4, 2, 2).permute(*at, n + 4, n + 2, n + 5, n, n + 3, n + 1).reshape(*lead, 16, d)
    return (k.float() - 128) * s[..., :1, None], (v.float() - 128) * s[..., 1:, None]


def _cache(case, lengths, gen, dev):
    """A cache with `lengths` tokens of every sequence: pages in no order, open rows, page table."""
    h, d, b = case["kv_heads"], case["dim"], case["batch"]
    per = max((n + BLOCK - 1) // BLOCK for n in lengths)
    need = [(n + BLOCK - 1) // BLOCK for n in lengths]
    pages = sum(need) + 3
    perm = torch.randperm(pages, device=dev, generator=gen).int()
    table = torch.zeros((b, per), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    pool = torch.empty((pages, h, 32 * d + 16), dtype=torch.uint8, device=dev)
    for p0 in range(0, pages, 4096):   # blocks whose largest value is 127, of magnitudes that differ from block to block
        n = min(4096, pages - p0)
        q = [(torch.randn((n, h, 16, d), device=dev, generator=gen, dtype=torch.float16) * 36).round().clamp(-127, 127).to(torch.int16) for _ in range(2)]
        for x in q:
            x[:, :, 5, 3] = 127
        scale = [0.03 * torch.exp(0.3 * torch.randn((n, h), device=dev, generator=gen)) for _ in range(2)]
        pool[p0:p0 + n] = pack(*q, *scale)
    rows = torch.randn((b, 2, h, 2, BLOCK, d), device=dev, generator=gen).bfloat16()
    return SimpleNamespace(pool=pool, rows=rows, table=table)


def _tables(positions, dim, dev):
    freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _axes(case, positions, gen, dev):
    """Positions on every axis [axes][rows], and the axis of every rotated pair: the first ones time, then height and width."""
    n, half = case["axes"], case["dim"] // 2
    pair = torch.tensor([min(i * n // half, n - 1) for i in range(half)], dtype=torch.uint8, device=dev)
    rows = positions.shape[0]
    across = torch.randint(0, 64, (n, rows), device=dev, generator=gen, dtype=torch.int32)
    across[0] = positions
    return across, pair


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 13)
    st = SimpleNamespace(case=case, made=None, status=torch.zeros(1, dtype=torch.int32, device=dev))
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    if case["op"] in ("rotate", "append"):
        if case["op"] == "rotate":
            st.positions = torch.arange(case["rows"], device=dev, dtype=torch.int32) + 11
        else:
            chunks = _chunks(case)
            st.positions = ints([i for s, n in chunks for i in range(s, s + n)])
        rows = st.positions.shape[0]
        dtype = torch.float32 if case.get("dtype") == "f32" else torch.bfloat16
        channel = torch.exp(0.5 * torch.randn(((h + 2 * g) * d,), device=dev, generator=gen))   # some channels are far larger than others
        st.qkv = (torch.randn((rows, (h + 2 * g) * d), device=dev, generator=gen) * channel).to(dtype)
        st.q_gain, st.k_gain = (1 + 0.3 * torch.randn(d, device=dev, generator=gen) for _ in range(2))
        st.cos, st.sin = _tables(int(st.positions.max()) + 65, d, dev)
        st.axis_positions, st.pair_axis = _axes(case, st.positions, gen, dev)
    if case["op"] == "append":
        st.cache = _cache(case, [s + n for s, n in chunks], gen, dev)
        slot, first, last, touched, source = [], [], [], [], []
        for i, (s, n) in enumerate(chunks):
            r0, b0 = len(slot), s // BLOCK * BLOCK
            slot += [i] * n
            first += [r0] * n
            last += [r0 + n - 1] * n
            touched += [(i, p) for p in range(b0, s + n)]
            # for the plain form: every token of the touched blocks comes from a new row or (-1 - its place) from an open row, -inf: none yet
            source += [-1 - ((i * 2 + p // BLOCK % 2) * BLOCK + p % BLOCK) if p < s else r0 + p - s if p < s + n else 1 << 40
                       for p in range(b0, (s + n + BLOCK - 1) // BLOCK * BLOCK)]
        st.slot, st.first, st.last, st.lengths = ints(slot), ints(first), ints(last), ints([s + n for s, n in chunks])
        st.touched_slot, st.touched_pos = ints([i for i, _ in touched]), ints([p for _, p in touched])
        st.source = torch.tensor(source, device=dev)
    if case["op"] in ("attend", "prompt"):
        lengths = _lengths(case)
        st.cache, st.lengths = _cache(case, lengths, gen, dev), ints(lengths)
        if case["op"] == "attend":
            st.slot, st.ctx = ints(range(case["batch"])), ints(lengths)
        else:
            chunks = _chunks(case)
            st.slot = ints([i for i, (_, n) in enumerate(chunks) for _ in range(n)])
            st.ctx = ints([p + 1 for s, n in chunks for p in range(s, s + n)])
        st.longest = max(lengths)
        st.q = (1.5 * torch.randn((st.slot.shape[0], h, d), device=dev, generator=gen)).bfloat16()
    return st


# ---- the operators in elementary operations -----------------------------------------------------------------------------------------
def _norm_rotate(x, gain, st):
    """x [rows][heads][dim] in f32: x / rms(x) gain, pairs (i, i + dim / 2) rotated by the angle of their axis's position."""
    half = x.shape[-1] // 2
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain
    pos = st.axis_positions[st.pair_axis.long()].long().t()                                # [rows][half]
    at = torch.arange(half, device=x.device)
    c, s = st.cos[pos, at][:, None], st.sin[pos, at][:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_rows(st):
    h, g, d = (st.case[k] for k in ("heads", "kv_heads", "dim"))
    x = st.qkv.float().view(-1, h + 2 * g, d)
    return _norm_rotate(x[:, :h], st.q_gain, st), _norm_rotate(x[:, h:h + g], st.k_gain, st), x[:, h + g:]


def _plain_append(st):
    q, k, v = _plain_rows(st)
    g, d = st.case["kv_heads"], st.case["dim"]
    n_new, n_open = k.shape[0], st.case["batch"] * 2 * BLOCK
    none = st.source == 1 << 40
    at = torch.where(none, n_new + n_open, torch.where(st.source < 0, n_new - 1 - st.source, st.source))
    out = []
    for x, which in ((k, 0), (v, 1)):
        old = st.cache.rows[:, :, :, which].transpose(2, 3).reshape(-1, g, d).float()
        x = torch.cat([x.bfloat16().float(), old, torch.zeros((1, g, d), device=x.device)])[at].view(-1, BLOCK, g, d)
        complete = ~none.view(-1, BLOCK).any(1)
        scale = (x.abs().amax((1, 3), keepdim=True) / 127).clamp_min(2.0 ** -60)
        held = (x / scale).round() * scale
        out.append(torch.where(complete[:, None, None, None], held, x).view(-1, g, d)[~none].bfloat16())
    return {"q": q.bfloat16(), "k": out[0], "v": out[1]}


def _plain_attention(st):
    """Rows side by side as [sequences][rows], every sequence's cache dense."""
    case, c = st.case, st.cache
    h, g, d = (case[k] for k in ("heads", "kv_heads", "dim"))
    b, per = c.table.shape
    k, v = (x.transpose(2, 3).reshape(b, per * BLOCK, g, d) for x in unpack(c.pool[c.table.long()], d))     # [b][keys][g][d]
    at = torch.arange(per * BLOCK, device=k.device)
    is_open = at[None] >= st.lengths[:, None] // BLOCK * BLOCK                              # the last, incomplete block comes from the open rows
    rows = c.rows[:, at // BLOCK % 2, :, :, at % BLOCK].permute(1, 0, 2, 3, 4).float()      # [b][keys][g][2][d]
    k = torch.where(is_open[:, :, None, None], rows[..., 0, :], k)
    v = torch.where(is_open[:, :, None, None], rows[..., 1, :], v)
    first = torch.searchsorted(st.slot, torch.arange(b, device=k.device, dtype=torch.int32))
    place = torch.arange(st.slot.shape[0], device=k.device) - first[st.slot.long()]
    most = 1 if case["op"] == "attend" else max(n for _, n in _chunks(case))
    q = torch.zeros((b, most, h, d), device=k.device)
    q[st.slot.long(), place] = st.q.float()
    ctx = torch.zeros((b, most), dtype=torch.int64, device=k.device)
    ctx[st.slot.long(), place] = st.ctx.long()
    seen = at < ctx[..., None]
    if case["window"]:
        seen &= at >= ctx[..., None] - case["window"]
    s = torch.einsum("bmgnd,bkgd->bgnmk", q.view(b, most, g, h // g, d) * d ** -0.5, k)
    s.masked_fill_(~seen[:, None, None], -torch.inf)
    s -= s.amax(-1, keepdim=True).clamp_min(-1e30)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.einsum("bgnmk,bkgd->bmgnd", s, v) / total.permute(0, 3, 1, 2, 4)
    return out.reshape(b, most, h * d)[st.slot.long(), place].bfloat16()


# ---- the framework's operators ------------------------------------------------------------------------------------------------------
def _make(st):
    """What a serving loop keeps from step to step: the calls with their buffers."""
    import __graft_entry__
    __graft_entry__.load_package()
    from gptrs_b200 import ops
    case = st.case
    h, g, d = (case[k] for k in ("heads", "kv_heads", "dim"))
    if case["op"] in ("rotate", "append"):
        rotation = ops.QkRotation(h, g, d, st.cos, st.sin, q_gain=st.q_gain, k_gain=st.k_gain, eps=EPS, axis_positions=st.axis_positions, pair_axis=st.pair_axis)
    if case["op"] == "rotate":
        return [ops.QkNormRope(rotation, st.qkv, st.positions, out=torch.empty_like(st.qkv), status=st.status)]
    a = ops.kv8_layout(h, g, d, window=case.get("window", 0))
    c = st.cache
    if case["op"] == "append":
        return [ops.Kv8Append(a, rotation, st.qkv, st.positions, st.slot, st.first, st.last, c.table, c.pool, c.rows, status=st.status),
                ops.Kv8Gather(a, c.pool, c.rows, c.table, st.touched_slot, st.touched_pos, st.lengths, status=st.status)]
    tiles = ops.kv8_tiles(a, [n for _, n in _chunks(case)], st.q.device) if case["op"] == "prompt" else None
    return [ops.Kv8Attention(a, st.q, c.pool, c.rows, c.table, st.slot, st.ctx, st.lengths, st.longest, tiles=tiles, status=st.status)]


def run(st):
    case = st.case
    h, g, d = (case[k] for k in ("heads", "kv_heads", "dim"))
    if own:
        if st.made is None:
            st.made = _make(st)
        if case["op"] == "append":
            q = st.made[0]()
            k, v = st.made[1]()
            return {"q": q, "k": k, "v": v}
        out = st.made[0]()
        return {"q": out.view(-1, h + 2 * g, d)[:, :h], "k": out.view(-1, h + 2 * g, d)[:, h:h + g]} if case["op"] == "rotate" else {"out": out}
    if case["op"] == "rotate":
        q, k, _ = _plain_rows(st)
        return {"q": q.to(st.qkv.dtype), "k": k.to(st.qkv.dtype)}
    return _plain_append(st) if case["op"] == "append" else {"out": _plain_attention(st)}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------------
def _exact_rows(st):
    h, g, d = (st.case[k] for k in ("heads", "kv_heads", "dim"))
    x = st.qkv.double().reshape(-1, h + 2 * g, d)
    rows = x.shape[0]
    angle_c, angle_s = (torch.empty((rows, d // 2), dtype=torch.float64, device=x.device) for _ in range(2))
    for i, axis in enumerate(st.pair_axis.tolist()):
        angle_c[:, i] = st.cos[st.axis_positions[axis].long(), i].double()
        angle_s[:, i] = st.sin[st.axis_positions[axis].long(), i].double()
    z = torch.complex(angle_c, angle_s)[:, None]
    out = []
    for part, gain in ((x[:, :h], st.q_gain), (x[:, h:h + g], st.k_gain)):
        y = part / (part.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * gain.double()
        y = torch.complex(y[..., :d // 2], y[..., d // 2:]) * z
        out.append(torch.cat([y.real, y.imag], -1))
    return out[0], out[1], x[:, h + g:]


def _exact_append(st):
    q, k, v = _exact_rows(st)
    found = {"q": q}
    for name, x, which in (("k", k, 0), ("v", v, 1)):
        parts, row = [], 0
        for i, (s, n) in enumerate(_chunks(st.case)):
            b0 = s // BLOCK * BLOCK
            old = st.cache.rows[i, s // BLOCK % 2, :, which, :s - b0].transpose(0, 1).double()
            t = torch.cat([old, x[row:row + n].bfloat16().double()])
            row += n
            full = t.shape[0] // BLOCK * BLOCK
            c = t[:full].reshape(-1, BLOCK, t.shape[1], t.shape[2])
            scale = torch.clamp((c.abs().amax(dim=3).amax(dim=1) / 127).float(), min=2.0 ** -60).double()[:, None, :, None]
            parts += [(torch.round(c / scale) * scale).reshape(full, t.shape[1], t.shape[2]), t[full:]]
        found[name] = torch.cat(parts)
    return found


def _exact_attention(st):
    case, c = st.case, st.cache
    h, g, d = (case[k] for k in ("heads", "kv_heads", "dim"))
    n = h // g
    out = torch.empty((st.slot.shape[0], h, d), dtype=torch.float64, device=st.q.device)
    row = 0
    spans = [(m - 1, 1) for m in _lengths(case)] if case["op"] == "attend" else _chunks(case)
    tok = torch.arange(BLOCK, device=st.q.device)
    dims = torch.arange(d, device=st.q.device)
    k_at = (dims // 32 * 512 + dims % 32 // 8 * 16 + dims % 8)[None] + (tok % 8 * 64 + tok // 8 * 8)[:, None]
    v_at = 16 * d + (dims // 32 * 512 + dims % 8 * 64 + dims % 32 // 8 * 4)[None] + (tok % 8 // 2 * 16 + tok // 8 * 2 + tok % 2)[:, None]
    for i, (start, new) in enumerate(spans):
        length = start + new
        for kv in range(g):
            blocks = c.pool[c.table[i, :(length + BLOCK - 1) // BLOCK].long(), kv]
            scale = blocks[:, 32 * d:32 * d + 8].contiguous().view(torch.float32).double()
            k = ((blocks[:, k_at.flatten()].double() - 128) * scale[:, :1]).reshape(-1, d)
            v = ((blocks[:, v_at.flatten()].double() - 128) * scale[:, 1:]).reshape(-1, d)
            b, rest = length // BLOCK, length % BLOCK
            if rest:
                k[b * BLOCK:length] = c.rows[i, b % 2, kv, 0, :rest].double()
                v[b * BLOCK:length] = c.rows[i, b % 2, kv, 1, :rest].double()
            k, v = k[:length], v[:length]
            keys = torch.arange(length, device=k.device)
            for r0 in range(0, new, 1024):
                m = min(1024, new - r0)
                at = start + r0 + torch.arange(m, device=k.device)
                lo = at - case["window"] + 1 if case["window"] else torch.zeros_like(at)
                hidden = (keys[None] > at[:, None]) | (keys[None] < lo[:, None])
                for j in range(kv * n, kv * n + n):
                    s = st.q[row + r0:row + r0 + m, j].double() @ k.t() / math.sqrt(d)
                    out[row + r0:row + r0 + m, j] = s.masked_fill(hidden, -math.inf).softmax(-1) @ v
        row += new
    return out.flatten(1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotate":
        q, k, _ = _exact_rows(st)
        return {"q": q, "k": k}
    return _exact_append(st) if case["op"] == "append" else {"out": _exact_attention(st)}
