"""Norms and rotation of queries and keys, the append to the 8-bit paged cache and the attention that reads it, against the oracle in 64 bits.

Tolerances. bf16 output: half a step, 2^-8 of the value that is rounded. Attention: weights times the values' scales are f16, off by 2^-11 of themselves,
or by half a step of the smallest numbers, 2^-25, where the largest is at least 1. The first moves the output by at most 2^-11 sum p |v|, the second by
2^-25 of what an error as large as the largest weight in every one of them would; the denominator is summed in front of the rounding. Values of the
block that is not complete are f16 too, with the largest in [1, 2): off by at most 2^-25 of the unit (bf16 has fewer bits). Scores
are f32 (sums of dim products; an error of 2^-24 of 2^6 in an exponent is 2^-18 of a weight), which the other half of 2^-10 sum p |v| covers. So
2^-8 |want| + (1 + 2^-8) (2^-10 sum p |v| + 2^-25 unit)."""
import numpy as np
import pytest
import torch

from gptrs_b200 import ops
from oracle import kv8_ref as kr

pytestmark = pytest.mark.gpu


def _np(t):
    return t.float().cpu().numpy()


def _ints(v, cuda):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=cuda)


# ---- norms and rotation --------------------------------------------------------------------------------------------------------
def _rotation(rng, heads, kv, dim, pairs, rows, cuda, gains, neighbours, axes, positions=40, interleaved=False):
    ang = rng.uniform(-4, 4, (positions, pairs))
    cos, sin = (torch.tensor(f(ang), dtype=torch.float32, device=cuda) for f in (np.cos, np.sin))
    gain = [torch.tensor(rng.normal(1, 0.5, dim), dtype=torch.float32, device=cuda) if gains else None for _ in range(2)]
    pos = rng.integers(0, positions, rows)
    axis_pos = np.stack([pos] + [rng.integers(0, positions, rows) for _ in range(axes - 1)])
    axis_of = np.arange(pairs) % axes if interleaved else np.arange(pairs) * axes // max(pairs, 1)
    many = axes > 1
    rot = ops.QkRotation(heads, kv, dim, cos if pairs else None, sin if pairs else None, *gain, eps=1e-5, neighbours=neighbours,
                         axis_positions=_ints(axis_pos, cuda) if many else None, pair_axis=torch.tensor(axis_of, dtype=torch.uint8, device=cuda) if many and pairs else None)
    c, s = (np.stack([_np(t)[axis_pos[axis_of[i]], i] for i in range(pairs)], 1) if pairs else None for t in (cos, sin))
    return rot, pos, c, s, [None if g is None else _np(g) for g in gain]


ROTATIONS = [  # heads, kv, dim, pairs, rows, gains, neighbours, axes
    (4, 2, 128, 64, 1, True, False, 1), (32, 8, 128, 64, 19, True, False, 3), (3, 1, 64, 32, 257, True, True, 1), (5, 5, 96, 24, 7, True, False, 2),
    (2, 1, 80, 40, 3, False, False, 1), (2, 2, 6, 3, 5, True, False, 3), (1, 1, 512, 256, 2, True, False, 1), (2, 1, 256, 128, 4, True, True, 4),
    (32, 8, 128, 64, 1201, True, False, 3), (3, 1, 64, 16, 901, True, True, 1), (40, 10, 64, 32, 610, False, False, 2), (2, 2, 32, 0, 700, True, False, 1), (5, 1, 96, 40, 400, True, False, 2),
    (2, 1, 62, 13, 9, True, True, 2), (8, 2, 128, 0, 6, True, False, 1), (7, 7, 64, 30, 8, False, True, 1), (2, 1, 2, 1, 33, True, False, 1), (1, 1, 264, 100, 3, True, False, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,pairs,rows,gains,neighbours,axes", ROTATIONS)
def test_norm_rope(cuda, dtype, heads, kv, dim, pairs, rows, gains, neighbours, axes):
    rng = np.random.default_rng(dim * 31 + rows)
    rot, pos, c, s, (qg, kg) = _rotation(rng, heads, kv, dim, pairs, rows, cuda, gains, neighbours, axes, interleaved=rows % 2 == 0)
    width = (heads + 2 * kv) * dim
    x = torch.tensor(rng.normal(0, 2, (rows, width)), dtype=torch.float32, device=cuda).to(dtype)
    out = ops.qk_norm_rope(rot, x, _ints(pos, cuda))
    got, y = _np(out).reshape(rows, -1, dim), _np(x).reshape(rows, -1, dim)
    want = np.concatenate([kr.norm_rotate(y[:, :heads], qg, 1e-5, c, s, neighbours), kr.norm_rotate(y[:, heads:heads + kv], kg, 1e-5, c, s, neighbours)], 1)
    assert np.array_equal(got[:, heads + kv:], y[:, heads + kv:])
    # one rounding, and f32: sums of squares (a few 2^-24, halved by the root), the root's 2^-22, three products and a sum of two terms of the
    # size of the pair's length
    size = np.abs(want).max(-1, keepdims=True)
    tol = (2 ** -8 if dtype == torch.bfloat16 else 0) * np.abs(want) + 2 ** -19 * size
    assert (np.abs(got[:, :heads + kv] - want) <= tol).all()
    # a strided source and target, and in place
    wide = torch.full((rows, width + 16), 7.0, dtype=dtype, device=cuda)
    wide[:, 8:8 + width] = x
    to = torch.full((rows, width + 5), 9.0, dtype=dtype, device=cuda)
    ops.qk_norm_rope(rot, wide[:, 8:8 + width], _ints(pos, cuda), out=to[:, 3:3 + width])
    ops.qk_norm_rope(rot, wide[:, 8:8 + width], _ints(pos, cuda), out=wide[:, 8:8 + width])
    # the other widths of loads sum the squares in another order
    near = (2 ** -7 if dtype == torch.bfloat16 else 2 ** -18) * np.maximum(np.abs(_np(out)), np.repeat(np.abs(_np(out)).reshape(rows, -1, dim).max(-1), dim, 1) * 2 ** -10)
    for t in (wide[:, 8:8 + width], to[:, 3:3 + width]):
        assert (np.abs(_np(t) - _np(out)) <= near + 2 ** -18 * np.repeat(np.abs(_np(out)).reshape(rows, -1, dim).max(-1), dim, 1)).all()
    assert (wide[:, :8] == 7).all() and (wide[:, 8 + width:] == 7).all() and (to[:, :3] == 9).all() and (to[:, 3 + width:] == 9).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,pairs,rows,gains,neighbours,axes", [  # pieces of eight bytes in bf16; rows that no stage of the ring holds; few and many rows
    (6, 2, 64, 20, 50, True, False, 3), (3, 1, 72, 36, 301, True, True, 1), (64, 8, 128, 64, 149, True, False, 1), (96, 8, 128, 48, 307, True, True, 2), (32, 8, 128, 64, 147, True, False, 1)])
def test_norm_rope_in_other_pieces(cuda, dtype, heads, kv, dim, pairs, rows, gains, neighbours, axes):
    test_norm_rope(cuda, dtype, heads, kv, dim, pairs, rows, gains, neighbours, axes)


def test_norm_rope_positions_outside_and_channels_that_stay(cuda):
    rng = np.random.default_rng(3)
    rot, pos, c, s, _ = _rotation(rng, 2, 1, 64, 16, 4, cuda, False, False, 1)
    x = torch.tensor(rng.normal(0, 1, (4, 256)), dtype=torch.float32, device=cuda)
    x[2, 40], x[3, 60] = float("inf"), float("nan")        # behind the rotated channels of a head: only they are touched
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    pos[1] = 40
    out = ops.qk_norm_rope(rot, x, _ints(pos, cuda), status=status)
    assert int(status) == 2
    ok = ops.qk_norm_rope(rot, x, _ints([pos[0], 0, pos[2], pos[3]], cuda))
    assert torch.equal(out.nan_to_num(nan=-5.0), ok.nan_to_num(nan=-5.0))                         # position 0 takes its place
    assert torch.isinf(out[2, 40]) and torch.isnan(out[3, 60]) and int((~torch.isfinite(out)).sum()) == 2
    assert torch.equal(out[:, 32:64].nan_to_num(nan=-5.0), x[:, 32:64].nan_to_num(nan=-5.0))


@pytest.mark.parametrize("rows", [3, 400])
def test_norm_rope_between_the_rows_of_the_source(cuda, rows):
    rng = np.random.default_rng(rows)
    rot, pos, c, s, _ = _rotation(rng, 4, 2, 64, 32, rows, cuda, True, False, 1)
    both = torch.randn((rows, 2 * 512), device=cuda).bfloat16()
    x = both[:, :512].clone()
    want = ops.qk_norm_rope(rot, x, _ints(pos, cuda))
    ops.qk_norm_rope(rot, both[:, :512], _ints(pos, cuda), out=both[:, 512:])
    assert torch.equal(both[:, :512], x) and torch.equal(both[:, 512:], want)


# ---- the cache -----------------------------------------------------------------------------------------------------------------
class Cache:
    """A cache on the GPU beside the oracle's sequences."""

    def __init__(self, cuda, heads, kv, dim, slots, per, window=0, scale=0.0, seed=0, extra=3):
        self.a, self.cuda, self.rng = ops.kv8_layout(heads, kv, dim, window, scale), cuda, np.random.default_rng(seed)
        self.heads, self.kv, self.dim, self.slots = heads, kv, dim, slots
        self.pool = torch.randint(0, 256, (slots * per + extra, kv, self.a.block_bytes), dtype=torch.uint8, device=cuda)   # nothing may depend on what was there
        self.rows = ops.new_kv8_open(self.a, slots, cuda)
        self.rows.fill_(float("nan"))
        self.table = _ints(self.rng.permutation(slots * per + extra)[:slots * per].reshape(slots, per), cuda)
        self.seq = [kr.Sequence(kv, dim) for _ in range(slots)]
        self.status = torch.zeros(1, dtype=torch.int32, device=cuda)
        self.halves = [{} for _ in range(slots)]   # block whose rows a half of a slot's open rows has

    def append(self, runs, qkv=None, rotation=None, pad=()):
        """runs: (slot, start, tokens) each; pad: rows of padding in front of those runs (by number)."""
        slot, pos, first, last, at = [], [], [], [], 0
        for i, (s, start, n) in enumerate(runs):
            if i in pad:
                slot, pos, first, last, at = slot + [-1], pos + [12345678], first + [-9], last + [99999], at + 1
            slot, pos, first, last = slot + [s] * n, pos + list(range(start, start + n)), first + [at] * n, last + [at + n - 1] * n
            at += n
        width = (self.heads + 2 * self.kv) * self.dim
        if qkv is None:
            qkv = torch.tensor(self.rng.normal(0, 1, (at, width)) * np.exp(self.rng.normal(0, 1, (1, width))), dtype=torch.float32).bfloat16().to(self.cuda)
        q = torch.full((at, self.heads, self.dim), 5.0, dtype=torch.bfloat16, device=self.cuda)
        ops.kv8_append(self.a, rotation, qkv, _ints(pos, self.cuda), _ints(slot, self.cuda), _ints(first, self.cuda), _ints(last, self.cuda), self.table, self.pool, self.rows, q=q,
                       status=self.status)
        x, r = _np(qkv).reshape(at, -1, self.dim), 0
        for i, (s, start, n) in enumerate(runs):
            r += i in pad
            if rotation is None:
                self.seq[s].append(start, x[r:r + n, self.heads:self.heads + self.kv], x[r:r + n, self.heads + self.kv:])
            for b in range(max(start // 16, (start + n - 1) // 16 - 1), (start + n - 1) // 16 + 1):
                self.halves[s][b % 2] = b
            r += n
        return qkv, q

    def fill(self, lengths):
        self.append([(i, 0, n) for i, n in enumerate(lengths) if n])

    def lengths(self):
        return _ints([len(s.k) for s in self.seq], self.cuda)

    def check_bytes(self):
        pool, table, rows = self.pool.cpu().numpy(), self.table.cpu().numpy(), _np(self.rows)
        for i, s in enumerate(self.seq):
            n = len(s.k)
            for b in range(n // 16):
                assert np.array_equal(pool[table[i, b]], s.page(b)), (i, b)
            for p in range(max(0, (n - 1) // 16 - 1) * 16, n):
                if self.halves[i][p // 16 % 2] != p // 16:
                    continue
                assert np.array_equal(rows[i, p // 16 % 2, :, 0, p % 16], s.k[p]) and np.array_equal(rows[i, p // 16 % 2, :, 1, p % 16], s.v[p]), (i, p)

    def attend(self, rows, tiles=None, splits=None, q=None, want=True, scale=None, longest=None):
        """rows: (slot, ctx_len) each; checks every row against the oracle."""
        n = len(rows)
        if q is None:
            q = torch.tensor(self.rng.normal(0, 1.5, (n, self.heads, self.dim)), dtype=torch.float32).bfloat16().to(self.cuda)
        out = torch.full((n, self.heads * self.dim), 3.0, dtype=torch.bfloat16, device=self.cuda)
        lengths = self.lengths()
        longest = max([c for _, c in rows] + [1]) if longest is None else longest
        ops.kv8_attention(self.a, q, self.pool, self.rows, self.table, _ints([s for s, _ in rows], self.cuda), _ints([c for _, c in rows], self.cuda), lengths, longest,
                          tiles=None if tiles is None else ops.kv8_tiles(self.a, tiles, self.cuda), splits=splits, out=out, status=self.status)
        if want:
            assert int(self.status) == 0
            self.check(rows, q, out)
        return q, out

    def check(self, rows, q, out, every=None):
        held = {}
        got, qn = _np(out).reshape(len(rows), self.heads, self.dim), _np(q)
        for i, (s, c) in enumerate(rows):
            if every and i % every and i < len(rows) - 3:
                continue
            if s < 0:
                assert (got[i] == 3).all()
                continue
            if s not in held:
                held[s] = *self.seq[s].held(), self.seq[s].value_scales()
            k, v, vs = held[s]
            begin = max(0, c - self.a.window) if self.a.window else 0
            w, size, unit = kr.attention(qn[i], k, v, begin, c, self.a.scale, vs)
            if c <= 0:
                assert (got[i] == 0).all()
            else:
                off = np.abs(got[i] - w) - 2 ** -8 * np.abs(w) - (1 + 2 ** -8) * (2 ** -10 * size + 2 ** -25 * unit)
                assert (off <= 0).all(), (i, s, c, off.max())


RUNS = [[(0, 0, 1)], [(0, 0, 16)], [(0, 0, 17), (1, 0, 15), (2, 0, 33)], [(1, 0, 100)], [(2, 0, 5), (0, 0, 290), (1, 0, 64)]]


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (3, 3, 64), (5, 1, 128)])
@pytest.mark.parametrize("runs", RUNS)
def test_append_writes_these_bytes(cuda, heads, kv, dim, runs):
    c = Cache(cuda, heads, kv, dim, 3, 20, seed=len(runs) + dim)
    qkv, q = c.append(runs)
    assert torch.equal(q.flatten(1), qkv[:, :heads * dim]) and int(c.status) == 0
    c.check_bytes()


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("prompts", [[150, 90], [2500, 1800], []])
def test_single_tokens_beside_prompts(cuda, heads, kv, dim, prompts):
    """Many runs of one row between long ones, some of them in the middle of a block: lists that are short, longer than the slots, and long."""
    c = Cache(cuda, heads, kv, dim, 40, 320, seed=sum(prompts) + dim)   # (9 + 2 x 2500 tokens: 314 blocks)
    singles = list(range(len(prompts), 40))
    c.append([(i, 0, 1 + (7 * i) % 33) for i in singles] + [(i, 0, 9) for i in range(len(prompts))])
    for turn in range(2):
        at = {i: 1 + (7 * i) % 33 + turn for i in singles}
        runs = [(i, at[i], 1) for i in singles]
        for i, n in enumerate(prompts):
            runs.insert(5 + 17 * i, (i, 9 + turn * n, n))
        qkv, q = c.append(runs, pad=(3,))
        q, flat = q.flatten(1), qkv[:, :heads * dim]
        pad = sum(n for _, _, n in runs[:3])
        assert (q[pad] == 5).all() and torch.equal(q[:pad], flat[:pad]) and torch.equal(q[pad + 1:], flat[pad + 1:])
        c.check_bytes()
    assert int(c.status) == 0


def test_bad_rows_among_many(cuda):
    """The same where sixteen rows go together: what is bad is reported, the others arrive."""
    c = Cache(cuda, 4, 2, 64, 3, 22)
    n = 310
    slot, pos = [0] * n + [7] * 20 + [1] * 17 + [2] * 16, list(range(n)) + list(range(20)) + list(range(17)) + list(range(-1, 15))
    first = [0] * n + [n] * 20 + [n + 20] * 17 + [n + 37] * 16
    last = [n - 1] * n + [n + 19] * 20 + [n + 36] * 17 + [n + 52] * 16
    rows = len(slot)
    qkv = torch.randn((rows, 8 * 64), device=cuda).bfloat16()
    before = c.pool.clone()
    ops.kv8_append(c.a, None, qkv, _ints(pos, cuda), _ints(slot, cuda), _ints(first, cuda), _ints(last, cuda), c.table, c.pool, c.rows, status=c.status)
    assert int(c.status) == 2
    x = _np(qkv).reshape(rows, -1, 64)
    for s, at, m in ((0, 0, n), (1, n + 20, 17)):
        c.seq[s].append(0, x[at:at + m, 4:6], x[at:at + m, 6:8])
        for b in range(max(0, (m - 1) // 16 - 1), (m - 1) // 16 + 1):
            c.halves[s][b % 2] = b
    c.check_bytes()
    table = c.table.cpu().numpy()
    others = [i for i in range(before.shape[0]) if i not in list(table[0, :n // 16]) + [table[1, 0]]]
    assert torch.equal(c.pool[others], before[others])


@pytest.mark.parametrize("step", [1, 3, 16, 21, 37, 300])
def test_cuts_do_not_matter(cuda, step):
    """The same tokens in calls of any size leave the same bytes; both sequences at once, out of step."""
    c = Cache(cuda, 4, 2, 64, 2, 22, seed=step)
    at = [0, 0]
    while min(at) < 300:
        runs = []
        for i, n in enumerate((step, step + 4)):
            n = min(n, 300 - at[i])
            if n > 0:
                runs.append((i, at[i], n))
                at[i] += n
        c.append(runs)
        if step > 2 or max(at) % 50 < 2:
            c.check_bytes()
    c.check_bytes()
    assert int(c.status) == 0


def test_going_back(cuda):
    """A sequence goes on from any position of a block whose rows are there and from the start of any block."""
    c = Cache(cuda, 4, 2, 128, 2, 10)
    for start, n in [(0, 40), (37, 9), (32, 1), (17, 20), (36, 1), (16, 3), (18, 30), (0, 7), (3, 100), (96, 30), (111, 1), (110, 40)]:
        assert start % 16 == 0 or c.halves[0][start // 16 % 2] == start // 16
        c.append([(0, start, n), (1, start, n)])
        c.check_bytes()
    assert int(c.status) == 0


def test_padding_rows_and_pages_that_are_not_kept(cuda):
    c = Cache(cuda, 4, 2, 64, 3, 8)
    before = c.pool.clone()
    c.table[1, 1] = -1
    _, q = c.append([(0, 0, 20), (1, 0, 50), (2, 0, 300 - 256)], pad=(0, 2))
    assert int(c.status) == 0 and (q[0] == 5).all() and (q[71] == 5).all() and not (q[1:71] == 5).all(2).any()
    c.seq[1].k, c.seq[1].v, keep = c.seq[1].k[:16], c.seq[1].v[:16], c.seq[1]
    table = c.table.cpu().numpy()
    assert np.array_equal(c.pool[table[1, 0]].cpu().numpy(), keep.page(0))
    written = [table[0, 0], table[1, 0], table[1, 2], table[2, 0], table[2, 1]]
    others = [i for i in range(before.shape[0]) if i not in written]
    assert torch.equal(c.pool[others], before[others])


@pytest.mark.parametrize("what", ["slot", "page", "far", "run", "before"])
def test_bad_rows_are_reported_and_left_out(cuda, what):
    """A bad entry writes nothing outside its own place; the other sequence's tokens arrive."""
    c = Cache(cuda, 4, 2, 64, 2, 4)
    before, rows_before = c.pool.clone(), c.rows.clone()
    slot, pos, first, last = [0] * 20 + [1] * 20, list(range(20)) * 2, [0] * 20 + [20] * 20, [19] * 20 + [39] * 20
    table = c.table.clone()
    if what == "slot":
        slot[20:] = [2] * 20
    elif what == "page":
        c.table[1, 0] = c.pool.shape[0]
    elif what == "far":
        pos[20:] = range(64, 84)
    elif what == "run":
        last[20:] = [40] * 20
    else:
        pos[20:] = range(-3, 17)
    width = 8 * 64
    qkv = torch.randn((40, width), device=cuda).bfloat16()
    ops.kv8_append(c.a, None, qkv, _ints(pos, cuda), _ints(slot, cuda), _ints(first, cuda), _ints(last, cuda), c.table, c.pool, c.rows, status=c.status)
    assert int(c.status) == 2
    x = _np(qkv).reshape(40, 8, 64)
    c.seq[0].append(0, x[:20, 4:6], x[:20, 6:])
    c.halves[0], c.table = {0: 0, 1: 1}, table
    c.check_bytes()
    others = [i for i in range(before.shape[0]) if i != int(table[0, 0])]
    if what != "run":
        assert torch.equal(c.pool[others], before[others])
    if what in ("slot", "run", "before"):
        assert torch.equal(c.rows[1].view(torch.int16), rows_before[1].view(torch.int16)) or what == "before"


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_positions_behind_the_page_table(cuda, n):
    """Rows behind the table's pages are reported and left out, whether they complete a block or not; rows in front of them arrive. Nothing is read back from there."""
    c = Cache(cuda, 4, 2, 64, 2, 4)       # 64 tokens
    c.append([(0, 0, 60), (1, 0, 64)])
    for slot, start in ((1, 64), (1, 70), (0, 60)):
        rows = n + (4 if start == 60 else 0)
        pool, opened = c.pool.clone(), c.rows.clone()
        qkv = torch.randn((rows, 8 * 64), device=cuda).bfloat16()
        q = torch.full((rows, 4, 64), 5.0, dtype=torch.bfloat16, device=cuda)
        c.status.zero_()
        ops.kv8_append(c.a, None, qkv, _ints(range(start, start + rows), cuda), _ints([slot] * rows, cuda), _ints([0] * rows, cuda), _ints([rows - 1] * rows, cuda), c.table, c.pool, c.rows,
                       q=q, status=c.status)
        assert int(c.status) == 2
        if start == 60:
            x = _np(qkv).reshape(rows, 8, 64)
            c.seq[0].append(60, x[:4, 4:6], x[:4, 6:])
            assert torch.equal(q[:4].flatten(1), qkv[:4, :256]) and (q[4:] == 5).all()
        else:
            assert torch.equal(c.pool, pool) and torch.equal(c.rows.view(torch.int16), opened.view(torch.int16)) and (q == 5).all()
        c.check_bytes()
    c.status.zero_()
    k, v = ops.kv8_gather(c.a, c.pool, c.rows, c.table, _ints([0, 0], cuda), _ints([63, 64], cuda), _ints([65, 65], cuda), status=c.status)
    assert int(c.status) == 2 and k[0].any() and not k[1].any() and not v[1].any()


@pytest.mark.parametrize("heads,kv,dim,pairs,neighbours,axes", [(8, 2, 128, 64, False, 1), (6, 3, 64, 32, True, 3), (8, 8, 128, 32, False, 2), (4, 1, 64, 8, True, 1), (16, 2, 128, 64, False, 3)])
@pytest.mark.parametrize("n", [1, 45, 700])
def test_append_norms_and_rotates(cuda, heads, kv, dim, pairs, neighbours, axes, n):
    c = Cache(cuda, heads, kv, dim, 2, 50, seed=dim + n)
    c.append([(0, 0, 37)])
    runs = [(0, 37, n), (1, 0, n)] if n > 1 else [(1, 0, 1), (0, 37, 1)]
    rot, _, cs, sn, (qg, kg) = _rotation(c.rng, heads, kv, dim, pairs, 2 * n, cuda, True, neighbours, axes, positions=800, interleaved=True)
    if axes == 1:   # the rows' own positions
        pos = np.concatenate([np.arange(s, s + m) for _, s, m in runs])
        cs, sn = (_np(rot.tensors[k])[pos] for k in ("cos", "sin"))
    qkv, q = c.append(runs, rotation=rot)
    assert int(c.status) == 0
    x = _np(qkv).reshape(2 * n, -1, dim)
    wq, wk = kr.norm_rotate(x[:, :heads], qg, 1e-5, cs, sn, neighbours), kr.norm_rotate(x[:, heads:heads + kv], kg, 1e-5, cs, sn, neighbours)
    # as in test_norm_rope
    assert (np.abs(_np(q) - wq) <= 2 ** -8 * np.abs(wq) + 2 ** -19 * np.abs(wq).max(-1, keepdims=True)).all()
    r = 0
    for s, start, m in runs:
        c.seq[s].append(start, kr.to_bf16(wk[r:r + m]), x[r:r + m, heads + kv:])
        r += m
    for s in range(2):
        total = len(c.seq[s].k)
        k, v = ops.kv8_gather(c.a, c.pool, c.rows, c.table, _ints([s] * total, cuda), _ints(range(total), cuda), c.lengths(), dtype=torch.float32, status=c.status)
        hk, hv = c.seq[s].held()
        assert np.array_equal(_np(v), hv.astype(np.float32))
        # a key may be rounded to the other neighbour in bf16 (2^-7 of it) and from there to the next whole number (a step); a scale that was
        # taken from such a key moves all values of the block by 2^-7 of themselves
        top = np.abs(hk).max(-1, keepdims=True)
        block = np.stack([np.abs(hk[p // 16 * 16:p // 16 * 16 + 16]).max((0, 2)) for p in range(total)])[..., None]
        assert (np.abs(_np(k) - hk) <= 2 ** -6 * top + 1.02 * block / 127).all()
        assert (np.abs(_np(k) - hk) > 2 ** -6 * np.abs(hk) + 2 ** -19 * top).mean() < 0.01      # few cross a border
    assert int(c.status) == 0


def test_gather(cuda):
    c = Cache(cuda, 4, 2, 128, 3, 6)
    c.append([(0, 0, 37), (2, 0, 80)])
    slot, pos = [0, 2, 0, 0, 2, 1, 0, 5, -1, 2], [0, 79, 36, 31, 16, 0, 37, 0, 0, -1]
    for dtype in (torch.float32, torch.bfloat16):
        k, v = ops.kv8_gather(c.a, c.pool, c.rows, c.table, _ints(slot, cuda), _ints(pos, cuda), c.lengths(), dtype=dtype, status=c.status)
        for i in range(10):
            for got, held in zip((k, v), zip(*[s.held() for s in c.seq])):
                if i < 5:
                    want = torch.tensor(held[slot[i]][pos[i]]).float().to(dtype)
                    assert torch.equal(got[i].cpu(), want)
                else:
                    assert not got[i].any()
        assert int(c.status) == 2      # tokens that are not there


def test_blocks_that_are_not_finite(cuda):
    """A key that is infinite or NaN makes its block's keys NaN: rows that see a token of that block are NaN, others know nothing of it."""
    c = Cache(cuda, 4, 2, 64, 1, 10, window=20)
    qkv = torch.randn((100, 512), device=cuda).bfloat16()
    qkv[20, 4 * 64 + 5] = float("inf")       # key of kv head 0, block 1
    qkv[70, 6 * 64 + 64 + 1] = float("nan")  # value of kv head 1, block 4
    c.append([(0, 0, 100)], qkv)
    with np.errstate(invalid="ignore"):
        rows = [(0, n) for n in range(1, 101)]
        q, out = c.attend(rows, want=False)
        assert int(c.status) == 0
        got = _np(out).reshape(100, 4, 64)
        for n in range(1, 101):
            blocks = {p // 16 for p in range(max(0, n - 20), n)}
            assert np.isnan(got[n - 1, :2]).all() == (1 in blocks) and np.isfinite(got[n - 1, :2]).all() == (1 not in blocks), n
            assert np.isnan(got[n - 1, 2:]).all() == (4 in blocks) and np.isfinite(got[n - 1, 2:]).all() == (4 not in blocks), n
    # and behind the last token: rows of the open block that no token has filled hold anything
    c = Cache(cuda, 4, 2, 64, 1, 10)
    c.append([(0, 0, 19)])
    c.rows[0, 1, :, :, 3:] = float("nan")
    c.attend([(0, 19), (0, 17), (0, 18), (0, 16)])


# ---- single tokens ---------------------------------------------------------------------------------------------------------------
LENGTHS = [[1], [16], [17, 15], [0, 40, 1, 33], [700], [129, 640, 32, 31, 64], [5] * 9, [4099]]


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (12, 1, 64), (32, 8, 128), (64, 1, 64)])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_single_tokens(cuda, heads, kv, dim, lengths):
    c = Cache(cuda, heads, kv, dim, len(lengths), max(lengths) // 16 + 2, seed=sum(lengths) + heads)
    c.fill(lengths)
    c.attend([(i, n) for i, n in enumerate(lengths)])


@pytest.mark.parametrize("splits", [1, 2, 3, 8, 40])
@pytest.mark.parametrize("window", [0, 1, 15, 16, 17, 100, 5000])
def test_windows_and_splits(cuda, splits, window):
    lengths = [1, 300, 1024, 1000, 17, 0]
    c = Cache(cuda, 8, 2, 128, 6, 66, window=window, seed=window + splits)
    c.fill(lengths)
    c.attend([(i, n) for i, n in enumerate(lengths)], splits=splits)
    c.attend([(2, 500), (2, 512), (1, 299), (2, 1), (-1, 77), (2, 1024), (3, 0)], splits=splits)    # less than the sequence has; padding; the same slot often


@pytest.mark.parametrize("heads,kv,dim", [(8, 4, 64), (16, 4, 128)])
@pytest.mark.parametrize("splits", [2, 5, 8, None])
def test_many_rows_in_parts(cuda, heads, kv, dim, splits):
    """More parts than places: they meet in scratch, whatever their number; rows of one part, of none and padding among them."""
    lengths = [1, 300, 1024, 1000, 17, 0, 3000]
    c = Cache(cuda, heads, kv, dim, 7, 190, seed=dim)
    c.fill(lengths)
    rows = [(i, n) for i, n in enumerate(lengths)] * 20 + [(-1, 5), (6, 2999), (6, 64), (2, 1), (1, 17)] * 10
    q = torch.tensor(c.rng.normal(0, 1.5, (len(rows), heads, dim)), dtype=torch.float32).bfloat16().to(cuda)
    _, out = c.attend(rows, splits=splits, q=q, want=False)
    assert int(c.status) == 0
    c.check(rows, q, out, every=13)
    assert all((out[i] == 3).all() for i, (s, _) in enumerate(rows) if s < 0)


def test_scales_of_very_different_size(cuda):
    """Blocks whose values differ by many powers of two, blocks of zeros, and scores that pick a block of small values."""
    c = Cache(cuda, 4, 1, 64, 1, 20)
    qkv = torch.randn((200, 6 * 64), device=cuda)
    size = torch.tensor([2.0 ** e for e in (0, -30, 12, -8, 60, 0, -59, 3, -100, 20, 0, 0, -14)], device=cuda).repeat_interleave(16)[:200]
    qkv[:, 5 * 64:] *= size[:, None]
    qkv[80:96, 5 * 64:] = 0                   # block 5: no values
    qkv[160:176, 4 * 64:5 * 64] = 0           # block 10: no keys
    c.append([(0, 0, 200)], qkv.bfloat16())
    for block in (1, 3, 5, 6, 8, 10, 12):     # queries that see little else than one token of that block
        q = torch.zeros((1, 4, 64), device=cuda)
        q[:] = qkv[16 * block + 3, 4 * 64:5 * 64] * 6
        c.attend([(0, 200)], q=q.bfloat16(), splits=1 + block % 3)
    # small and large queries, and none
    q = torch.randn((5, 4, 64), device=cuda) * torch.tensor([1e-30, 1e-3, 0.0, 30.0, 1e-38], device=cuda)[:, None, None]
    c.append([(0, 0, 200)], torch.randn((200, 6 * 64), device=cuda).bfloat16())
    c.attend([(0, 200)] * 5, q=q.bfloat16())


def test_bad_entries_of_the_attention_are_reported(cuda):
    for what in ("page", "none", "slot", "length", "bound"):
        c = Cache(cuda, 4, 2, 64, 2, 6)
        c.fill([90, 60])
        rows, longest = [(0, 90), (1, 60)], 90
        table = c.table.clone()
        if what in ("page", "none"):
            c.table[1, 1] = c.pool.shape[0] if what == "page" else -1
        elif what == "slot":
            rows[1] = (2, 60)
        elif what == "length":
            rows[1] = (1, 61)
        else:
            longest = 89
        q, out = c.attend(rows, want=False, longest=longest)
        assert int(c.status) == 2, what
        c.table = table
        if what != "bound":
            c.check(rows[:1], q[:1], out[:1])


@pytest.mark.parametrize("tiles,splits", [(False, 1), (False, 2), (True, 1), (True, 2)])
def test_tokens_of_a_page_that_is_none_do_not_count(cuda, tiles, splits):
    """A page that is not there is reported, and its tokens are left out of the sums, row by row and in tiles alike."""
    n = 300
    for page in (-1, 1 << 30):
        c = Cache(cuda, 32, 8, 128, 1, 20)
        c.fill([n])
        c.table[0, 3] = page
        rows = [(0, p + 1) for p in range(0 if tiles else 290, n)]
        q, out = c.attend(rows, tiles=[n] if tiles else None, splits=splits, want=False)
        assert int(c.status) == 2
        s, got, qn = c.seq[0], _np(out).reshape(-1, 32, 128), _np(q)
        (k, v), vs = s.held(), s.value_scales()
        for i, (_, end) in enumerate(rows):
            if i % 23 and end < n - 2:
                continue
            at = [t for t in range(end) if t // 16 != 3]
            w, size, unit = kr.attention(qn[i], k[at], v[at], 0, len(at), c.a.scale, vs[at])
            off = np.abs(got[i] - w) - 2 ** -8 * np.abs(w) - (1 + 2 ** -8) * (2 ** -10 * size + 2 ** -25 * unit)
            assert (off <= 0).all(), (end, off.max())


@pytest.mark.parametrize("slot", [2, 1 << 30])
@pytest.mark.parametrize("splits", [None, 2])
def test_tiles_of_no_sequence_are_reported(cuda, slot, splits):
    """A tile whose slot is none: nothing is looked up with it, the other tile's rows are right."""
    c = Cache(cuda, 4, 2, 64, 2, 12)
    c.fill([190, 60])
    rows = [(0, i + 1) for i in range(60, 190)] + [(slot, i + 1) for i in range(20)]
    q, out = c.attend(rows, tiles=[130, 20], splits=splits, want=False)
    assert int(c.status) == 2
    c.check(rows[:130], q[:130], out[:130])


def test_positions_past_32_bits_of_bytes(cuda):
    """Pages whose bytes lie more than 4 GB into the pool, and a page table row far into its table."""
    c = Cache(cuda, 8, 8, 128, 1, 4)
    far = (1 << 32) // c.a.page_bytes + 9
    c.pool = torch.empty((far, 8, c.a.block_bytes), dtype=torch.uint8, device=cuda)
    c.table = _ints([[far - 1, 3, far - 2, far - 5]], cuda)
    c.fill([60])
    c.check_bytes()
    c.attend([(0, 60), (0, 33)])
    c.attend([(0, i + 1) for i in range(60)], tiles=[60])


def test_strided_queries_and_more_rows_than_a_grid_holds(cuda):
    c = Cache(cuda, 2, 1, 64, 1, 2)
    c.fill([20])
    wide = torch.randn((5, 400), device=cuda).bfloat16()
    q = wide[:, 8:136].unflatten(1, (2, 64))
    c.attend([(0, n) for n in (1, 20, 16, 17, 4)], q=q)
    n = 70000
    q = torch.randn((1, 2, 64), device=cuda).bfloat16().expand(n, 2, 64).contiguous()
    _, out = c.attend([(0, 20)] * n, q=q, want=False)
    assert int(c.status) == 0
    c.check([(0, 20)], q[:1], out[:1])
    assert torch.equal(out, out[:1].expand(n, -1))


# ---- prompts ---------------------------------------------------------------------------------------------------------------------
PROMPTS = [[(0, 1)], [(0, 16)], [(0, 129)], [(5, 40), (0, 77)], [(100, 300)], [(0, 257), (33, 1), (0, 15), (500, 130)], [(1000, 64)]]


@pytest.mark.parametrize("heads,kv,dim,window", [(8, 2, 128, 0), (4, 4, 64, 0), (8, 1, 128, 50), (6, 2, 64, 130), (5, 1, 128, 0), (32, 4, 64, 0)])
@pytest.mark.parametrize("prompts", PROMPTS)
def test_prompts(cuda, heads, kv, dim, window, prompts):
    """Every token of a chunk sees the cache as it is behind the append, up to itself."""
    c = Cache(cuda, heads, kv, dim, len(prompts), max(s + n for s, n in prompts) // 16 + 2, window=window, seed=heads + sum(n for _, n in prompts))
    c.fill([s + n for s, n in prompts])
    for splits in (None, 2):   # short ones go row by row unless they are cut
        c.attend([(i, p + 1) for i, (s, n) in enumerate(prompts) for p in range(s, s + n)], tiles=[n for _, n in prompts], splits=splits)


@pytest.mark.parametrize("heads,kv,dim,window", [(32, 8, 128, 0), (12, 12, 64, 0), (24, 8, 128, 300), (20, 4, 64, 0), (16, 8, 64, 129)])
@pytest.mark.parametrize("prompts", [[(0, 1100)], [(700, 333), (5, 800), (0, 64)]])
def test_longer_prompts(cuda, heads, kv, dim, window, prompts):
    c = Cache(cuda, heads, kv, dim, len(prompts), max(s + n for s, n in prompts) // 16 + 2, window=window, seed=heads + sum(n for _, n in prompts))
    c.fill([s + n for s, n in prompts])
    rows = [(i, p + 1) for i, (s, n) in enumerate(prompts) for p in range(s, s + n)]
    q, out = c.attend(rows, tiles=[n for _, n in prompts], splits=1, want=False)
    c.check(rows, q, out, every=41)
    assert int(c.status) == 0


@pytest.mark.parametrize("splits", [1, 2, 9])
@pytest.mark.parametrize("n", [40, 1000])
def test_rows_in_no_tile_and_tiles_that_are_none(cuda, splits, n):
    """Rows that no tile holds stay as they were; a tile outside the rows is reported and the others are right."""
    c = Cache(cuda, 32, 8, 128, 1, 70, seed=n)
    c.fill([n])
    rows = [(0, i + 1) for i in range(n)]
    q = torch.randn((n, 32, 128), device=cuda).bfloat16()
    for extra in ((), ((n - 10, 11),), ((-1, 5),), ((0, 65),), ((3, -1),)):
        first, count = zip(*([(5, 20), (30, 0)] + ([(100, 64), (200, 1), (300, 64)] if n > 40 else []) + list(extra)))
        out = torch.full((n, 32 * 128), 3.0, dtype=torch.bfloat16, device=cuda)
        c.status.zero_()
        ops.kv8_attention(c.a, q, c.pool, c.rows, c.table, _ints([0] * n, cuda), _ints([x for _, x in rows], cuda), c.lengths(), n, tiles=(_ints(first, cuda), _ints(count, cuda)), splits=splits,
                          out=out, status=c.status)
        assert int(c.status) == (2 if extra else 0)
        inside = sorted({r for f, k in zip(first[:2 if n == 40 else 5], count) for r in range(f, f + k)})
        outside = [r for r in range(n) if r not in set(inside)]
        assert (out[outside] == 3).all()
        c.status.zero_()
        at = inside[::7]
        c.check([rows[r] for r in at], q[at], out[at])


def test_no_tiles_at_all(cuda):
    """Rows that no tile holds stay as they were, where there is no tile too."""
    c = Cache(cuda, 8, 2, 128, 1, 4)
    c.fill([40])
    q, out = c.attend([(0, 5), (0, 40)], tiles=[0, 0], want=False)
    assert (out == 3).all() and int(c.status) == 0


@pytest.mark.parametrize("size", [1e3, 3e3, 1e4, 3e4, 1e12, 1e15])
@pytest.mark.parametrize("tiles,splits", [(False, 1), (False, 3), (False, 20), (True, 1), (True, 2)])
def test_scores_of_any_size(cuda, size, tiles, splits):
    """Queries and keys so large that a step of an f32 score is many powers of two of a weight: the largest score has all of the weight."""
    n = 400
    c = Cache(cuda, 32, 8, 128, 1, 26, seed=9)
    qkv = torch.randn((n, 48 * 128), device=cuda)
    qkv[:, 32 * 128:40 * 128] *= size
    c.append([(0, 0, n)], qkv.bfloat16())
    rows = [(0, p + 1) for p in range(n)]
    q = (torch.randn((n, 32, 128), device=cuda) * size).bfloat16()
    _, out = c.attend(rows, tiles=[n] if tiles else None, q=q, splits=splits, want=False)
    assert int(c.status) == 0
    (k, v), qn = c.seq[0].held(), _np(q).astype(np.float64)
    got = _np(out).reshape(n, 32, 128)
    assert np.isfinite(got).all()
    for i in list(range(0, n, 29)) + [n - 1]:
        for h in range(32):
            s = k[:i + 1, h // 4] @ qn[i, h]
            top = np.argsort(s)[::-1]
            if i and s[top[0]] - s[top[1]] < 2 ** -10 * np.abs(s).max():   # (f32 sums of 128 products: 2^-17 of the largest; 2^-10 of 2^20 is far more than 40)
                continue
            want = v[top[0], h // 4]
            assert (np.abs(got[i, h] - want) <= 2 ** -7 * np.abs(want)).all(), (i, h)     # bf16, and as much for the weight in front and behind


def test_scores_that_grow_along_the_keys(cuda):
    """The reference of the weights has to follow: every block's scores are far above the one before, and then far below."""
    c = Cache(cuda, 32, 8, 128, 1, 72, seed=3)
    n = 1100
    qkv = torch.randn((n, 48 * 128), device=cuda)
    ramp = torch.cat([torch.linspace(0, 30, n // 2), torch.linspace(30, -30, n - n // 2)]).to(cuda)
    qkv[:, 32 * 128:40 * 128] = ramp[:, None]
    c.append([(0, 0, n)], qkv.bfloat16())
    q = (torch.rand((n, 32, 128), device=cuda) * 0.3).bfloat16()
    rows = [(0, i + 1) for i in range(n)]
    _, out = c.attend(rows, tiles=[n], q=q, splits=1, want=False)
    c.check(rows, q, out, every=23)
    for splits in (2, 3):
        _, out = c.attend(rows, tiles=[n], q=q, splits=splits, want=False)
        c.check(rows, q, out, every=61)
    _, out = c.attend(rows[-40:], q=q[-40:].contiguous(), want=False)
    c.check(rows[-40:], q[-40:], out)
    assert int(c.status) == 0


@pytest.mark.parametrize("tiles", [False, True])
def test_waits_that_run_out_end_the_kernel(cuda, tiles):
    """Keys that are never asked for: every wait ends, the status says so, and the next call is right."""
    from gptrs_b200 import lib
    c = Cache(cuda, 32, 8, 128, 1, 72, seed=5)
    c.fill([1100])
    rows = [(0, i + 1) for i in range(1100)] if tiles else [(0, 1100), (0, 300)]
    try:
        assert lib().gptrs_cuda_debug_prefill_tc_fault(1, 64) == 0
        q, _ = c.attend(rows, tiles=[1100] if tiles else None, splits=1, want=False)
        torch.cuda.synchronize()
    finally:
        lib().gptrs_cuda_debug_prefill_tc_fault(0, 0)
    assert int(c.status) == 3
    c.status.zero_()
    q, out = c.attend(rows, tiles=[1100] if tiles else None, splits=1, want=False, q=q)
    c.check(rows, q, out, every=97)
    assert int(c.status) == 0


@pytest.mark.parametrize("splits", [1, 2, 5])
def test_prompt_in_parts(cuda, splits):
    c = Cache(cuda, 8, 2, 128, 2, 80, seed=splits)
    c.fill([1200, 700])
    c.attend([(0, p + 1) for p in range(1100, 1200)] + [(1, p + 1) for p in range(640, 700)], tiles=[100, 60], splits=splits)


@pytest.mark.parametrize("rows,splits", [(1100, 1), (20, 2)])
def test_pages_that_arrive_at_different_times(cuda, rows, splits):
    """Pages of one of the warps that widen them are in L2, the others' are not: that warp is ahead of the others and of the products, whose operands stay
    as they are until they have been read. The bits are those of a run whose pages are all there. 20 rows: a row tile without a row."""
    c = Cache(cuda, 32, 8, 128, 1, 72, seed=rows)
    c.fill([1100])
    seen = [(0, p + 1) for p in range(1100 - rows, 1100)]
    q, out = c.attend(seen, tiles=[rows], splits=splits, want=False)
    c.check(seen, q, out, every=67)
    slot, ctx = _ints([0] * rows, cuda), _ints([n for _, n in seen], cuda)
    step = ops.Kv8Attention(c.a, q, c.pool, c.rows, c.table, slot, ctx, c.lengths(), 1100, tiles=ops.kv8_tiles(c.a, [rows], cuda), splits=splits, status=c.status)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=cuda)
    for turn in range(12):
        flush.fill_(turn)
        warm = c.table[0, [b for b in range(68) if b % 8 // 2 == turn % 4]].long()
        c.pool[warm].sum()
        torch.cuda.synchronize()
        assert torch.equal(step(), out), turn
    assert int(c.status) == 0


@pytest.mark.parametrize("tiles,splits", [(False, 1), (False, 3), (True, 1), (True, 2)])
@pytest.mark.parametrize("window", [0, 5])
def test_open_block_that_is_not_finite(cuda, window, tiles, splits):
    """A key or value that is not finite in the block that is not complete: rows that see its token are NaN there, others know nothing of it, row by row and in
    tiles alike."""
    n = 300
    c = Cache(cuda, 32, 8, 128, 1, 20, window=window)
    qkv = torch.randn((n, 48 * 128), device=cuda).bfloat16()
    bad = {290: (40 + 3, "nan"), 294: (32 + 5, "inf"), 296: (40 + 6, "-inf")}     # token: head of the row (32 keys, 40 values)
    for token, (head, x) in bad.items():
        qkv[token, head * 128 + 7] = float(x)
    c.append([(0, 0, n)], qkv)
    rows = [(0, p + 1) for p in range(0 if tiles else 280, n)]
    q, out = c.attend(rows, tiles=[n] if tiles else None, splits=splits, want=False)
    assert int(c.status) == 0
    s, got = c.seq[0], _np(out).reshape(-1, 32, 128)
    s.k, s.v = (np.where(np.isfinite(x), x, np.float32(0)) for x in (s.k, s.v))
    (k, v), vs, qn = s.held(), s.value_scales(), _np(q)
    for i, (_, end) in enumerate(rows):
        if end < 280 and end % 37:
            continue
        begin = max(0, end - window) if window else 0
        w, size, unit = kr.attention(qn[i], k, v, begin, end, c.a.scale, vs)
        sees = np.isin(np.arange(32) // 4, [(head - 32) % 8 for token, (head, _) in bad.items() if begin <= token < end])
        assert np.isnan(got[i, sees]).all(), end
        off = np.abs(got[i] - w) - 2 ** -8 * np.abs(w) - (1 + 2 ** -8) * (2 ** -10 * size + 2 ** -25 * unit)
        assert (off[~sees] <= 0).all(), end


@pytest.mark.parametrize("tiles", [False, True])
def test_a_long_tail_beside_one_token(cuda, tiles):
    """One token with nearly all of the weight in front of 131071 with 2^-24.9 or 2^-25.2 of it each: together they are 0.3 to 0.4 % of the sum and all of the output.
    Their weights are f16, off by 2^-25 at most, with 2^15 for the largest of a row, 2^2 or more in tiles."""
    n = 1 << 17
    c = Cache(cuda, 2, 1, 64, 1, n // 16)
    qkv = torch.zeros((n, 4 * 64), device=cuda)
    qkv[0, 2 * 64] = 16
    qkv[1:, 3 * 64:] = 1
    c.append([(0, 0, n)], qkv.bfloat16())
    rows = [(0, p + 1) for p in range(n - (1000 if tiles else 3), n)]
    q = torch.zeros((len(rows), 2, 64), device=cuda)
    q[:, 0, 0], q[:, 1, 0] = 8.625, 8.75
    q, out = c.attend(rows, tiles=[len(rows)] if tiles else None, splits=1, q=q.bfloat16(), want=False)
    assert int(c.status) == 0
    (k, v), vs, qn, got = c.seq[0].held(), c.seq[0].value_scales(), _np(q), _np(out).reshape(-1, 2, 64)
    for i in [0, len(rows) // 2, len(rows) - 1]:
        w, size, unit = kr.attention(qn[i], k, v, 0, rows[i][1], c.a.scale, vs)
        assert (np.abs(got[i] - w) <= 2 ** -8 * w + (1 + 2 ** -8) * (2 ** -10 * size + 2 ** (-25 - (2 if tiles else 15)) * unit)).all(), (got[i, :, 0], w[:, 0])


def test_calls_without_rows(cuda):
    """No rows: nothing to do, whatever the tensors' addresses."""
    c = Cache(cuda, 8, 2, 128, 2, 4)
    c.fill([20, 7])
    none, empty = _ints([], cuda), torch.empty((0, 12 * 128), dtype=torch.bfloat16, device=cuda)
    rot = ops.QkRotation(8, 2, 128)
    assert ops.qk_norm_rope(rot, empty, none).shape == (0, 12 * 128)
    before = c.pool.clone()
    assert ops.kv8_append(c.a, rot, empty, none, none, none, none, c.table, c.pool, c.rows, status=c.status).shape == (0, 8, 128)
    for tiles in (None, ops.kv8_tiles(c.a, [], cuda)):
        assert ops.kv8_attention(c.a, empty.reshape(0, 12, 128)[:, :8], c.pool, c.rows, c.table, none, none, c.lengths(), 100, tiles=tiles, status=c.status).shape == (0, 8 * 128)
    k, v = ops.kv8_gather(c.a, c.pool, c.rows, c.table, none, none, c.lengths(), status=c.status)
    assert k.shape == v.shape == (0, 2, 128) and torch.equal(c.pool, before) and int(c.status) == 0


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("splits", [1, 2, 20])
def test_output_over_the_queries(cuda, tiles, splits):
    """The output in the place of packed queries: the same bits."""
    c = Cache(cuda, 20, 2, 128, 1, 40, seed=splits)
    c.fill([600])
    rows = [(0, p + 1) for p in range(0 if tiles else 560, 600)]
    q, out = c.attend(rows, tiles=[600] if tiles else None, splits=splits, want=False)
    c.check(rows, q, out, every=41)
    same = q.clone()
    ops.kv8_attention(c.a, same, c.pool, c.rows, c.table, _ints([0] * len(rows), cuda), _ints([n for _, n in rows], cuda), c.lengths(), 600,
                      tiles=ops.kv8_tiles(c.a, [600], cuda) if tiles else None, splits=splits, out=same.view(len(rows), -1), status=c.status)
    assert torch.equal(same.view(len(rows), -1), out) and int(c.status) == 0


# ---- together ----------------------------------------------------------------------------------------------------------------------
def test_prompt_then_steps_in_a_graph(cuda):
    """A prompt, then tokens one by one as a server has them: append and attention recorded once, replayed with new rows, positions and lengths."""
    c = Cache(cuda, 8, 2, 128, 3, 8, seed=11)
    starts = [0, 30, 46]
    runs = [(i, 0, s) for i, s in enumerate(starts) if s]
    c.append(runs)
    c.attend([(i, p + 1) for i, _, n in runs for p in range(n)], tiles=[n for _, _, n in runs])
    width = 12 * 128
    qkv, pos, ctx = torch.zeros((3, width), dtype=torch.bfloat16, device=cuda), _ints(starts, cuda), _ints([s + 1 for s in starts], cuda)
    slot, each = _ints([0, 1, 2], cuda), _ints([0, 1, 2], cuda)
    out = torch.zeros((3, 8 * 128), dtype=torch.bfloat16, device=cuda)
    append = ops.Kv8Append(c.a, None, qkv, pos, slot, each, each, c.table, c.pool, c.rows, status=c.status)
    attend = ops.Kv8Attention(c.a, append.q, c.pool, c.rows, c.table, slot, ctx, ctx, 100, out=out, status=c.status, splits=3)
    snapshot = c.pool.clone(), c.rows.clone()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        append()
        attend()
    assert torch.equal(c.pool, snapshot[0])
    for step in range(40):
        x = torch.randn((3, width), device=cuda).bfloat16()
        qkv.copy_(x)
        graph.replay()
        for i in range(3):
            r = _np(x[i]).reshape(12, 128)
            at = starts[i] + step
            c.seq[i].append(at, r[None, 8:10], r[None, 10:])
            c.halves[i][at // 16 % 2] = at // 16
        c.check([(i, s + step + 1) for i, s in enumerate(starts)], x[:, :1024].reshape(3, 8, 128), out)
        pos += 1
        ctx += 1
    c.check_bytes()
    assert int(c.status) == 0


def test_other_streams_and_two_calls_at_once(cuda):
    """Calls of two caches on two streams do not touch each other, and the same call twice gives the same bits."""
    caches = [Cache(cuda, 8, 2, 128, 4, 40, seed=s) for s in (1, 2)]
    steps, refs = [], []
    for c in caches:
        c.fill([600, 33, 128, 1])
        rows = [(i, n) for i, n in enumerate([600, 33, 128, 1])]
        q, out = c.attend(rows, splits=5)
        refs.append(out.clone())
        steps.append(ops.Kv8Attention(c.a, q, c.pool, c.rows, c.table, _ints(range(4), cuda), c.lengths(), c.lengths(), 600, splits=5, status=c.status))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    outs = [[], []]
    for _ in range(20):
        for i, (stream, step) in enumerate(zip(streams, steps)):
            with torch.cuda.stream(stream):
                outs[i].append(step().clone())
    torch.cuda.synchronize()
    for ref, got in zip(refs, outs):
        assert all(torch.equal(ref, g) for g in got)


@pytest.mark.parametrize("what", ["attention", "append", "gather", "rope"])
def test_an_object_that_goes_away_while_its_call_runs_elsewhere(cuda, what):
    """Memory of an object that was called on another stream is not given out again before that call has ended."""
    c = Cache(cuda, 8, 2, 128, 2, 130, seed=5)
    c.fill([2000, 1900])
    slot, ctx = _ints([0, 1], cuda), _ints([2000, 1900], cuda)
    rows = torch.zeros((2, 12 * 128), dtype=torch.bfloat16, device=cuda)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=cuda)
    make = {"attention": lambda: ops.Kv8Attention(c.a, q, c.pool, c.rows, c.table, slot, ctx, ctx, 2000, splits=200),
            "append": lambda: ops.Kv8Append(c.a, None, rows, ctx, slot, _ints([0, 1], cuda), _ints([0, 1], cuda), c.table, c.pool, c.rows),
            "gather": lambda: ops.Kv8Gather(c.a, c.pool, c.rows, c.table, slot, slot, ctx), "rope": lambda: ops.QkNormRope(ops.QkRotation(8, 2, 128), rows, None)}[what]
    make()()                                     # (kernels are loaded)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    step = make()
    owned = {t.data_ptr(): t.untyped_storage().nbytes() for n, t in step._tensors.items() if n in ("scratch", "out", "q", "k", "v", "status") and t is not q}
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(400_000_000)           # a fifth of a second, and then the call
        step()
        step()
    del step
    new = [torch.empty(size, dtype=torch.uint8, device=cuda) for size in list(owned.values()) * 400]
    assert not stream.query()
    assert not {t.data_ptr() for t in new} & set(owned)
    torch.cuda.synchronize()


@pytest.mark.parametrize("tiles", [None, [70, 60]])
def test_two_graphs_of_one_cache_at_once(cuda, tiles):
    """Two objects over one cache whose parts meet in scratch, captured each and replayed side by side: either has scratch of its own."""
    c = Cache(cuda, 8, 2, 128, 2, 130, seed=5)
    c.fill([2000, 1900])
    rows = [(0, 2000), (1, 1900)] if tiles is None else [(0, i + 1) for i in range(1930, 2000)] + [(1, i + 1) for i in range(1840, 1900)]
    slot, ctx, lengths = _ints([s for s, _ in rows], cuda), _ints([n for _, n in rows], cuda), c.lengths()
    tiled = None if tiles is None else ops.kv8_tiles(c.a, tiles, cuda)
    qs = [torch.randn((len(rows), 8, 128), device=cuda).bfloat16() for _ in range(2)]
    steps = [ops.Kv8Attention(c.a, q, c.pool, c.rows, c.table, slot, ctx, lengths, 2000, tiles=tiled, splits=12, status=c.status) for q in qs]
    streams, graphs = [torch.cuda.Stream() for _ in qs], [torch.cuda.CUDAGraph() for _ in qs]
    for step, stream in zip(steps, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
    torch.cuda.synchronize()
    wants = [step.out.clone() for step in steps]
    for step, q, want in zip(steps, qs, wants):
        c.check(rows, q, want, every=17)
    for step, stream, graph in zip(steps, streams, graphs):
        with torch.cuda.graph(graph, stream=stream):
            step()
    for _ in range(30):
        for step in steps:
            step.out.zero_()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(step.out, want) for step, want in zip(steps, wants))
    assert int(c.status) == 0
