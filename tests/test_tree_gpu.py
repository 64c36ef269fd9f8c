"""Trees of drafted tokens over the paged bf16 cache (append, attention, acceptance) against the oracle in 64 bits.

Tolerances. Attention: the output is rounded to bf16 once, off by at most 2^-8 of the value; the weights are rounded to bf16 in front of the products with the
values, off by at most 2^-8 of themselves, which moves the output by at most 2^-8 sum p |v|; the denominator is summed in front of that rounding. Scores are f32
sums of 128 products and an exponential: 2^-16 of sum p |v| covers an error of 2^-17 in every exponent (scores up to 2^6 in f32) and those of the f32 sums. So
2^-8 |want| + (1 + 2^-8) (2^-8 + 2^-16) sum p |v|. Append: one rounding (2^-8 of the value), and f32 products and a sum of two terms, 2^-22 of the pair's size."""
import numpy as np
import pytest
import torch

import gptrs_b200
from gptrs_b200 import ops
from oracle import tree_ref as tr

pytestmark = pytest.mark.gpu

PAGE, DIM = 16, 128


def _np(t):
    return t.float().cpu().numpy()


def _ints(v, cuda):
    return torch.tensor(np.asarray(v, dtype=np.int64), dtype=torch.int32, device=cuda)


def chain(n):
    return list(range(-1, n - 1))


def bushy(n, rng, reach=6):
    return [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, n)]


class Trees:
    """Trees over a cache on the GPU, beside dense keys and values. Whatever no tree has appended is NaN in the pool. forest: (length, parents) of every tree, None: padding."""

    def __init__(self, cuda, heads, kv, forest, seed=0, scale=0.0, max_nodes=None, extra_rows=0, fill=True, spare=2):
        self.rng = rng = np.random.default_rng(seed)
        self.cuda, self.heads, self.kv, self.forest, self.scale = cuda, heads, kv, forest, scale
        n = len(forest)
        need = [0 if f is None else (f[0] + len(f[1]) + PAGE - 1) // PAGE for f in forest]
        self.pages = max(1, sum(need)) + spare
        self.slots = rng.permutation(n + 1)[:n]
        perm, at = rng.permutation(self.pages), 0
        table = np.full((n + 1, max(need + [1])), -7)
        for s, k in enumerate(need):
            table[self.slots[s], :k] = perm[at:at + k]
            at += k
        self.table = _ints(table, cuda)
        first = np.cumsum([0] + [0 if f is None else len(f[1]) for f in forest])
        self.first, self.rows = _ints(first, cuda), int(first[-1]) + extra_rows
        self.row0 = first
        self.slot = _ints([-1 if f is None else self.slots[s] for s, f in enumerate(forest)], cuda)
        self.length = _ints([0 if f is None else f[0] for f in forest], cuda)
        self.parent = _ints(sum([[] if f is None else list(f[1]) for f in forest], []) + [99] * extra_rows, cuda)
        self.max_nodes = max_nodes or max([1] + [len(f[1]) for f in forest if f is not None])
        self.pool = torch.full((ops.kv_pool_bytes(self.pages, kv),), 255, dtype=torch.uint8, device=cuda)
        self.status = torch.zeros(1, dtype=torch.int32, device=cuda)
        self.trees = ops.DraftTrees(heads, kv, self.first, self.slot, self.length, self.parent, self.table, self.max_nodes, scale)
        self.kvs = [None if f is None else rng.normal(0, 1, (2, f[0] + len(f[1]), kv, DIM)) for f in forest]
        if fill:
            for s, x in enumerate(self.kvs):
                if x is not None:
                    self.kvs[s] = self.write(s, np.arange(x.shape[1]), torch.tensor(x, dtype=torch.float32).bfloat16())

    def view(self, pool=None):
        return (self.pool if pool is None else pool).view(torch.bfloat16).view(self.pages, self.kv, 2, PAGE, 16, 8)

    def place(self, s, positions):
        p = torch.as_tensor(np.asarray(positions), device=self.cuda)
        page, tok = self.table[int(self.slots[s])].long()[p // PAGE], p % PAGE
        return page[:, None], tok[:, None], torch.arange(16, device=self.cuda) ^ (tok[:, None] % 8)

    def write(self, s, positions, x, pool=None):
        """x bf16 [2][positions][kv][dim]; returns it as numpy."""
        page, tok, chunk = self.place(s, positions)
        self.view(pool)[page, :, :, tok, chunk] = x.to(self.cuda).view(2, -1, self.kv, 16, 8).permute(1, 3, 2, 0, 4)
        return _np(x)

    def read(self, s, positions, pool=None):
        page, tok, chunk = self.place(s, positions)
        return _np(self.view(pool)[page, :, :, tok, chunk].permute(3, 0, 2, 1, 4).reshape(2, -1, self.kv, DIM))

    def queries(self, size=1.0):
        return torch.tensor(self.rng.normal(0, size, (self.rows, self.heads, DIM)), dtype=torch.float32).bfloat16().to(self.cuda)

    def attention(self, q, **kw):
        return ops.tree_attention(self.trees, q, self.pool, status=self.status, **kw)

    def check(self, got, q, lost=None):
        got, q = _np(got).reshape(self.rows, self.heads, DIM), _np(q)
        for s, f in enumerate(self.forest):
            if f is None:
                continue
            a, b = self.row0[s], self.row0[s + 1]
            want, mass = tr.attention(q[a:b], *self.kvs[s], f[1], f[0], self.scale or DIM ** -0.5, (lost or {}).get(s, ()))
            off = np.abs(got[a:b] - want) - (2 ** -8 * np.abs(want) + (1 + 2 ** -8) * (2 ** -8 + 2 ** -16) * mass)
            assert (off <= 0).all(), (s, f[0], len(f[1]), float(off.max()))


# ---- attention -----------------------------------------------------------------------------------------------------------------
LAYOUTS = [(32, 8), (8, 1), (12, 12), (6, 2), (5, 1), (14, 2), (1, 1), (24, 2), (32, 1)]


@pytest.mark.parametrize("heads,kv", LAYOUTS)
def test_attention_head_layouts(cuda, heads, kv):
    rng = np.random.default_rng(heads * 50 + kv)
    t = Trees(cuda, heads, kv, [(75, bushy(26, rng)), (0, chain(3)), (130, bushy(9, rng)), (1, [-1])], seed=heads)
    q = t.queries()
    t.check(t.attention(q), q)
    assert int(t.status) == 0


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 48, 63, 64, 65, 100, 127, 128, 129, 191, 500, 1023, 2500])
@pytest.mark.parametrize("nodes", [1, 2, 16, 33, 64])
def test_attention_lengths(cuda, length, nodes):
    rng = np.random.default_rng(length * 100 + nodes)
    t = Trees(cuda, 8, 2, [(length, bushy(nodes, rng))], seed=length + nodes)
    q = t.queries(1.5)
    t.check(t.attention(q), q)
    assert int(t.status) == 0


@pytest.mark.parametrize("heads,kv,nodes,length", [(4, 4, 256, 70), (8, 1, 256, 33), (16, 2, 250, 700), (32, 1, 255, 5), (12, 4, 100, 257), (2, 1, 129, 0), (5, 1, 77, 300), (32, 8, 200, 1000)])
def test_attention_large_trees(cuda, heads, kv, nodes, length):
    rng = np.random.default_rng(nodes)
    t = Trees(cuda, heads, kv, [(length, bushy(nodes, rng, 40)), (length // 2, chain(nodes // 3 + 1))], seed=nodes)
    q = t.queries()
    t.check(t.attention(q), q)


@pytest.mark.parametrize("shape", ["chain", "star", "forest", "comb"])
def test_attention_shapes(cuda, shape):
    n = 70
    parents = {"chain": chain(n), "star": [-1] + [0] * (n - 1), "forest": [-1] * n, "comb": [-1] + [(i - 1) // 2 * 2 for i in range(1, n)]}[shape]
    t = Trees(cuda, 8, 2, [(37, parents), (200, parents[:33])], seed=7)
    q = t.queries()
    t.check(t.attention(q), q)


def test_attention_many_trees_and_long_ones(cuda):
    rng = np.random.default_rng(5)
    forest = [(int(rng.integers(0, 900)), bushy(int(rng.integers(1, 40)), rng)) for _ in range(70)] + [(20011, bushy(17, rng)), (9000, [-1])]
    t = Trees(cuda, 8, 2, forest, seed=11)
    q = t.queries()
    t.check(t.attention(q), q)


def test_attention_padding_rows_behind_and_strides(cuda):
    rng = np.random.default_rng(6)
    t = Trees(cuda, 8, 2, [None, (40, bushy(9, rng)), None, (3, []), (150, bushy(30, rng)), None], seed=3, extra_rows=4, max_nodes=47)
    wide = torch.full((t.rows, 8 + 3, DIM), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 1:9] = t.queries()
    out = torch.full((t.rows, 8 * DIM), 5.0, dtype=torch.bfloat16, device=cuda)
    got = t.attention(wide[:, 1:9], out=out)
    assert got is out
    t.check(got, wide[:, 1:9])
    assert (out[39:] == 5).all() and int(t.status) == 0


def test_attention_scale_and_peaked_scores(cuda):
    rng = np.random.default_rng(8)
    t = Trees(cuda, 4, 1, [(333, bushy(40, rng))], seed=9, scale=0.9)   # scores of +- 30: one token takes most of a row
    q = t.queries(3.0)
    t.check(t.attention(q), q)


def test_attention_what_a_node_does_not_see_does_not_touch_it(cuda):
    rng = np.random.default_rng(10)
    parents = [-1, 0, 0, 1, 2, 4, 1, 3]
    for bad in (float("nan"), float("inf"), -float("inf")):
        for which in (0, 1):
            t = Trees(cuda, 8, 2, [(90, parents), (21, parents)], seed=1)
            q = t.queries()
            want = t.attention(q).clone()
            for s, (length, _) in enumerate(t.forest):
                page, tok, chunk = t.place(s, [length + 2])
                t.view()[page, 1, which, tok, chunk, 3] = bad           # node 2, kv head 1, channels 3, 11, ...
            got = t.attention(q)
            sees = np.array([2 in a for a in tr.ancestors(parents)] * 2)
            same = (got == want).view(t.rows, 8, DIM).cpu().numpy()
            assert same[~sees].all() and same[sees][:, :4].all(), (bad, which)
            seen = _np(got).reshape(t.rows, 8, DIM)[sees][:, 4:]
            if which:   # its own channels say so, the others stay
                near = np.abs(seen - _np(want).reshape(t.rows, 8, DIM)[sees][:, 4:])
                at = np.arange(DIM) % 8 == 3
                assert (np.isnan(seen[..., at]).all() if bad != bad else (seen[..., at] == bad).all()) and np.isfinite(near[..., ~at]).all()


def test_attention_huge_scores(cuda):
    rng = np.random.default_rng(16)
    t = Trees(cuda, 2, 1, [(20, chain(4)), (150, bushy(30, rng))], seed=2)
    q = t.queries()
    for s, at in ((0, 5), (1, 3), (1, 151)):                            # a key of -1e36: its scores are +- 1e36, it takes all of a row or nothing
        t.write(s, [at], torch.tensor(np.stack([np.full((1, 1, DIM), -1e36), t.kvs[s][1, at:at + 1]])).bfloat16())
        t.kvs[s] = t.read(s, np.arange(t.kvs[s].shape[1]))
    t.check(t.attention(q), q)


def test_attention_pages_out_of_range(cuda):
    rng = np.random.default_rng(12)
    t = Trees(cuda, 8, 2, [(100, bushy(20, rng)), (40, bushy(5, rng))], seed=4)
    lost = {0: [], 1: []}
    for s, page, value in ((0, 2, -1), (0, 5, t.pages), (1, 1, 1 << 30)):
        t.table[int(t.slots[s]), page] = value
        lost[s] += list(range(16 * page, 16 * page + 16))
    q = t.queries()
    got = t.attention(q)
    assert int(t.status) == 2
    t.check(got, q, lost)


def test_attention_nothing_to_see_gives_zeros(cuda):
    t = Trees(cuda, 4, 2, [(0, chain(3)), (17, chain(2))], seed=4)
    t.table[int(t.slots[0]), 0] = -1
    q = t.queries()
    got = t.attention(q)
    assert int(t.status) == 2 and (got[:3] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("what", ["slot", "length", "negative length", "nodes", "first", "rows"])
def test_trees_out_of_range_count_as_padding(cuda, what):
    rng = np.random.default_rng(13)
    t = Trees(cuda, 4, 2, [(30, bushy(6, rng)), (50, bushy(8, rng)), (5, bushy(4, rng))], seed=5, max_nodes=7 if what == "nodes" else 8)
    q = t.queries()
    out = torch.full((t.rows, 4 * DIM), 5.0, dtype=torch.bfloat16, device=cuda)
    if what == "slot":
        t.slot[1] = 4
    if what == "length":
        t.length[1] = 16 * t.table.shape[1] - 7
    if what == "negative length":
        t.length[1] = -1
    if what == "first":
        t.first[1], t.first[2] = 14, 6
    if what == "rows":
        t.first[3] = t.rows + 1
    got = t.attention(q, out=out)
    assert int(t.status) == 2
    if what == "first":
        return                                                          # (its neighbours' rows are out of order too)
    left = slice(14, 18) if what == "rows" else slice(6, 14)
    assert (got[left] == 5).all()
    t.forest[2 if what == "rows" else 1] = None
    t.check(got, q)


def test_parents_out_of_range_count_as_none(cuda):
    t = Trees(cuda, 4, 2, [(30, [-1, 0, 1, 1, 2])], seed=6)
    t.parent[2], t.parent[4] = 2, -5
    q = t.queries()
    got = t.attention(q)
    t.forest[0] = (30, [-1, 0, -1, 1, -1])
    t.check(got, q)
    assert int(t.status) == 2


def test_attention_twice_and_on_another_stream(cuda):
    rng = np.random.default_rng(14)
    t = Trees(cuda, 32, 8, [(int(rng.integers(0, 3000)), bushy(int(rng.integers(1, 60)), rng)) for _ in range(9)], seed=7)
    q = t.queries()
    call = ops.TreeAttention(t.trees, q, t.pool, status=t.status)
    want = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert call().equal(want)
        assert call().equal(want)
    torch.cuda.current_stream().wait_stream(side)


def test_attention_two_graphs_at_once_with_new_trees(cuda):
    rng = np.random.default_rng(15)
    t = Trees(cuda, 8, 2, [(700, bushy(30, rng)), (90, bushy(12, rng)), (0, bushy(3, rng))], seed=8)
    calls = [(q, ops.TreeAttention(t.trees, q, t.pool, status=t.status)) for q in (t.queries(), t.queries())]
    for _, call in calls:
        call()
    torch.cuda.synchronize()
    graphs = []
    for _, call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    for step in range(3):
        for g, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for q, call in calls:
            t.check(call.out, q)
        t.length[0] = 650 - 13 * step                                   # the next step's trees in the same tensors
        t.kvs[0] = t.read(0, np.arange(650 - 13 * step + 30))
        t.forest[0] = (650 - 13 * step, t.forest[0][1])
        if step == 1:
            t.slot[1], t.forest[1] = -1, None


def test_attention_behind_four_gigabytes(cuda):
    """Pages whose bytes lie behind 2^32."""
    t = Trees(cuda, 8, 8, [(60, bushy(20, np.random.default_rng(1)))], seed=9, spare=70000)
    far = torch.arange(5, dtype=torch.int32, device=cuda) + (t.pages - 5)
    old = t.view()[t.table[int(t.slots[0]), :5].long()].clone()
    t.table[int(t.slots[0]), :5] = far
    t.view()[far.long()] = old
    q = t.queries()
    t.check(t.attention(q), q)


# How a call is cut goes by the table's width, the trees, heads and rows: clusters of 8, 4, 2 and 1 CTAs, more of them than are on the GPU at a time, equal shares with parts
# joined by warps (at several levels), and by the second kernel; each with one row tile and with several.
CUTS = [  # heads, kv, trees, nodes, lengths
    (4, 2, 3, 20, (1, 1400)), (4, 1, 1, 33, (5000, 5000)), (8, 8, 4, 40, (10, 700)), (8, 8, 9, 17, (0, 900)), (12, 12, 13, 9, (0, 700)), (12, 12, 40, 5, (0, 300)),
    (4, 1, 2, 256, (20, 1000)), (32, 4, 3, 100, (0, 400)),
    (4, 2, 2, 20, (9000, 21000)), (2, 1, 1, 3, (30000, 30000)), (8, 1, 1, 100, (20000, 20000)), (8, 8, 30, 6, (1500, 3000)), (4, 4, 60, 11, (100, 6000)), (16, 2, 20, 60, (300, 5000))]


@pytest.mark.parametrize("heads,kv,trees,nodes,lengths", CUTS)
def test_attention_however_it_is_cut(cuda, heads, kv, trees, nodes, lengths):
    rng = np.random.default_rng(trees * nodes)
    low, high = lengths
    forest = [(high if i == 0 else int(rng.integers(low, high + 1)), bushy(nodes if i == 0 else int(rng.integers(1, nodes + 1)), rng, 12)) for i in range(trees)]
    t = Trees(cuda, heads, kv, forest, seed=nodes)
    q = t.queries(1.3)
    call = ops.TreeAttention(t.trees, q, t.pool, status=t.status)
    got = call().clone()
    t.check(got, q)
    assert int(t.status) == 0
    for _ in range(3):
        assert call().equal(got)                                        # whoever was last
    if call.scratch is not None:
        other = ops.TreeAttention(t.trees, q, t.pool, status=t.status, scratch_of=call)
        assert other().equal(got)


# (length of the first tree, of the others): clusters of eight (a node alone in its part, and many blocks to a part), several tiles, whole items, joins by warps at one level and at several,
# with one tile and two, the second kernel.
MINUS_INFINITY = [(4, 2, 1, 1, (64, 0)), (4, 2, 1, 1, (63, 0)), (4, 2, 3, 20, (1400, 1300)), (4, 1, 2, 256, (1000, 900)), (8, 8, 30, 6, (3000, 2900)), (4, 4, 60, 11, (9000, 300)),
                  (2, 1, 80, 3, (20000, 300)), (16, 2, 20, 60, (5000, 300)), (2, 1, 1, 3, (30000, 0))]


@pytest.mark.parametrize("finite", ["context", "first", "middle", "root", "none"])
@pytest.mark.parametrize("heads,kv,trees,nodes,lengths", MINUS_INFINITY)
def test_attention_parts_whose_scores_are_all_minus_infinity(cuda, heads, kv, trees, nodes, lengths, finite):
    """Keys that make scores of -inf have weight 0 beside finite ones, whichever of a call's parts they are in; where a row sees no others it is NaN."""
    rng = np.random.default_rng(nodes)
    t = Trees(cuda, heads, kv, [(lengths[min(s, 1)], bushy(nodes, rng)) for s in range(trees)], seed=lengths[0])
    q = t.queries()
    q[..., 3] = q[..., 3].abs() + 0.5
    for s, (n, _) in enumerate(t.forest):
        keep = {"context": slice(0, n), "first": 0, "middle": n // 2, "root": n, "none": slice(0, 0)}[finite]
        keys = t.kvs[s][0].copy()
        t.kvs[s][0, ..., 3] = -np.inf
        t.kvs[s][0, keep] = keys[keep]
        t.write(s, np.arange(t.kvs[s].shape[1]), torch.tensor(t.kvs[s], dtype=torch.float32).bfloat16())
    got = t.attention(q)
    if finite == "none":
        assert got.isnan().all()
    else:
        t.check(got, q)


@pytest.mark.parametrize("at", ["first", "root"])
@pytest.mark.parametrize("heads,kv,trees,nodes,lengths", MINUS_INFINITY)
def test_attention_a_score_that_is_nan_reaches_its_rows_from_any_part(cuda, heads, kv, trees, nodes, lengths, at):
    """Beside scores of -inf in its part, and finite ones in others."""
    rng = np.random.default_rng(nodes)
    t = Trees(cuda, heads, kv, [(lengths[min(s, 1)], bushy(nodes, rng)) for s in range(trees)], seed=lengths[0])
    q = t.queries()
    q[..., 3] = q[..., 3].abs() + 0.5
    for s, (n, _) in enumerate(t.forest):
        bad = 0 if at == "first" else n
        t.kvs[s][0, max(0, bad - 70):bad + 70, ..., 3] = -np.inf
        t.kvs[s][0, bad, 0, 3] = np.nan                                    # kv head 0
        t.write(s, np.arange(t.kvs[s].shape[1]), torch.tensor(t.kvs[s], dtype=torch.float32).bfloat16())
    got = t.attention(q).view(t.rows, kv, -1)
    assert got[:, 0].isnan().all()
    if kv > 1 and lengths[1] > 200:
        assert torch.isfinite(got[:, 1:]).all()


@pytest.mark.parametrize("heads,kv,forest", [(8, 2, [(20, 9), (3, 2), (0, 40)]), (32, 8, [(900, 26)]), (8, 8, [(300, 7)] * 30), (4, 1, [(500, 200)] * 2), (2, 1, [(20000, 3)] + [(300, 3)] * 79),
                                             (2, 1, [(30000, 3)])])
def test_attention_loses_no_more_than_the_rounding_of_its_results(cuda, heads, kv, forest):
    """Weights in two bf16 terms are off by at most 2^-8 2^-8 of themselves. A score is summed in eight steps, off by at most 2^-23 of sum |q k| scale (below 10 for these queries) each, which
    moves an exponent to base 2 by at most 8 2^-23 10 log2(e) < 2^-16, and a row's weights against their sum by at most twice that times ln 2; a part of 512 keys is summed in 64 steps, off by
    2^-23 each, and at most 60 parts are joined, off by 2^-24 each. Together less than 2^-14 of sum p |v|, beside the rounding of the result, at most 2^-8 of it."""
    rng = np.random.default_rng(heads + kv)
    t = Trees(cuda, heads, kv, [(n, bushy(m, rng, 20)) for n, m in forest], seed=len(forest))
    q = t.queries()
    got, x = _np(t.attention(q)).reshape(t.rows, heads, DIM), _np(q)
    for s, (n, parents) in enumerate(t.forest):
        a, b = t.row0[s], t.row0[s + 1]
        want, mass = tr.attention(x[a:b], *t.kvs[s], parents, n, DIM ** -0.5)
        assert (np.abs(got[a:b] - want) <= 2 ** -8 * np.abs(want) + 2 ** -14 * mass).all(), (s, n)
    assert int(t.status) == 0


def test_attention_shares_scratch_with_calls_of_its_shape_alone(cuda):
    rng = np.random.default_rng(2)
    a, b = (Trees(cuda, 4, 2, [(9000, bushy(5, rng))] * n, seed=1) for n in (1, 2))
    first = ops.TreeAttention(a.trees, a.queries(), a.pool)
    with pytest.raises(ValueError, match="another shape"):
        ops.TreeAttention(b.trees, b.queries(), b.pool, scratch_of=first)


@pytest.mark.parametrize("heads,kv,length", [(8, 2, 700), (2, 1, 30000), (4, 4, 6000)])
def test_attention_waits_that_run_out(cuda, heads, kv, length):
    """The keys of every CTA's first block are never asked for: code 3, and the GPU stays usable."""
    rng = np.random.default_rng(17)
    trees = 60 if kv == 4 else 1
    t = Trees(cuda, heads, kv, [(length if i == 0 else 300, bushy(9, rng)) for i in range(trees)], seed=3)
    q = t.queries()
    lib = gptrs_b200.lib()
    lib.gptrs_cuda_debug_prefill_tc_fault(1, 500)
    try:
        ops.tree_attention(t.trees, q, t.pool, status=t.status)
        torch.cuda.synchronize()
    finally:
        lib.gptrs_cuda_debug_prefill_tc_fault(0, 0)
    assert int(t.status) == 3
    t.status.zero_()
    t.check(t.attention(q), q)
    assert int(t.status) == 0


def test_attention_of_trees_that_change_in_place(cuda):
    """One object, and trees, lengths and parents that are written into its tensors: fewer nodes, padding, longer contexts than the call before."""
    rng = np.random.default_rng(18)
    t = Trees(cuda, 8, 2, [(300, bushy(20, rng)), (2000, bushy(20, rng)), (90, bushy(20, rng))], seed=6, max_nodes=24)
    q = t.queries()
    call = ops.TreeAttention(t.trees, q, t.pool, status=t.status)
    for step in range(4):
        t.check(call(), q)
        parents = [bushy(20, rng) for _ in range(3)]
        t.parent[:] = _ints(sum(parents, []), cuda)
        t.forest = [(f[0] - 7 * step, parents[i]) for i, f in enumerate(t.forest)]
        t.length[:] = _ints([f[0] for f in t.forest], cuda)
        t.kvs = [t.read(i, np.arange(f[0] + 20)) for i, f in enumerate(t.forest)]
    assert int(t.status) == 0


@pytest.mark.parametrize("wide", [1, 4000])
@pytest.mark.parametrize("heads,kv", [(2, 1), (32, 1), (12, 3)])
def test_as_many_trees_as_a_call_may_have(cuda, heads, kv, wide):
    """A few trees among 65535, the others padding or without nodes, under a narrow and a wide page table: the same as by themselves, within roundings."""
    rng = np.random.default_rng(heads)
    t = Trees(cuda, heads, kv, [(150, bushy(20, rng)), (0, bushy(3, rng)), (60, bushy(11, rng))], seed=1)
    q, n, at = t.queries(), 65535, np.array([0, 40000, 65534])
    table = torch.full((t.table.shape[0], max(wide, t.table.shape[1])), -1, dtype=torch.int32, device=cuda)
    table[:, :t.table.shape[1]] = t.table
    first = np.zeros(n + 1, dtype=np.int64)
    for k, a in enumerate(at):
        first[a + 1:] = t.row0[k + 1]
    slot, length = np.full(n, -1), np.full(n, -5)
    slot[1::7], length[1::7] = t.slots[0], 33                              # of no nodes
    slot[at], length[at] = t.slots, [150, 0, 60]
    many = ops.DraftTrees(heads, kv, _ints(first, cuda), _ints(slot, cuda), _ints(length, cuda), t.parent, table, t.max_nodes)
    t.check(ops.tree_attention(many, q, t.pool, status=t.status), q)
    token, pick = _ints(rng.integers(0, 3, t.rows), cuda), _ints(rng.integers(0, 3, t.rows), cuda)
    got, alone = ops.tree_accept(many, token, pick, status=t.status), ops.tree_accept(t.trees, token, pick, status=t.status)
    for a, b in zip(got, alone):
        assert a[torch.as_tensor(at, device=cuda)].equal(b)
    rest = torch.ones(n, dtype=torch.bool, device=cuda)
    rest[torch.as_tensor(at, device=cuda)] = False
    assert (got.count[rest] == 0).all() and (got.next[rest] == -1).all() and (got.path[rest] == -1).all() and got.length[rest].equal(many.tensors["length"][rest])
    assert int(t.status) == 0


def test_a_captured_step_reads_its_trees_when_it_runs(cuda):
    """Append, attention and acceptance of one layer in a graph, replayed with other lengths and parents: as eager calls on the same pool."""
    rng = np.random.default_rng(23)
    t = Trees(cuda, 8, 2, [(300, bushy(20, rng)), (45, bushy(13, rng))], seed=8)
    qkv = torch.randn((t.rows, 12 * DIM), device=cuda).bfloat16()
    cos, sin = (torch.randn((400, 64), device=cuda) for _ in range(2))
    token, pick = _ints(rng.integers(0, 3, t.rows), cuda), _ints(rng.integers(0, 3, t.rows), cuda)
    start = t.pool.clone()
    append = ops.TreeAppend(t.trees, qkv, cos, sin, t.pool, status=t.status)
    attend = ops.TreeAttention(t.trees, append.q, t.pool, status=t.status)
    accept = ops.TreeAccept(t.trees, token, pick, [t.pool], status=t.status)
    for call in (append, attend, accept):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append()
        out = attend()
        told = accept()
    for step in range(3):
        t.parent[:] = _ints(bushy(20, rng) + bushy(13, rng), cuda)
        t.length[:] = _ints([300 - 50 * step, 45 - 20 * step], cuda)
        t.pool.copy_(start)
        graph.replay()
        got, pool = [out.clone(), *(x.clone() for x in told)], t.pool.clone()
        t.pool.copy_(start)
        want = [append() is None or attend().clone(), *(x.clone() for x in accept())]
        for a, b in zip(got, want):
            assert a.equal(b)
        assert pool.equal(t.pool)
    assert int(t.status) == 0


# ---- append --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,rotary", [(32, 8, 128), (8, 1, 64), (12, 12, 16), (5, 1, 96), (3, 3, 0), (14, 2, 112)])
def test_append(cuda, heads, kv, rotary):
    rng = np.random.default_rng(heads + rotary)
    t = Trees(cuda, heads, kv, [(75, bushy(26, rng)), (0, chain(3)), None, (31, bushy(17, rng)), (1, [-1])], seed=heads, extra_rows=2, fill=False, max_nodes=30)
    qkv = torch.tensor(rng.normal(0, 1, (t.rows, heads + 2 * kv, DIM)), dtype=torch.float32).bfloat16().to(cuda)
    ang = rng.uniform(-4, 4, (110, rotary // 2))
    cos, sin = (torch.tensor(f(ang), dtype=torch.float32, device=cuda) for f in (np.cos, np.sin)) if rotary else (None, None)
    wide = torch.full((t.rows, (heads + 2 * kv) * DIM + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 8:8 + (heads + 2 * kv) * DIM] = qkv.view(t.rows, -1)
    q = torch.full((t.rows, heads, DIM), 5.0, dtype=torch.bfloat16, device=cuda)
    got = ops.tree_append(t.trees, wide[:, 8:8 + (heads + 2 * kv) * DIM], cos, sin, t.pool, q=q, status=t.status)
    assert int(t.status) == 0 and (q[47:] == 5).all()
    x = _np(qkv)
    for s, f in enumerate(t.forest):
        if f is None:
            continue
        a, b = t.row0[s], t.row0[s + 1]
        at = f[0] + np.array([len(c) - 1 for c in tr.ancestors(f[1])], dtype=int)
        want = tr.rotate(x[a:b, :heads + kv], at, _np(cos), _np(sin)) if rotary else x[a:b, :heads + kv].astype(float)
        keys, values = t.read(s, np.arange(f[0], f[0] + len(f[1])))
        size = np.abs(x[a:b, :heads + kv]).max(-1, keepdims=True)
        tol = 2 ** -8 * np.abs(want) + 2 ** -21 * size
        assert (np.abs(np.concatenate([_np(got)[a:b], keys], 1) - want) <= tol).all()
        assert np.array_equal(values, x[a:b, heads + kv:])
        if f[0]:
            assert np.isnan(t.read(s, np.arange(f[0]))).all()            # what the cache held stays
    ok = ~torch.isnan(t.view()).view(t.pages, -1)
    assert int(ok.sum()) == sum(len(f[1]) for f in t.forest if f) * kv * 2 * DIM


def test_append_out_of_range(cuda):
    rng = np.random.default_rng(3)
    t = Trees(cuda, 4, 2, [(30, chain(6)), (9, chain(4))], seed=2, fill=False)
    qkv = torch.randn((t.rows, 8 * DIM), device=cuda).bfloat16()
    cos, sin = torch.rand((33, 64), device=cuda), torch.rand((33, 64), device=cuda)
    t.table[int(t.slots[1]), 0] = -1
    got = ops.tree_append(t.trees, qkv, cos, sin, t.pool, status=t.status)
    assert int(t.status) == 2
    x = _np(qkv).reshape(-1, 8, DIM)
    want = tr.rotate(x[:, :4], np.array([30, 31, 32, 0, 0, 0, 9, 10, 11, 12]), _np(cos), _np(sin))
    assert (np.abs(_np(got) - want) <= 2 ** -8 * np.abs(want) + 2 ** -20 * np.abs(x[:, :4]).max(-1, keepdims=True)).all()
    assert int((~torch.isnan(t.view())).sum()) == 6 * 2 * 2 * DIM


# ---- acceptance ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,layers,seed", [(8, 3, 0), (1, 1, 1), (12, 2, 2), (2, 0, 3), (3, 5, 4)])
def test_accept(cuda, kv, layers, seed):
    rng = np.random.default_rng(seed)
    forest = [(int(rng.integers(0, 60)), bushy(int(rng.integers(1, 60)), rng)) for _ in range(6)] + [None, (5, []), (14, chain(40)), (33, [-1, -1, 0, 2, 2, 3])]
    t = Trees(cuda, 2 * kv, kv, forest, seed=seed, max_nodes=70, extra_rows=3)
    token, pick = rng.integers(0, 4, t.rows), rng.integers(0, 4, t.rows)   # few tokens: paths, and children of one parent with the same one
    a = t.row0[8]
    token[a:a + 40] = pick[a - 1:a + 39]
    pick[a:a + 39] = token[a + 1:a + 40]                                   # all of a chain
    pools = [(torch.rand(t.pool.numel() // 2, device=cuda) - 0.5).bfloat16().view(torch.uint8) for _ in range(layers)]
    old = [p.clone() for p in pools]
    got = ops.tree_accept(t.trees, _ints(token, cuda), _ints(pick, cuda), pools, status=t.status)
    assert int(t.status) == 0
    for s, f in enumerate(t.forest):
        a, b = t.row0[s], t.row0[s + 1]
        path, follows = tr.accept([], [], []) if f is None else tr.accept(f[1], token[a:b], pick[a:b])
        assert got.path[s].tolist() == path + [-1] * (70 - len(path))
        assert (int(got.count[s]), int(got.next[s]), int(got.length[s])) == (len(path), follows, (f[0] if f else 0) + len(path))
        for p, o in zip(pools, old):
            if path:
                moved = t.read(s, [f[0] + i for i in path], o)
                assert np.array_equal(t.read(s, np.arange(f[0], f[0] + len(path)), p), moved)
                t.write(s, np.arange(f[0], f[0] + len(path)), torch.tensor(moved).bfloat16(), o)
    for p, o in zip(pools, old):
        assert p.equal(o)                                                  # nothing else moved


def test_accept_pages_and_trees_out_of_range(cuda):
    t = Trees(cuda, 2, 1, [(14, [-1, 0, 0, 2, 2, 4]), (3, chain(3))], seed=1)
    token = [9, 1, 2, 3, 4, 5, 9, 1, 2]
    pick = [2, 0, 4, 0, 5, 7, 1, 2, 3]
    t.slot[1] = 3
    t.table[int(t.slots[0]), 1] = t.pages
    old = t.pool.clone()
    got = ops.tree_accept(t.trees, _ints(token, cuda), _ints(pick, cuda), [t.pool], status=t.status)
    assert int(t.status) == 2 and got.count.tolist() == [4, 0] and got.path[0].tolist() == [0, 2, 4, 5, -1, -1] and got.next.tolist() == [7, -1] and got.length.tolist() == [18, 3]
    assert t.pool.equal(old)                                               # from the page that is none, nothing
