"""A step of speculative decoding: drafted tokens that form a tree go into the paged bf16 cache, attend to what they see of it, are scored against the
vocabulary without logits in memory, and the accepted path's keys and values move to their places.

Trees. Tree s is the rows first[s] .. first[s + 1] - 1 of a call; node i of it has parent[i] < i (a node of the same tree) or -1. Its sequence holds
length[s] tokens; node i lies in the cache at position length + i and is rotated by position length + depth(i). It sees the length tokens, its
ancestors and itself. Node 0 is the token that was chosen last, the others are drafts.

The cache. A page holds 16 tokens; pool[page][kv head][key, value][token][128] in bf16, the eight channels 8 c .. 8 c + 7 of token t at chunk c ^ (t % 8).

Scores. z = hidden . weight^T; of every row the log-probability of a given token, log sum exp z, and a pick: the first largest z, or with a temperature
T the largest z / T - log(-log(1 - v)), v = (h + 1/2) / 2^32 in f32, h a hash of (seed, row, token), with that token's log-probability (at T = 1).

Acceptance. From node 0 on, the child with the lowest number whose token is its parent's pick, until there is none.

Where `own` is false, `run` computes the operators with elementary torch operations; where it is true, with the framework's. `exact` computes
them in 64 bits."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

PAGE, DIM = 16, 128


def listed():
    return [
        # One user's draft of 26 tokens behind a chat of 1500.
        dict(name="append-one", op="append", trees=1, few=26, nodes=26, low=1500, high=1500, heads=32, kv_heads=8),
        # A server's full batch, trees of unequal sizes.
        dict(name="append-batch", op="append", trees=64, few=20, nodes=64, low=200, high=4000, heads=32, kv_heads=8),
        # One user: the shortest wait for a verified draft.
        dict(name="attend-one", op="attend", trees=1, few=26, nodes=26, low=1500, high=1500, heads=32, kv_heads=8),
        # A server's batch with 512 to 8192 cached tokens each.
        dict(name="attend-batch", op="attend", trees=64, few=32, nodes=32, low=512, high=8192, heads=32, kv_heads=8),
        # Two readers of whole books with small drafts.
        dict(name="attend-long", op="attend", trees=2, few=13, nodes=16, low=100003, high=131072, heads=32, kv_heads=8),
        # Few sequences with large trees, eight query heads per kv head.
        dict(name="attend-wide", op="attend", trees=6, few=201, nodes=250, low=700, high=4000, heads=16, kv_heads=2),
        # Fresh and short sequences with drafts of one to seventeen tokens, heads without groups.
        dict(name="attend-short", op="attend", trees=13, few=1, nodes=17, low=0, high=700, heads=12, kv_heads=12),
        # The next token of one user, sampled, from a vocabulary of odd size.
        dict(name="score-one", op="score", rows=1, dim=2048, vocab=50257, temperature=0.8),
        # The drafts of sixteen users, sampled.
        dict(name="score-drafts", op="score", rows=416, dim=4096, vocab=131072, temperature=0.7),
        # How likely a text is: every token of long prompts, greedy picks.
        dict(name="score-prompt", op="score", rows=4001, dim=2048, vocab=131072, temperature=0.0),
        # One user's accepted draft in all layers.
        dict(name="accept-one", op="accept", trees=1, few=26, nodes=26, low=1500, high=1500, accepted=5, layers=26, heads=32, kv_heads=8),
        # A server's batch.
        dict(name="accept-batch", op="accept", trees=64, few=20, nodes=64, low=200, high=4000, accepted=9, layers=26, heads=32, kv_heads=8),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _one(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "score", "score", "score", "accept"])
    if op == "score":
        dim = 8 * _log_uniform(rng, 32, 640)
        temperature = rng.choice([0.0, 0.0, 0.6, 1.0])
        return dict(op=op, rows=_log_uniform(rng, 1, 512 if temperature else 4001), dim=dim, vocab=_log_uniform(rng, 1000, 160000), temperature=temperature)
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 4), (16, 2), (12, 12), (24, 8), (40, 8), (28, 4), (8, 1), (6, 6)])
    trees = _log_uniform(rng, 1, 96)
    few, nodes = sorted((_log_uniform(rng, 1, 256), _log_uniform(rng, 1, 256)))
    longest = 6000 if op == "accept" else 250000 // trees
    low, high = sorted((_log_uniform(rng, 1, longest) - 1, _log_uniform(rng, 1, longest) - 1))
    case = dict(op=op, trees=trees, few=few, nodes=nodes, low=low, high=high, heads=heads, kv_heads=kv_heads)
    return case if op != "accept" else dict(case, accepted=_log_uniform(rng, 1, 16), layers=_log_uniform(rng, 1, 40))


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        most[case["op"]] = {k: max(w[k], most.get(case["op"], w)[k]) for k in w}
    while True:   # no more than the operator's largest listed case
        case = _one(rng)
        w = work(case)
        if all(w[k] <= most[case["op"]][k] for k in w):
            return case


def _spread(n, low, high):
    """n whole numbers over the range, unequal, the largest one among them."""
    if n == 1:
        return [high]
    at = [(i * 37) % n for i in range(n)] if math.gcd(37, n) == 1 else list(range(n))
    return [low + (high - low) * a // (n - 1) for a in at]


def _sizes(case):
    """(committed tokens, nodes) of every tree."""
    return list(zip(_spread(case["trees"], case["low"], case["high"]), _spread(case["trees"], case["few"], case["nodes"])[::-1]))


def _accepted(case):
    """Nodes of the accepted path of every tree: the larger half of a tree has room for the nodes that move."""
    return [max(1, min(a, n // 2)) for a, (_, n) in zip(_spread(case["trees"], 1, case["accepted"]), _sizes(case))]


def work(case):
    if case["op"] == "score":
        r, d, v = case["rows"], case["dim"], case["vocab"]
        return {"bytes": 2 * d * (v + r) + 20 * r, "flops": 2 * r * d * v}
    h, g = case["heads"], case["kv_heads"]
    rows = sum(n for _, n in _sizes(case))
    if case["op"] == "append":
        return {"bytes": rows * 2 * DIM * (2 * h + 4 * g), "flops": rows * 6 * DIM * (h + g)}
    if case["op"] == "attend":   # a node sees at least the committed tokens and itself
        return {"bytes": sum(m + n for m, n in _sizes(case)) * g * 4 * DIM + rows * h * 4 * DIM, "flops": sum(n * (m + 1) for m, n in _sizes(case)) * h * 4 * DIM}
    moved = sum(a - 1 for a in _accepted(case))
    return {"bytes": moved * case["layers"] * g * 8 * DIM + 12 * rows, "flops": 4 * rows}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _trees(case, gen, dev):
    """Parents, tokens and picks. A path of the accepted length runs through the nodes; it moves to places that no other node of it comes from."""
    rand = torch.Generator().manual_seed(int(torch.randint(0, 1 << 30, (1,), generator=gen, device=dev)))
    parents, tokens, picks = [], [], []
    for (_, n), a in zip(_sizes(case), _accepted(dict(case, accepted=case.get("accepted", 8)))):
        up = (torch.rand(n, generator=rand) * torch.arange(n).clamp_max(12)).long()             # among the last dozen: trees of some depth
        up = torch.arange(n) - 1 - up
        up[0] = -1
        path = [0] + sorted((torch.randperm(n - a, generator=rand)[:a - 1] + a).tolist())
        up[path[1:]] = torch.tensor(path[:-1], dtype=torch.int64)
        token = torch.randperm(50000, generator=rand)[:n]
        pick = torch.randint(50000, 60000, (n,), generator=rand)
        off = torch.rand(n, generator=rand) < 0.5                                                # some nodes off the path are right about a child of theirs
        off[path] = False
        child = torch.arange(n)[off[up] & (up >= 0)]
        pick[up[child]] = token[child]
        pick[path[:-1]] = token[path[1:]]
        parents.append(up)
        tokens.append(token)
        picks.append(pick)
    ints = lambda v: torch.cat(v).int().to(dev)  # noqa: E731
    return ints(parents), ints(tokens), ints(picks)


def _pool(case, gen, dev, layers, shared):
    """Page table and pools [layers][bytes]; `shared`: all pages in front of the last few hold one prompt that the sequences have in common."""
    sizes, g = _sizes(case), case["kv_heads"]
    need = [(m + n + PAGE - 1) // PAGE for m, n in sizes]
    first = [m // PAGE if shared else 0 for m, _ in sizes]
    pages = sum(b - a for a, b in zip(first, need)) + max(first) + 3
    perm = torch.randperm(pages, device=dev, generator=gen).int()
    table, at = torch.zeros((case["trees"], max(need)), dtype=torch.int32, device=dev), max(first)
    for i, (a, b) in enumerate(zip(first, need)):
        table[i, :a] = perm[:a]
        table[i, a:b] = perm[at:at + b - a]
        at += b - a
    pool = torch.empty((layers, pages, g, 2, PAGE, DIM), dtype=torch.bfloat16, device=dev)
    for layer in range(layers):
        for p in range(0, pages, 4096):
            pool[layer, p:p + 4096] = torch.randn(pool[layer, p:p + 4096].shape, device=dev, generator=gen, dtype=torch.float16)
    return table, pool.view(torch.uint8).view(layers, -1)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    st = SimpleNamespace(case=case, made=None, status=torch.zeros(1, dtype=torch.int32, device=dev))
    if case["op"] == "score":   # a model that is more or less sure of one token
        r, d, v = case["rows"], case["dim"], case["vocab"]
        st.weight = torch.empty((v, d), dtype=torch.bfloat16, device=dev)
        for i in range(0, v, 16384):
            st.weight[i:i + 16384] = torch.randn(st.weight[i:i + 16384].shape, device=dev, generator=gen) * (2.5 / math.sqrt(d))
        sure = torch.randint(0, v, (r,), device=dev, generator=gen)
        size = 4 + 18 * torch.rand((r, 1), device=dev, generator=gen)
        st.hidden = (torch.randn((r, d), device=dev, generator=gen) + st.weight[sure].float() * (size / 6.25)).bfloat16()
        other = torch.randint(0, v, (r,), device=dev, generator=gen)
        st.target = torch.where(torch.rand(r, device=dev, generator=gen) < 0.5, sure, other).int()
        st.seed = seed % (1 << 32)
        return st
    h, g = case["heads"], case["kv_heads"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    sizes = _sizes(case)
    st.parent, st.token, st.pick = _trees(case, gen, dev)
    st.length = ints([m for m, _ in sizes])
    st.first = ints([sum(n for _, n in sizes[:i]) for i in range(len(sizes) + 1)])
    st.slot = torch.randperm(case["trees"], device=dev, generator=gen).int()
    st.table, st.pools = _pool(case, gen, dev, case.get("layers", 1), shared=case["op"] != "attend")
    table = st.table.clone()
    table[st.slot.long()] = st.table                                                             # tree s has the pages of its slot
    st.table = table
    rows = st.parent.shape[0]
    if case["op"] == "append":
        st.qkv = torch.randn((rows, (h + 2 * g) * DIM), device=dev, generator=gen).bfloat16()
        freq = 1e6 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device=dev) / DIM)
        angle = torch.arange(max(m + n for m, n in sizes), dtype=torch.float64, device=dev)[:, None] * freq
        st.cos, st.sin = angle.cos().float(), angle.sin().float()
    if case["op"] == "attend":
        st.q = (1.5 * torch.randn((rows, h, DIM), device=dev, generator=gen)).bfloat16()
    return st


# ---- the operators in elementary operations -----------------------------------------------------------------------------------------
def _dense(st):
    """Trees side by side: (tree of each row, number of each row in it, parents [trees][nodes] with -1 where there is none, what each node has above it or is)."""
    rows, t, n = torch.arange(st.parent.shape[0], device=st.parent.device), st.case["trees"], st.case["nodes"]
    tree = torch.searchsorted(st.first.long(), rows, right=True) - 1
    node = rows - st.first.long()[tree]
    parent = torch.full((t, n), -1, dtype=torch.int64, device=rows.device)
    parent[tree, node] = st.parent.long()
    every = torch.arange(n, device=rows.device)
    above = ((parent[:, :, None] == every) | (every[:, None] == every)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        above = (above @ above).clamp_max(1)
    return tree, node, parent, above > 0


def _place(st, tree, position):
    """Page, token and chunks [.., 16] of positions of trees' sequences."""
    page = st.table.long()[st.slot.long()[tree], position // PAGE]
    tok = position % PAGE
    return page[..., None], tok[..., None], torch.arange(16, device=page.device) ^ (tok[..., None] % 8)


def _view(st):
    return st.pools.view(torch.bfloat16).view(st.pools.shape[0], -1, st.case["kv_heads"], 2, PAGE, 16, 8)


def _plain_append(st):
    h, g = st.case["heads"], st.case["kv_heads"]
    tree, node, _, above = _dense(st)
    base = st.length.long()[tree]
    at = base + above.sum(-1)[tree, node] - 1
    x = st.qkv.float().view(-1, h + 2 * g, DIM)
    a, b = x[:, :h + g, :DIM // 2], x[:, :h + g, DIM // 2:]
    c, s = st.cos[at][:, None], st.sin[at][:, None]
    turned = torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16()
    kv = torch.stack([turned[:, h:], st.qkv.view(-1, h + 2 * g, DIM)[:, h + g:]], 2)             # [rows][g][2][128]
    page, tok, chunk = _place(st, tree, base + node)
    _view(st)[0][page, :, :, tok, chunk] = kv.view(-1, g, 2, 16, 8).permute(0, 3, 1, 2, 4)
    return {"q": turned[:, :h].contiguous(), "pool": st.pools.view(torch.bfloat16)}


def _plain_attention(st):
    h, g, t, n = (st.case[k] for k in ("heads", "kv_heads", "trees", "nodes"))
    tree, node, _, above = _dense(st)
    per = st.table.shape[1] * PAGE
    tok = torch.arange(PAGE, device=st.q.device)[:, None]
    pages = _view(st)[0][st.table.long()[st.slot.long()]]                                        # [trees][pages][g][2][16][16][8]
    kv = pages[..., tok, torch.arange(16, device=st.q.device) ^ (tok % 8), :].permute(3, 0, 1, 4, 2, 5, 6).reshape(2, t, per, g, DIM).float()
    q = torch.zeros((t, n, h, DIM), device=st.q.device)
    q[tree, node] = st.q.float() * DIM ** -0.5
    behind = torch.arange(per, device=q.device) - st.length.long()[:, None]                      # number of the node at a position
    seen = torch.gather(above, 2, behind.clamp(0, n - 1)[:, None].expand(t, n, per)) & (behind < n)[:, None]
    seen |= (behind < 0)[:, None]
    s = torch.einsum("bmgnd,bkgd->bgnmk", q.view(t, n, g, h // g, DIM), kv[0])
    s.masked_fill_(~seen[:, None, None], -torch.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.einsum("bgnmk,bkgd->bmgnd", s, kv[1]) / total.permute(0, 3, 1, 2, 4)
    return {"out": out.reshape(t, n, h * DIM)[tree, node].bfloat16()}


def _hash(x):
    x = (x ^ (x >> 16)) * 0x7feb352d & 0xffffffff
    x = (x ^ (x >> 15)) * 0x846ca68b & 0xffffffff
    return x ^ (x >> 16)


def _uniform(st, row, tokens):
    """v of row `row` (a column of them) and every token, in f32."""
    h = _hash(st.seed ^ _hash((tokens + 0x9e3779b9 * (row + 1)) & 0xffffffff))
    return (h.float() + 0.5) * 2.0 ** -32


def _plain_scores(st):
    z = st.hidden.float() @ st.weight.float().t()
    m = z.amax(-1, keepdim=True)
    lse = (m + (z - m).exp().sum(-1, keepdim=True).log())[:, 0]
    given = z.gather(1, st.target.long()[:, None])[:, 0] - lse
    if st.case["temperature"] > 0:
        rows, tokens = (torch.arange(n, device=z.device) for n in z.shape)
        pick = (z / st.case["temperature"] - (-torch.log1p(-_uniform(st, rows[:, None], tokens))).log()).argmax(-1)
    else:
        pick = z.argmax(-1)
    return {"pick": pick.int(), "pick_logprob": z.gather(1, pick[:, None])[:, 0] - lse, "logprob": given, "lse": lse}


def _plain_accept(st):
    t, n = st.case["trees"], st.case["nodes"]
    tree, node, parent, above = _dense(st)
    token, pick = (torch.full((t, n), -1 - i, dtype=torch.int64, device=parent.device) for i in range(2))
    token[tree, node], pick[tree, node] = st.token.long(), st.pick.long()
    right = (parent >= 0) & (token == pick.gather(1, parent.clamp_min(0)))
    every = torch.arange(n, device=parent.device)
    twin = (parent[:, :, None] == parent[:, None]) & right[:, None] & (every[:, None] > every)   # a right one of the same parent in front
    right &= ~twin.any(-1)
    right[:, 0] = True
    taken = ~(above & ~right[:, None]).any(-1) & above[:, :, 0]
    count = taken.sum(-1)
    path = torch.where(taken, every, n).sort(-1).values
    path = torch.where(every < count[:, None], path, -1)
    follow = pick.gather(1, path.gather(1, count[:, None] - 1))[:, 0]
    who, k = torch.nonzero((path >= 0) & (every > 0), as_tuple=True)
    base, view = st.length.long()[who], _view(st)
    page, tok, chunk = _place(st, who, base + path[who, k])
    moved = view[:, page, :, :, tok, chunk]
    page, tok, chunk = _place(st, who, base + k)
    view[:, page, :, :, tok, chunk] = moved
    return {"count": count.int(), "path": path.int(), "next": follow.int(), "length": st.length + count.int(), "pool": st.pools.view(torch.bfloat16)}


# ---- the framework's operators ------------------------------------------------------------------------------------------------------
def _make(st):
    """What a serving loop keeps from step to step: the calls with their buffers."""
    import __graft_entry__
    __graft_entry__.load_package()
    from gptrs_b200 import ops
    case = st.case
    if case["op"] == "score":
        return ops.VocabScores(st.hidden, st.weight, target=st.target, temperature=case["temperature"], seed=st.seed, status=st.status)
    trees = ops.DraftTrees(case["heads"], case["kv_heads"], st.first, st.slot, st.length, st.parent, st.table, max_nodes=case["nodes"])
    if case["op"] == "append":
        return ops.TreeAppend(trees, st.qkv, st.cos, st.sin, st.pools[0], status=st.status)
    if case["op"] == "attend":
        return ops.TreeAttention(trees, st.q, st.pools[0], status=st.status)
    return ops.TreeAccept(trees, st.token, st.pick, list(st.pools), status=st.status)


def run(st):
    if own:
        if st.made is None:
            st.made = _make(st)
        got = st.made()
        if st.case["op"] == "score":
            return {"pick": got.pick, "pick_logprob": got.pick_logprob, "logprob": got.logprob, "lse": got.lse}
        if st.case["op"] == "accept":
            return {"count": got.count, "path": got.path, "next": got.next, "length": got.length, "pool": st.pools.view(torch.bfloat16)}
        return {"q": got, "pool": st.pools.view(torch.bfloat16)} if st.case["op"] == "append" else {"out": got}
    return {"append": _plain_append, "attend": _plain_attention, "score": _plain_scores, "accept": _plain_accept}[st.case["op"]](st)


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------------
def _chains(st):
    """For every row its tree, its number, and the numbers of its ancestors and itself."""
    found, first, parent = [], st.first.tolist(), st.parent.tolist()
    for s in range(st.case["trees"]):
        seen = []
        for i in range(first[s + 1] - first[s]):
            up = parent[first[s] + i]
            seen.append((seen[up] if up >= 0 else []) + [i])
            found.append((s, i, seen[i]))
    return found


def _offsets(st, s, positions):
    """Where in a layer's pool the keys of kv head 0 at these positions of tree s lie: [positions][128] values."""
    page = st.table[int(st.slot[s])].long()[positions // PAGE]
    tok, dim = positions % PAGE, torch.arange(DIM, device=positions.device)
    return ((page * (2 * st.case["kv_heads"] * PAGE) + tok) * DIM)[:, None] + (dim // 8 ^ tok[:, None] % 8) * 8 + dim % 8


def _exact_append(st):
    h, g = st.case["heads"], st.case["kv_heads"]
    chains = _chains(st)
    base = st.length.long()
    tree, node, depth = (torch.tensor(v, device=base.device) for v in ([c[0] for c in chains], [c[1] for c in chains], [len(c[2]) - 1 for c in chains]))
    turn = torch.complex(st.cos.double(), st.sin.double())[base[tree] + depth][:, None]
    x = st.qkv.double().reshape(-1, h + 2 * g, DIM)
    z = torch.complex(x[:, :h + g, :64], x[:, :h + g, 64:]) * turn
    z = torch.cat([z.real, z.imag], -1)
    pool = st.pools.view(torch.bfloat16)[0].double()
    for s in range(st.case["trees"]):
        mine = tree == s
        at = _offsets(st, s, base[s] + node[mine])
        for kv in range(g):
            pool[at + kv * 2 * PAGE * DIM] = z[mine, h + kv]
            pool[at + (kv * 2 + 1) * PAGE * DIM] = x[mine, h + g + kv]
    return {"q": z[:, :h].contiguous(), "pool": pool[None]}


def _exact_attention(st):
    h, g, per = st.case["heads"], st.case["kv_heads"], st.case["heads"] // st.case["kv_heads"]
    chains, pool = _chains(st), st.pools.view(torch.bfloat16)[0]
    out = torch.empty((len(chains), h, DIM), dtype=torch.float64, device=pool.device)
    row = 0
    for s, (length, n) in enumerate(_sizes(st.case)):
        at = _offsets(st, s, torch.arange(length + n, device=pool.device))
        hidden = torch.zeros((n, length + n), dtype=torch.bool)
        hidden[:, length:] = True
        for _, i, seen in chains[row:row + n]:
            hidden[i, [length + j for j in seen]] = False
        hidden = hidden.to(pool.device)
        for kv in range(g):
            k, v = pool[at + kv * 2 * PAGE * DIM].double(), pool[at + (kv * 2 + 1) * PAGE * DIM].double()
            for j in range(kv * per, kv * per + per):
                z = st.q[row:row + n, j].double() @ k.t() / math.sqrt(DIM)
                out[row:row + n, j] = z.masked_fill(hidden, -math.inf).softmax(-1) @ v
        row += n
    return {"out": out.flatten(1)}


def _exact_scores(st):
    r, v = st.case["rows"], st.case["vocab"]
    pick, tokens = torch.empty(r, dtype=torch.int32, device=st.hidden.device), torch.arange(v, device=st.hidden.device)
    picked, given, lse = (torch.empty(r, dtype=torch.float64, device=pick.device) for _ in range(3))
    weight = st.weight.double()
    for a in range(0, r, 256):
        part = slice(a, min(a + 256, r))
        z = st.hidden[part].double() @ weight.t()
        lse[part] = z.logsumexp(-1)
        given[part] = z.gather(1, st.target[part].long()[:, None])[:, 0] - lse[part]
        noisy = z
        if st.case["temperature"] > 0:
            rows = torch.arange(part.start, part.stop, device=z.device)[:, None]
            noisy = z / st.case["temperature"] - torch.log(-torch.log1p(-_uniform(st, rows, tokens).double()))
        at = noisy.argmax(-1)
        pick[part] = at.int()
        picked[part] = z.gather(1, at[:, None])[:, 0] - lse[part]
    return {"pick": pick, "pick_logprob": picked, "logprob": given, "lse": lse}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "accept":   # whole numbers and copies
        return None
    return {"append": _exact_append, "attend": _exact_attention, "score": _exact_scores}[case["op"]](st)
