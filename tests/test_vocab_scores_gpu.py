"""Scores of rows against a vocabulary without logits in memory, against the oracle in 64 bits.

Tolerances. Products of bf16 are exact; the tensor cores add 16 of them at a time to an f32 sum and cut what does not fit, off by at most 2^-23 of the sum of magnitudes
A = sum |x w| each time: (dim / 16 + 8) 2^-23 A for a logit (e; a soft cap makes it no larger, a bias adds a rounding, 2^-24 of the logit). lse moves by the largest e at
most, log-probabilities by twice that; exponentials, logarithms and the last differences are f32: 2^-20 of the numbers that meet. A pick is one whose own value is
within the errors of the largest one's."""
import math

import numpy as np
import pytest
import torch

import gptrs_b200
from gptrs_b200 import ops
from oracle import tree_ref as tr

pytestmark = pytest.mark.gpu


def _np(t):
    return t.float().cpu().numpy()


def _inputs(cuda, rows, dim, vocab, seed=0, sure=True):
    rng = np.random.default_rng(seed)
    w = rng.normal(0, 2.5 / np.sqrt(dim), (vocab, dim))
    x = rng.normal(0, 1, (rows, dim))
    if sure:
        x += w[rng.integers(0, vocab, rows)] * rng.uniform(0, 3, (rows, 1))
    bf = lambda v: torch.tensor(v, dtype=torch.float32).bfloat16().to(cuda)  # noqa: E731
    return rng, bf(x), bf(w)


def _check(got, x, w, target, bias=None, cap=0.0, temperature=0.0, seed=0):
    z, mass = tr.logits(_np(x), _np(w), None if bias is None else _np(bias), cap)
    e = (x.shape[1] / 16 + 8) * 2 ** -23 * mass + 2 ** -23 * np.where(np.isfinite(z), np.abs(z), 0) * (2 if cap else 1)
    most, lse = e.max(-1), tr.lse(z)
    rows = np.arange(len(z))
    assert (np.abs(_np(got.lse) - lse) <= most + 2 ** -20 * (1 + np.abs(lse))).all()
    for lp, at in ((got.logprob, target), (got.pick_logprob, got.pick.cpu().numpy())):
        if lp is None:
            continue
        at = np.asarray(at)
        assert (at < w.shape[0]).all()
        want = np.where(at < 0, 0, z[rows, np.maximum(at, 0)] - lse)
        tol = 2 * most + 2 ** -20 * (1 + np.abs(lse) + np.abs(np.where(np.isfinite(want), want, 0)))
        ok = np.isfinite(want)
        assert (np.abs(_np(lp)[ok] - want[ok]) <= tol[ok]).all() and np.array_equal(_np(lp)[~ok], want[~ok])
    value, slack = z, 2 * most + 2 ** -22 * np.abs(z.max(-1))
    if temperature > 0:
        g = tr.noise(seed, *z.shape)
        value = z / temperature + g
        slack = 2 * (most + 2 ** -22 * np.abs(z.max(-1))) / temperature + 2 ** -18 * 24
    pick = got.pick.cpu().numpy()
    assert (value.max(-1) - value[rows, pick] <= slack).all()
    second = np.partition(value, -2, -1)[:, -2] if w.shape[0] > 1 else np.full(len(z), -np.inf)
    clear = value.max(-1) - second > slack
    assert np.array_equal(pick[clear], value.argmax(-1)[clear])


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 63, 64, 65, 127, 128, 129, 200, 256, 257, 300])
@pytest.mark.parametrize("dim,vocab", [(64, 1000), (136, 257), (512, 3001)])
def test_rows(cuda, rows, dim, vocab):
    rng, x, w = _inputs(cuda, rows, dim, vocab, seed=rows + dim)
    target = rng.integers(-1, vocab, rows)
    got = ops.vocab_scores(x, w, target=torch.tensor(target, dtype=torch.int32, device=cuda))
    _check(got, x, w, target)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 5000, 50257, 131072])
def test_vocabularies(cuda, vocab):
    rng, x, w = _inputs(cuda, 5, 72, vocab, seed=vocab)
    target = np.array([0, vocab - 1, vocab // 2, -1, vocab // 3])
    for temperature in (0.0, 0.7):
        got = ops.vocab_scores(x, w, target=torch.tensor(target, dtype=torch.int32, device=cuda), temperature=temperature, seed=77)
        _check(got, x, w, target, temperature=temperature, seed=77)


@pytest.mark.parametrize("dim", [8, 16, 24, 64, 72, 200, 256, 520, 1024, 2048, 4104, 8192])
def test_dims(cuda, dim):
    rng, x, w = _inputs(cuda, 9, dim, 777, seed=dim)
    target = rng.integers(0, 777, 9)
    got = ops.vocab_scores(x, w, target=torch.tensor(target, dtype=torch.int32, device=cuda))
    _check(got, x, w, target)


@pytest.mark.parametrize("rows,dim,vocab", [(33, 256, 1999), (300, 128, 700), (1000, 264, 5003)])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 5.0])
def test_bias_cap_and_temperature(cuda, rows, dim, vocab, temperature):
    rng, x, w = _inputs(cuda, rows, dim, vocab, seed=rows)
    bias = rng.normal(0, 1, vocab)
    bias[rng.integers(0, vocab, vocab // 3)] = -np.inf                       # tokens that are not allowed
    bias = torch.tensor(bias, dtype=torch.float32, device=cuda)
    target = rng.integers(0, vocab, rows)
    t = torch.tensor(target, dtype=torch.int32, device=cuda)
    _check(ops.vocab_scores(x, w, target=t, bias=bias, temperature=temperature, seed=5), x, w, target, bias=bias, temperature=temperature, seed=5)
    _check(ops.vocab_scores(x, w, target=t, soft_cap=6.0, temperature=temperature, seed=6), x, w, target, cap=6.0, temperature=temperature, seed=6)


def test_strides_and_only_what_is_asked_for(cuda):
    rng, x, w = _inputs(cuda, 70, 96, 900, seed=3)
    wide_x = torch.full((70, 120), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_w = torch.full((900, 104), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide_x[:, 8:104], wide_w[:, :96] = x, w
    want = ops.vocab_scores(x, w)
    got = ops.vocab_scores(wide_x[:, 8:104], wide_w[:, :96])
    assert want.logprob is None and all(a is None or a.equal(b) for a, b in zip(got, want))
    call = ops.VocabScores(x, w)
    call.step.d_pick = call.step.d_lse = None
    for r in (call.result.pick, call.result.lse):
        r.fill_(-9)
    call()
    assert (call.result.pick == -9).all() and (call.result.lse == -9).all() and call.result.pick_logprob.equal(want.pick_logprob)


def test_equal_logits_give_the_first_token(cuda):
    x = torch.ones((130, 64), device=cuda).bfloat16()
    w = torch.zeros((3000, 64), device=cuda).bfloat16()
    assert (ops.vocab_scores(x, w).pick == 0).all()
    w[[1234, 2999, 1235, 700]] = 0.25
    got = ops.vocab_scores(x, w)
    assert (got.pick == 700).all()
    assert (got.lse - np.log(2996 + 4 * np.exp(16.0))).abs().max() < 1e-5


def test_what_is_not_finite(cuda):
    rng, x, w = _inputs(cuda, 140, 64, 600, seed=4)
    want = ops.vocab_scores(x, w, target=torch.zeros(140, dtype=torch.int32, device=cuda))
    x[3, 5] = float("nan")
    x[131, 0] = float("nan")
    for temperature in (0.0, 1.0):
        got = ops.vocab_scores(x, w, target=torch.zeros(140, dtype=torch.int32, device=cuda), temperature=temperature)
        bad = torch.zeros(140, dtype=torch.bool, device=cuda)
        bad[[3, 131]] = True
        assert torch.isnan(got.lse).equal(bad) and torch.isnan(got.logprob).equal(bad) and torch.isnan(got.pick_logprob).equal(bad)
        assert ((got.pick >= 0) & (got.pick < 600)).all() and got.lse[~bad].equal(want.lse[~bad])
    none = torch.full((600,), float("-inf"), device=cuda)
    none[17] = 2.0
    got = ops.vocab_scores(x[:3].contiguous(), w, bias=none)
    assert (got.pick == 17).all() and (got.pick_logprob == 0).all()


def test_targets_out_of_range(cuda):
    rng, x, w = _inputs(cuda, 3, 64, 600, seed=5)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = ops.vocab_scores(x, w, target=torch.tensor([5, 600, -3], dtype=torch.int32, device=cuda), status=status)
    assert int(status) == 2 and torch.isnan(got.logprob).tolist() == [False, True, False] and got.logprob[2] == 0


def test_draws_follow_the_distribution(cuda):
    w = torch.zeros((8, 8), device=cuda).bfloat16()
    w[:, 0] = torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0, 0.25, 1.5, 3.0])
    x = torch.zeros((20000, 8), device=cuda).bfloat16()
    x[:, 0] = 1
    got = ops.vocab_scores(x, w, temperature=2.0, seed=123)
    p = torch.softmax(w[:, 0].float() / 2, 0)
    share = torch.bincount(got.pick, minlength=8).float() / 20000
    assert ((share - p).abs() < 5 * (p * (1 - p) / 20000).sqrt()).all()      # five standard deviations


def test_a_graph_draws_anew_with_the_seed_in_memory(cuda):
    rng, x, w = _inputs(cuda, 20, 128, 4000, seed=6, sure=False)
    seed = torch.zeros(1, dtype=torch.int32, device=cuda)
    call = ops.VocabScores(x, w, temperature=1.5, seed=seed)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    seen = []
    for s in (1, 2, -3):
        seed.fill_(s)
        g.replay()
        seen.append(call.result.pick.clone())
        assert call.result.pick.equal(ops.vocab_scores(x, w, temperature=1.5, seed=s).pick)
    assert not seen[0].equal(seen[1])


def test_twice_and_two_at_once(cuda):
    rng, x, w = _inputs(cuda, 300, 512, 20000, seed=7)
    calls = [ops.VocabScores(x, w, temperature=0.9, seed=1) for _ in range(2)]
    want = [r.clone() for r in calls[0]() if r is not None]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c()
    torch.cuda.synchronize()
    for c in calls:
        assert all(a.equal(b) for a, b in zip(want, [r for r in c.result if r is not None]))


@pytest.mark.parametrize("rows", [3, 100, 300])
def test_the_only_token_is_picked_whatever_its_noise(cuda, rows):
    """h of (this seed, row 0, token 5) is 2^32 - 94, which rounds to 2^32."""
    rng, x, w = _inputs(cuda, rows, 64, 700, seed=4)
    bias = torch.full((700,), -math.inf, device=cuda)
    bias[5] = 0
    got = ops.vocab_scores(x, w, bias=bias, temperature=1.0, seed=23192014)
    assert (got.pick == 5).all() and (got.pick_logprob.abs() < 1e-5).all()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("rows", [3, 100, 300])
def test_no_token_is_left(cuda, rows, temperature):
    """A bias of -inf everywhere: lse -inf, and a pick, the first token, that has no log-probability."""
    rng, x, w = _inputs(cuda, rows, 64, 700, seed=4)
    bias = torch.full((700,), -math.inf, device=cuda)
    target = torch.full((rows,), 5, dtype=torch.int32, device=cuda)
    got = ops.vocab_scores(x, w, bias=bias, target=target, temperature=temperature)
    assert (got.lse == -math.inf).all() and (got.pick == 0).all() and got.pick_logprob.isnan().all() and got.logprob.isnan().all()


@pytest.mark.parametrize("rows", [3, 100, 300])
def test_waits_that_run_out(cuda, rows):
    """The rows of every CTA's first stage are never asked for: code 3, and the GPU stays usable."""
    rng, x, w = _inputs(cuda, rows, 256, 3000, seed=9)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    lib = gptrs_b200.lib()
    lib.gptrs_cuda_debug_prefill_tc_fault(1, 500)
    try:
        ops.vocab_scores(x, w, status=status)
        torch.cuda.synchronize()
    finally:
        lib.gptrs_cuda_debug_prefill_tc_fault(0, 0)
    assert int(status) == 3
    status.zero_()
    _check(ops.vocab_scores(x, w, status=status), x, w, None)
    assert int(status) == 0


@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("rows", [3, 16, 100, 300])
def test_tokens_that_are_nearly_certain_keep_their_digits(cuda, rows, temperature):
    """One token of a row has all but 1e-7 to 1e-4 of the probability, lse is about 20. log p = z - m - log1p(rest), rest the sum of the others' exp(z - m): differences of logits are off by 2 e,
    an exponential's argument (below 32) by two roundings, and the exponential itself by 2^-21, all of it relative to rest / (1 + rest) = 1 - p. The last two steps round the result."""
    rng = np.random.default_rng(rows)
    dim, vocab = 512, 1200
    x, w = rng.normal(0, 1, (rows, dim)), rng.normal(0, dim ** -0.5, (vocab, dim))
    sure, size = rng.permutation(vocab)[:rows], np.log(vocab * np.exp(0.5)) - rng.uniform(np.log(1e-7), np.log(1e-4), rows)
    w[sure] = x * (size / (x * x).sum(-1))[:, None]
    x, w = (torch.tensor(v, dtype=torch.float32).bfloat16().to(cuda) for v in (x, w))
    target = np.where(rng.random(rows) < 0.5, sure, rng.integers(0, vocab, rows))
    got = ops.vocab_scores(x, w, target=torch.tensor(target, dtype=torch.int32, device=cuda), temperature=temperature, seed=9)
    z, mass = tr.logits(_np(x), _np(w))
    e = ((dim / 16 + 8) * 2 ** -23 * mass).max(-1)
    assert (z.argmax(-1) == sure).all()
    for lp, at in ((got.logprob, target), (got.pick_logprob, got.pick.cpu().numpy())):
        apart = np.exp(z - z[np.arange(rows), at][:, None])
        apart[np.arange(rows), at] = 0
        rest = apart.sum(-1)
        want, others = -np.log1p(rest), rest / (1 + rest)
        assert (np.abs(_np(lp) - want) <= others * (2 * e + 2 ** -20 + 32 * 2 ** -23) + 2 ** -22 * np.abs(want)).all()
    assert (got.pick.cpu().numpy() == sure).mean() > 0.9


@pytest.mark.parametrize("temperature,logit", [(0.3, 21.25), (1.3e-3, 21.25), (1.7e-6, 17.625), (1.1e-6, 21.25), (7e-7, 17.625), (1e-12, 3.296875)])
def test_draws_do_not_depend_on_how_many_rows_a_call_has(cuda, temperature, logit):
    """Logits without an error, most of them equal. At a small temperature z / T is so large that the noise is worth a few steps of f32: the value z / T + g is rounded alike whichever way a call
    goes, and the first of the largest is taken."""
    x, w = torch.zeros((300, 16), device=cuda).bfloat16(), torch.zeros((60000, 16), device=cuda).bfloat16()
    x[:, 0] = 1
    w[:, 0] = logit
    w[::9, 0] = -5.5
    for seed in range(60):
        few, some, many = (ops.vocab_scores(x[:rows], w, temperature=temperature, seed=seed).pick[:16] for rows in (16, 100, 300))
        assert few.equal(some) and few.equal(many)


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("rows", [3, 100, 300])
def test_tokens_that_a_bias_leaves_out_stay_out_under_a_cap(cuda, rows, temperature):
    rng, x, w = _inputs(cuda, rows, 64, 700, seed=rows)
    bias = rng.normal(0, 1, 700)
    bias[rng.permutation(700)[:650]] = -np.inf
    target = rng.integers(0, 700, rows)
    bias, t = torch.tensor(bias, dtype=torch.float32, device=cuda), torch.tensor(target, dtype=torch.int32, device=cuda)
    got = ops.vocab_scores(x, w, target=t, bias=bias, soft_cap=3.0, temperature=temperature, seed=8)
    _check(got, x, w, target, bias=bias, cap=3.0, temperature=temperature, seed=8)
    assert torch.isfinite(bias[got.pick.long()]).all() and (got.logprob == -math.inf).equal(bias[t.long()] == -math.inf)
    got = ops.vocab_scores(x, w, target=t, bias=torch.full_like(bias, -math.inf), soft_cap=3.0, temperature=temperature)
    assert (got.lse == -math.inf).all() and (got.pick == 0).all() and got.logprob.isnan().all()


@pytest.mark.parametrize("rows,dim,vocab", [(129, 520, 700), (140, 1024, 3001), (300, 1032, 700), (257, 2048, 999), (300, 2368, 2000), (140, 3080, 500), (300, 4104, 1500), (520, 5120, 600),
                                            (129, 8192, 300), (100, 4104, 1500), (17, 8192, 300), (16, 5120, 600)])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_several_accumulators_to_a_tile(cuda, rows, dim, vocab, temperature):
    """More of dim than an accumulator adds up, with a remainder and without, and the longer accumulators that draws have at a tile's beginning."""
    rng, x, w = _inputs(cuda, rows, dim, vocab, seed=dim)
    target = rng.integers(0, vocab, rows)
    got = ops.vocab_scores(x, w, target=torch.tensor(target, dtype=torch.int32, device=cuda), temperature=temperature, seed=31)
    _check(got, x, w, target, temperature=temperature, seed=31)


@pytest.mark.parametrize("rows", [1, 16, 100])
@pytest.mark.parametrize("dim", [2048, 4096])
def test_sums_are_read_out_every_128_of_dim(cuda, rows, dim):
    """Products of one sign, one token, so that lse is its logit. An accumulator cuts each of its eight sums S j / 8 by at most a step of f32, half of one on the average, so 2^-24 (1 + ... + 8) / 8
    = 4.5 2^-24 of the logit; what is added in f32 is rounded either way. Five standard deviations of the mean on top (a logit's: below 2 2^-24)."""
    low, n = 0.0, 3200 // rows
    gen = torch.Generator(device=cuda).manual_seed(rows)
    for _ in range(n):
        x, w = (torch.randn((k, dim), device=cuda, generator=gen).abs().bfloat16() for k in (rows, 1))
        z = (x.double() @ w.double().t())[:, 0]
        low += float(((z - ops.vocab_scores(x, w).lse.double()) / z).mean()) / n
    assert abs(low) <= (4.5 + 5 * 2 / (n * rows) ** 0.5) * 2 ** -24


def test_many_tiles_of_several_accumulators(cuda):
    """Several row tiles and tiles of tokens to a pair of CTAs, each of several accumulators. Logits are multiples of 2^-8 that f32 holds, so they are without an error, and lse is off by its own
    rounding and that of m, 2^-23 lse (below 32), and by the exponentials', 2^-20."""
    rng, x, w = _inputs(cuda, 530, 2568, 60000, seed=41)
    x, w = (x * 4).round() / 4, (w * 64).round() / 64                       # products and sums without an error
    for temperature in (0.0, 0.9):
        got = ops.vocab_scores(x, w, temperature=temperature, seed=5)
        z = (x.double() @ w.double().t()).float()
        assert (got.lse - z.double().logsumexp(-1)).abs().max() < 32 * 2 ** -23 + 2 ** -20
        few = ops.vocab_scores(x[:16], w, temperature=temperature, seed=5)
        assert got.pick[:16].equal(few.pick)
        if temperature == 0:
            first = torch.where(z == z.amax(-1, keepdim=True), torch.arange(60000, device=cuda), 60000).amin(-1)
            assert got.pick.equal(first.int())


@pytest.mark.parametrize("rows,vocab", [(2, 30), (17, 33), (128, 4096), (129, 100), (700, 12345), (1300, 64), (2500, 999)])
def test_however_it_is_cut(cuda, rows, vocab):
    rng, x, w = _inputs(cuda, rows, 80, vocab, seed=rows)
    target = rng.integers(0, vocab, rows)
    t = torch.tensor(target, dtype=torch.int32, device=cuda)
    for temperature in (0.0, 1.0):
        call = ops.VocabScores(x, w, target=t, temperature=temperature, seed=3)
        got = [r.clone() for r in call()]
        _check(call.result, x, w, target, temperature=temperature, seed=3)
        assert all(a.equal(b) for a, b in zip(got, call()))


def test_a_step_of_speculative_decoding(cuda):
    """Append, attention, scores, acceptance, as a serving loop has them, against the oracle; then the next step's cache."""
    from tests.test_tree_gpu import DIM, PAGE, Trees, bushy
    rng = np.random.default_rng(21)
    heads, kv, vocab = 8, 2, 500
    t = Trees(cuda, heads, kv, [(37, bushy(12, rng, 3)), (90, bushy(20, rng, 4)), None, (5, [-1])], seed=5)
    qkv = torch.tensor(rng.normal(0, 1, (t.rows, (heads + 2 * kv) * DIM)), dtype=torch.float32).bfloat16().to(cuda)
    ang = rng.uniform(-4, 4, (130, DIM // 2))
    cos, sin = (torch.tensor(f(ang), dtype=torch.float32, device=cuda) for f in (np.cos, np.sin))
    q = ops.tree_append(t.trees, qkv, cos, sin, t.pool, status=t.status)
    for s, f in enumerate(t.forest):
        if f is not None:
            t.kvs[s] = t.read(s, np.arange(f[0] + len(f[1])))
    out = t.attention(q)
    t.check(out, q)
    w = torch.tensor(rng.normal(0, 1, (vocab, heads * DIM)), dtype=torch.float32).bfloat16().to(cuda)
    scores = ops.vocab_scores(out, w, status=t.status)
    _check(scores, out, w, None)
    pick = scores.pick.cpu().numpy()
    token = rng.integers(0, vocab, t.rows)
    for s, f in enumerate(t.forest):
        for i, up in enumerate(f[1] if f else []):                            # half of the drafts are what the model says
            if up >= 0 and rng.random() < 0.5:
                token[t.row0[s] + i] = pick[t.row0[s] + up]
    got = ops.tree_accept(t.trees, torch.tensor(token, dtype=torch.int32, device=cuda), scores.pick, [t.pool], status=t.status)
    assert int(t.status) == 0
    for s, f in enumerate(t.forest):
        if f is None:
            assert int(got.count[s]) == 0
            continue
        a, b = t.row0[s], t.row0[s + 1]
        path, follows = tr.accept(f[1], token[a:b], pick[a:b])
        assert got.path[s, :len(path)].tolist() == path and int(got.count[s]) == len(path) and int(got.next[s]) == follows
        assert np.array_equal(t.read(s, np.arange(f[0] + len(path))), t.kvs[s][:, list(range(f[0])) + [f[0] + i for i in path]])
        assert int(got.length[s]) == f[0] + len(path)
    assert PAGE == ops.PAGE_TOKENS
