"""Trees of drafted tokens and scores against a vocabulary: what the calls refuse, on the CPU, and the oracle's own checks."""
import ctypes

import numpy as np
import pytest
import torch

import gptrs_b200
from gptrs_b200 import _abi, ops
from oracle import tree_ref as tr

OK, REFUSED = 0, 1


def _trees(**kw):
    t = _abi.DraftTrees(8, 2, 128, 16, 0.0, 16, 16, 16, 16, 2, 20, 16, 3, 10, 50)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _calls():
    lib = gptrs_b200.lib()
    append = _abi.TreeAppendStep(1 << 20, 0, 16, 16, 128, 40, 1 << 24, 16, 16)
    attend = _abi.TreeAttentionStep(1 << 20, 0, 16, 1 << 24, 16, 1 << 40, 16)
    accept = _abi.TreeAcceptStep(16, 16, 16, 2, 16, 16, 16, 1 << 20, 16)
    return [(lib.gptrs_cuda_tree_append, append), (lib.gptrs_cuda_tree_attention, attend), (lib.gptrs_cuda_tree_accept, accept)]


@pytest.mark.parametrize("bad", [dict(dim=64), dict(q_heads=7), dict(kv_heads=0), dict(q_heads=66), dict(max_nodes=0), dict(max_nodes=257), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(n_trees=-1), dict(n_trees=65536), dict(rows=-1), dict(rows=513), dict(d_first=None), dict(d_slot=None), dict(d_length=None), dict(d_parent=None),
                                 dict(d_page_table=None), dict(max_pages=0), dict(max_pages=1 << 27), dict(n_slots=0), dict(n_pages=0)])
def test_trees_are_checked(bad):
    for fn, step in _calls():
        assert fn(ctypes.byref(_trees(**bad)), ctypes.byref(step), None) == REFUSED


@pytest.mark.parametrize("call,bad", [(0, dict(d_qkv=None)), (0, dict(d_q=None)), (0, dict(d_pool=None)), (0, dict(d_status=None)), (0, dict(d_cos=None)), (0, dict(rotary_dim=120)),
                                      (0, dict(rotary_dim=144)), (0, dict(rotary_dim=-16)), (0, dict(positions=0)), (0, dict(ld=1528)), (0, dict(ld=1540)), (0, dict(d_qkv=(1 << 20) + 8)),
                                      (0, dict(d_q=(1 << 20) + 4096)), (0, dict(d_cos=8)),
                                      (1, dict(d_q=None)), (1, dict(d_out=None)), (1, dict(d_pool=None)), (1, dict(d_status=None)), (1, dict(ldq=1016)), (1, dict(ldq=1028)),
                                      (1, dict(d_q=(1 << 20) + 2)), (1, dict(d_out=1 << 20)), (1, dict(d_out=(1 << 20) + 2048)),
                                      (2, dict(d_token=None)), (2, dict(d_pick=None)), (2, dict(d_status=None)), (2, dict(d_count=None)), (2, dict(d_path=None)), (2, dict(d_next=None)),
                                      (2, dict(d_new_length=None)), (2, dict(d_new_length=16)), (2, dict(d_new_length=20)), (2, dict(n_layers=-1)), (2, dict(d_pools=None))])
def test_steps_are_checked(call, bad):
    fn, step = _calls()[call]
    for k, v in bad.items():
        setattr(step, k, v)
    assert fn(ctypes.byref(_trees()), ctypes.byref(step), None) == REFUSED
    assert gptrs_b200.lib().gptrs_cuda_last_error()


def test_scratch_is_checked():
    fn, step = _calls()[1]
    long = _trees(max_pages=4000)
    need = gptrs_b200.lib().gptrs_cuda_tree_scratch_bytes(ctypes.byref(long))
    assert need > 0 and gptrs_b200.lib().gptrs_cuda_tree_scratch_bytes(ctypes.byref(_trees())) == 0   # short contexts need none
    for bad in (dict(d_scratch=None), dict(scratch_bytes=need - 1), dict(d_scratch=8)):
        step = _abi.TreeAttentionStep(1 << 20, 0, 16, 1 << 24, 16, need, 16)
        for k, v in bad.items():
            setattr(step, k, v)
        assert fn(ctypes.byref(long), ctypes.byref(step), None) == REFUSED
    assert gptrs_b200.lib().gptrs_cuda_tree_scratch_bytes(None) == 0


def test_calls_without_rows_do_nothing():
    for fn, step in _calls()[:2]:
        assert fn(ctypes.byref(_trees(rows=0, d_parent=None)), ctypes.byref(step), None) == OK
    fn, step = _calls()[2]
    assert fn(ctypes.byref(_trees(rows=0, n_trees=0)), ctypes.byref(step), None) == OK


def test_null_arguments_are_refused():
    for fn, step in _calls():
        assert fn(None, ctypes.byref(step), None) == REFUSED and fn(ctypes.byref(_trees()), None, None) == REFUSED
    assert gptrs_b200.lib().gptrs_cuda_vocab_scores(None, None) == REFUSED


def _scores(**kw):
    s = _abi.VocabScores(16, 0, 16, 0, 4, 64, 100, None, 0.0, 0.0, 0, None, 16, 16, 16, 16, 16, 32, 1 << 40, 16)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("bad", [dict(d_hidden=None), dict(d_weight=None), dict(d_status=None), dict(rows=-1), dict(vocab=0), dict(dim=0), dict(dim=12), dict(ldh=56), dict(ldh=68),
                                 dict(ldw=56), dict(ldw=66), dict(d_hidden=8), dict(d_weight=24), dict(d_scratch=None), dict(d_scratch=8), dict(scratch_bytes=1), dict(d_target=None),
                                 dict(soft_cap=-1.0), dict(soft_cap=float("nan")), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-30)])
def test_scores_are_checked(bad):
    assert gptrs_b200.lib().gptrs_cuda_vocab_scores(ctypes.byref(_scores(**bad)), None) == REFUSED


def test_scores_without_rows_do_nothing():
    assert gptrs_b200.lib().gptrs_cuda_vocab_scores(ctypes.byref(_scores(rows=0, d_hidden=None)), None) == OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="what a call does where kernels cannot be asked for their registers")
def test_scores_are_not_launched_before_their_registers_are_known():
    """The kernel's warps share out the registers that it was compiled for, and would wait without end for more than there are."""
    lib = gptrs_b200.lib()
    for rows in (4, 100, 300):
        assert lib.gptrs_cuda_vocab_scores(ctypes.byref(_scores(rows=rows)), None) not in (OK, REFUSED)
        assert b"registers" in lib.gptrs_cuda_last_error()


def test_python_checks_its_tensors():
    ints = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table = torch.zeros((2, 4), dtype=torch.int32)
    good = (4, 2, ints(0, 3), ints(0), ints(5), ints(-1, 0, 0), table, 8)
    pool = torch.zeros(2 * ops.kv_pool_bytes(1, 2), dtype=torch.uint8)
    t = ops.DraftTrees(*good)
    assert (t.over(pool).n_pages, t.rows, t.n_trees) == (2, 3, 1)
    for i, bad in ((2, ints(0)), (3, torch.zeros(1)), (4, ints(1, 2)), (5, torch.zeros(3)), (6, ints(0))):
        with pytest.raises(ValueError):
            ops.DraftTrees(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError):
        t.over(pool[:-16])
    with pytest.raises(ValueError):
        ops.TreeAppend(t, torch.zeros((2, 8 * 128), dtype=torch.bfloat16), None, None, pool)
    with pytest.raises(ValueError):
        ops.TreeAttention(t, torch.zeros((3, 4, 128)), pool)
    with pytest.raises(ValueError):
        ops.TreeAccept(t, ints(1, 2, 3), ints(1, 2, 3), [pool, pool])
    with pytest.raises(ValueError):
        ops.TreeAccept(t, ints(1, 2, 3), ints(1, 2, 3), [pool, pool[:pool.numel() // 2]])
    with pytest.raises(ValueError):
        ops.VocabScores(torch.zeros((2, 16)), torch.zeros((9, 16), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.TreeAttention(t, torch.zeros((3, 4, 128), dtype=torch.bfloat16), pool)   # not on a GPU


def test_oracle_walks():
    assert tr.ancestors([-1, 0, 0, 1, 3, -1]) == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [5]]
    assert tr.accept([-1, 0, 0, 1, 2, 2], [7, 4, 4, 5, 5, 6], [4, 5, 6, 9, 1, 2]) == ([0, 1, 3], 9)   # the first of two children with one token
    assert tr.accept([], [], []) == ([], -1)
    g = tr.noise(3, 50, 400)
    assert abs(g.mean() - 0.5772) < 0.05 and abs(g.var() - np.pi ** 2 / 6) < 0.1 and not np.isnan(g).any()
