"""The 8-bit cache without a GPU: sizes, refusals (all of them in front of the first CUDA call), the byte order, and the formula that the kernels
compute the softmax with."""
import ctypes

import numpy as np
import pytest

import gptrs_b200
from gptrs_b200 import BackendError, _abi, ops
from oracle import kv8_ref as kr

SPEC, UNIMPLEMENTED = 1, 2


def _status(fn, *args):
    return getattr(gptrs_b200.lib(), fn)(*args)


def test_layout_sizes():
    a = ops.kv8_layout(32, 8, 128)
    assert (a.block_bytes, a.page_bytes, a.open_bytes, a.tile_tokens) == (4112, 8 * 4112, 2 * 8 * 2 * 16 * 128 * 2, 64)
    assert a.scale == pytest.approx(128 ** -0.5)
    a = ops.kv8_layout(12, 12, 64, window=5, scale=0.25)
    assert (a.block_bytes, a.scale, a.window, a.tile_tokens) == (2064, 0.25, 5, 256)


@pytest.mark.parametrize("heads,kv,dim,window,scale,status", [(0, 1, 64, 0, 0, SPEC), (8, 0, 64, 0, 0, SPEC), (8, 3, 64, 0, 0, SPEC), (8, 8, 64, -1, 0, SPEC), (8, 8, 64, 0, -1, SPEC),
                                                              (8, 8, 64, 0, float("nan"), SPEC), (8, 8, 80, 0, 0, UNIMPLEMENTED), (130, 2, 128, 0, 0, UNIMPLEMENTED)])
def test_layout_refusals(heads, kv, dim, window, scale, status):
    a = _abi.Kv8Cache(heads, kv, dim, window, scale)
    assert _status("gptrs_cuda_kv8_layout", ctypes.byref(a)) == status


def _rotation(**kw):
    r = _abi.QkRotation(8, 2, 64)
    r.rot_half, r.positions, r.d_cos, r.d_sin, r.d_q_gain, r.d_k_gain, r.eps = 32, 10, 4096, 4096, 4096, 4096, 1e-6
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("change,args", [
    (dict(q_heads=0), {}), (dict(dim=63), {}), (dict(dim=514), {}), (dict(rot_half=33), {}), (dict(rot_half=-1), {}), (dict(pairs=2), {}), (dict(d_k_gain=None), {}),
    (dict(d_sin=None), {}), (dict(positions=0), {}), (dict(axes=2), {}), (dict(axes=2, d_axis_positions=64), {}), (dict(axes=300, d_axis_positions=64, d_pair_axis=64), {}),
    (dict(axis_stride=3), {}), ({}, dict(qkv=None)), ({}, dict(out=None)), ({}, dict(status=None)), ({}, dict(positions=None)), ({}, dict(dtype=1)), ({}, dict(ld_in=767)),
    ({}, dict(ld_out=10)), ({}, dict(rows=-1)), ({}, dict(out=4096, ld_out=1000))])
def test_norm_rope_refusals(change, args):
    a = dict(qkv=4096, dtype=0, ld_in=0, positions=64, out=8192, ld_out=0, status=64, rows=5)
    a.update(args)
    r = _rotation(**change)
    assert _status("gptrs_cuda_qk_norm_rope", ctypes.byref(r), a["qkv"], a["dtype"], a["ld_in"], a["positions"], a["out"], a["ld_out"], a["status"], a["rows"], None) == SPEC


def _append_step(a, **kw):
    s = _abi.Kv8AppendStep()
    for n, _ in s._fields_:
        if n.startswith("d_"):
            setattr(s, n, 4096)
    s.max_pages = s.n_pages = s.n_slots = s.rows = 4
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_append_refusals():
    a = ops.kv8_layout(8, 2, 64)
    pointers = [n for n, _ in _abi.Kv8AppendStep._fields_ if n.startswith("d_")]
    for change in [{n: None} for n in pointers] + [{n: 4104} for n in ("d_qkv", "d_pool", "d_open", "d_q")] + [dict(rows=-1), dict(ld=760), dict(ld=772), dict(max_pages=0),
                                                                                                           dict(n_pages=0), dict(n_slots=0)]:
        assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(_append_step(a, **change)), None) == SPEC, change
    for change, want in [(dict(q_heads=4), SPEC), (dict(dim=128), SPEC), (dict(rot_half=30), UNIMPLEMENTED), (dict(d_cos=4100), SPEC), (dict(d_q_gain=4100), SPEC), (dict(axes=3), SPEC)]:
        r = _rotation(**change)
        assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(_append_step(a, rotation=ctypes.addressof(r))), None) == want, change
    raw = _abi.Kv8Cache(8, 2, 64)   # not filled in
    assert _status("gptrs_cuda_kv8_append", ctypes.byref(raw), ctypes.byref(_append_step(a)), None) == SPEC
    assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), None, None) == SPEC
    assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(_append_step(a, rows=0)), None) == 0


def test_targets_in_the_source_are_refused():
    """Rows are worked on in no order, so the target may lie beside or between the source's rows, not in them; rows of 768 f32 or bf16 values."""
    r, at = _rotation(), 1 << 20
    for out, ld in [(at + 4 * 4, 0), (at - 4 * 4, 0), (at + 4 * 768 * 4, 0), (at + 767 * 4, 1536), (at + 769 * 4, 1536), (at - 1000 * 4, 1536)]:
        assert _status("gptrs_cuda_qk_norm_rope", ctypes.byref(r), at, 0, ld, 64, out, ld, 64, 5, None) == SPEC, (out, ld)
        assert "lie in the source" in gptrs_b200.lib().gptrs_cuda_last_error().decode()
    a = ops.kv8_layout(8, 2, 64)
    for d_q in (4096, 4096 + 2 * 768 * 3 + 2 * 752, 4096 - 2 * 512 * 4 + 16):
        assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(_append_step(a, d_q=d_q)), None) == SPEC, d_q
        assert "queries go into rows" in gptrs_b200.lib().gptrs_cuda_last_error().decode()


def test_attention_and_gather_refusals():
    a = ops.kv8_layout(8, 2, 64)

    def step(**kw):
        s = _abi.Kv8AttentionStep()
        for n in ("d_q", "d_pool", "d_open", "d_page_table", "d_slot", "d_ctx_len", "d_length", "d_out", "d_status"):
            setattr(s, n, 4096)
        s.n_pages = s.n_slots = s.max_pages = s.rows = 4
        s.max_ctx_len, s.splits = 64, 1
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    changes = [{n: None} for n in ("d_q", "d_pool", "d_open", "d_page_table", "d_slot", "d_ctx_len", "d_length", "d_out", "d_status")]
    changes += [{n: 4104} for n in ("d_q", "d_pool", "d_open", "d_out")]
    changes += [dict(rows=-1), dict(n_tiles=-1), dict(n_tiles=1), dict(n_tiles=1, d_tile_row=64), dict(max_pages=0), dict(max_pages=1 << 28), dict(n_pages=0), dict(n_slots=0), dict(n_slots=1 << 31),
                dict(max_ctx_len=-1), dict(max_ctx_len=1 << 31), dict(splits=0), dict(splits=1 << 17), dict(ldq=504), dict(ldq=513), dict(splits=9),
                dict(splits=9, d_scratch=4096, scratch_bytes=16), dict(splits=2, n_tiles=1, d_tile_row=64, d_tile_rows=64)]
    for change in changes:
        assert _status("gptrs_cuda_kv8_attention", ctypes.byref(a), ctypes.byref(step(**change)), None) == SPEC, change
    assert _status("gptrs_cuda_kv8_attention", ctypes.byref(a), ctypes.byref(step(rows=0)), None) == 0
    good = [ctypes.byref(a), 4096, 4, 4096, 4, 4096, 4, 4096, 4096, 4096, 2, 4096, 4096, 4096, 4, None]
    for at, bad in [(1, None), (1, 4104), (2, 0), (3, None), (4, 0), (5, None), (6, 0), (7, None), (8, None), (9, None), (10, 1), (11, None), (12, 8), (13, None), (14, -1)]:
        args = list(good)
        args[at] = bad
        assert _status("gptrs_cuda_kv8_gather", *args) == SPEC, (at, bad)


def test_calls_without_rows_need_no_rows():
    """Empty tensors have no address: a call without rows does nothing, and still refuses what is wrong with the rest."""
    a = ops.kv8_layout(8, 2, 64)
    r = _rotation(axes=2, d_pair_axis=64)
    assert _status("gptrs_cuda_qk_norm_rope", ctypes.byref(r), None, 0, 0, None, None, 0, 64, 0, None) == 0
    s = _append_step(a, rows=0, **{n: None for n in ("d_qkv", "d_positions", "d_slot", "d_run_first", "d_run_last", "d_q")})
    assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(s), None) == 0
    t = _abi.Kv8AttentionStep()
    for n in ("d_pool", "d_open", "d_page_table", "d_length", "d_status"):
        setattr(t, n, 4096)
    t.n_pages = t.n_slots = t.max_pages = 4
    t.max_ctx_len, t.splits = 64, 1
    assert _status("gptrs_cuda_kv8_attention", ctypes.byref(a), ctypes.byref(t), None) == 0
    assert _status("gptrs_cuda_kv8_gather", ctypes.byref(a), 4096, 4, 4096, 4, 4096, 4, None, None, 4096, 2, None, None, 4096, 0, None) == 0
    s.d_pool = t.d_pool = None
    assert _status("gptrs_cuda_kv8_append", ctypes.byref(a), ctypes.byref(s), None) == SPEC
    assert _status("gptrs_cuda_kv8_attention", ctypes.byref(a), ctypes.byref(t), None) == SPEC
    assert _status("gptrs_cuda_qk_norm_rope", ctypes.byref(_rotation(dim=63)), None, 0, 0, None, None, 0, 64, 0, None) == SPEC


def test_outputs_in_the_queries_are_refused():
    """Rows are worked on in no order: the output may be the packed queries themselves (which this test leaves alone) or lie beside them."""
    a, at = ops.kv8_layout(8, 2, 64), 1 << 20
    for out, ldq in [(at + 16, 0), (at - 16, 0), (at + 1024 * 2, 512), (at - 1024 * 2 - 1008, 0), (at, 768), (at + 1024, 1024), (at + 3 * 1536 + 1008, 768)]:
        s = _abi.Kv8AttentionStep()
        for n in ("d_pool", "d_open", "d_page_table", "d_slot", "d_ctx_len", "d_length", "d_status"):
            setattr(s, n, 4096)
        s.n_pages = s.n_slots = s.max_pages = s.rows = 4
        s.max_ctx_len, s.splits, s.d_q, s.d_out, s.ldq = 64, 1, at, out, ldq
        assert _status("gptrs_cuda_kv8_attention", ctypes.byref(a), ctypes.byref(s), None) == SPEC, (out, ldq)
        assert "rows of other queries" in gptrs_b200.lib().gptrs_cuda_last_error().decode()


def test_objects_refuse_wrong_tensors():
    """Shapes and types are looked at in front of the device."""
    import torch
    a = ops.kv8_layout(8, 2, 64)
    pool, rows, table = ops.new_kv8_pool(a, 3, "cpu"), ops.new_kv8_open(a, 2, "cpu"), torch.zeros((2, 4), dtype=torch.int32)
    qkv, ints = torch.zeros((5, 768), dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.Kv8Append(a, None, qkv, ints, ints, ints, ints, table, pool, rows)
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :700]), dict(slot=ints.long()), dict(pool=pool[:, :1]), dict(rows=rows.float()), dict(table=table[:1])):
        x = dict(qkv=qkv, slot=ints, pool=pool, rows=rows, table=table) | bad
        with pytest.raises(ValueError, match="expected"):
            ops.Kv8Append(a, None, x["qkv"], ints, x["slot"], ints, ints, x["table"], x["pool"], x["rows"])
    with pytest.raises(ValueError, match="q: expected"):
        ops.Kv8Attention(a, torch.zeros((5, 8, 128), dtype=torch.bfloat16), pool, rows, table, ints, ints, ints[:2], 64)
    with pytest.raises(ValueError, match="axis_positions"):
        ops.QkNormRope(ops.QkRotation(8, 2, 64, axis_positions=torch.zeros((1, 4), dtype=torch.int32)), qkv, ints)


def test_parts_and_scratch():
    """Scratch is asked for where parts are more than a wave or more than a cluster holds; nothing is computed from heads that are none."""
    a, lib = ops.kv8_layout(32, 8, 128), gptrs_b200.lib()
    parts = lambda rows, n_tiles, longest: lib.gptrs_cuda_kv8_splits(ctypes.byref(a), rows, n_tiles, longest)
    assert parts(0, 0, 100) == 1 and parts(1, 0, 0) == 1 and parts(1, 0, 17) == 1 and parts(1, 0, 1000) == 8 and parts(4096, 0, 131072) == 1
    for rows, longest in [(1, 100), (1, 1 << 20), (7, 5000), (64, 8192), (64, 300), (300, 131072), (70000, 4000)]:
        n = parts(rows, 0, longest)
        size = lib.gptrs_cuda_kv8_scratch_bytes(ctypes.byref(a), rows, 0, n)
        assert 1 <= n <= 65535 and size in (0, rows * 32 * n * 130 * 4) and (size == 0 if n == 1 else size > 0 if n > 8 else True)
    assert lib.gptrs_cuda_kv8_scratch_bytes(ctypes.byref(a), 1, 0, 8) == 0 and lib.gptrs_cuda_kv8_scratch_bytes(ctypes.byref(a), 64, 0, 8) == 64 * 32 * 8 * 130 * 4
    for bad in (_abi.Kv8Cache(0, 0, 128), _abi.Kv8Cache(4, 0, 128), _abi.Kv8Cache(1, 2, 128)):
        assert lib.gptrs_cuda_kv8_splits(ctypes.byref(bad), 5, 0, 1000) == 1 and lib.gptrs_cuda_kv8_scratch_bytes(ctypes.byref(bad), 5, 0, 4) == 0


def test_tiles():
    a = ops.kv8_layout(32, 8, 128)
    first, n = ops.kv8_tiles(a, [1, 64, 0, 130], "cpu")
    assert first.tolist() == [0, 1, 65, 129, 193] and n.tolist() == [1, 64, 64, 64, 2]


def test_every_byte_of_a_block_has_one_place():
    for dim in (64, 128):
        k = {d // 32 * 512 + t % 8 * 64 + d % 32 // 8 * 16 + t // 8 * 8 + d % 8 for t in range(16) for d in range(dim)}
        v = {d // 32 * 512 + d % 8 * 64 + t % 8 // 2 * 16 + d % 32 // 8 * 4 + t // 8 * 2 + t % 2 for t in range(16) for d in range(dim)}
        assert k == v == set(range(16 * dim))


def test_scales_in_the_exponent():
    """sum w b / sum (w / s) with w = 2^(t + log2 s - M) is the softmax of the values s b, for scales that differ by many powers of two."""
    rng = np.random.default_rng(0)
    s, b = 2.0 ** rng.uniform(-50, 50, 40), rng.integers(-127, 128, (40, 16, 8)).astype(float)
    t = rng.normal(0, 30, (40, 16)) - np.log2(s)[:, None] * (rng.random((40, 1)) < 0.5)
    e = t + np.log2(s)[:, None]
    w = 2.0 ** (e - e.max())
    got = np.einsum("it,itd->d", w, b) / (w / s[:, None]).sum()
    p = 2.0 ** (t - t.max())
    want = np.einsum("it,itd->d", p, b * s[:, None, None]) / p.sum()
    assert np.allclose(got, want, rtol=1e-9, atol=1e-12 * np.abs(want).max())


def test_quantised_once_whatever_the_cuts():
    rng = np.random.default_rng(1)
    k, v = (kr.to_bf16(rng.normal(size=(50, 2, 64))) for _ in range(2))
    one, many = kr.Sequence(2, 64), kr.Sequence(2, 64)
    one.append(0, k, v)
    for at in range(0, 50, 7):
        many.append(at, k[at:at + 7], v[at:at + 7])
    for x, y in zip(one.held(), many.held()):
        assert np.array_equal(x, y)
    held = one.held()[0]
    step = np.abs(k[:48].reshape(3, 16, 2, 64)).max((1, 3)) / 127
    # half a step, and what f32 adds: the scale is off by 2^-24 of itself, which 127 of them make 2^-17 steps, and so may the quotient be
    assert (np.abs(held[:48] - k[:48]).reshape(3, 16, 2, 64).max((1, 3)) <= (0.5 + 2 * 2 ** -17) * step).all() and np.array_equal(held[48:], k[48:])


def test_refusal_reaches_python():
    with pytest.raises(BackendError, match="64 and 128 channels"):
        ops.kv8_layout(4, 4, 32)
