"""Pointers that miss their natural alignment are refused by the C entry points: a kernel that read through one would fault.  Addresses are looked at
only."""

from __future__ import annotations

import ctypes

import pytest

ALIGN = -4


def _point(a, where, value):
    *path, name = where.split(".")
    for part in path:
        a = getattr(a, part)
    kind = dict(type(a)._fields_)[name]
    setattr(a, name, value if kind is ctypes.c_void_p else ctypes.cast(ctypes.c_void_p(value), kind))


def _delta(io=1):
    from ssm_b200 import _lib

    g = _lib.GatedDeltaBwdArgs()
    a = g.fwd
    a.batch, a.len, a.heads, a.key_heads, a.kdim, a.vdim, a.io_dtype, a.g_dtype, a.num_seqs, a.cu_is_64 = 1, 4, 2, 1, 8, 8, io, 0, 1, 1
    a.q_sh = a.k_sh = a.v_sh = 8
    a.q_st = a.k_st = a.v_st = 16
    a.q_sb = a.k_sb = a.v_sb = 64
    for name in ("q", "k", "v", "g", "beta", "cu_seqlens", "initial_state", "o", "final_state", "table", "rest", "states"):
        _point(a, name, 4096)
    for name, _ in type(g)._fields_[1:]:
        _point(g, name, 4096)
    return g


@pytest.mark.parametrize("where,off", [("fwd.q", 1), ("fwd.k", 1), ("fwd.v", 1), ("fwd.g", 2), ("fwd.beta", 2), ("fwd.cu_seqlens", 4), ("fwd.initial_state", 2), ("fwd.o", 1),
                                       ("fwd.final_state", 2), ("fwd.table", 2), ("fwd.rest", 2), ("fwd.states", 1), ("dout", 1), ("dfinal", 2), ("dq", 1), ("dk", 1), ("dv", 1),
                                       ("dg", 2), ("dbeta", 2), ("dinitial", 2), ("dv32", 2), ("dstates", 2), ("dqk", 2)])
def test_gated_delta(where, off):
    from ssm_b200 import _lib

    lib = _lib.load()
    g = _delta()
    _point(g, where, 4096 + off)
    if where.startswith("fwd."):
        assert lib.ssm_gated_delta_fwd(ctypes.byref(g.fwd), None) == ALIGN
    assert lib.ssm_gated_delta_bwd(ctypes.byref(g), None) == ALIGN
    if where in ("dg", "dbeta", "dinitial"):
        assert lib.ssm_gated_delta_chunked_bwd(ctypes.byref(g), 4096, 4096, None, None) == ALIGN


def test_gated_delta_scratch_and_status():
    from ssm_b200 import _lib

    lib = _lib.load()
    g = _delta()
    for scratch, kept, status in ((4097, 4096, None), (4096, 4224, None), (4096, 4096, 4098)):
        assert lib.ssm_gated_delta_chunked_fwd(ctypes.byref(g.fwd), scratch, kept, 0, status, None) == ALIGN
        assert lib.ssm_gated_delta_chunked_bwd(ctypes.byref(g), kept, scratch, status, None) == ALIGN


@pytest.mark.parametrize("where,off", [("state", 2), ("q", 1), ("k", 1), ("v", 1), ("g", 2), ("beta", 2), ("o", 1)])
def test_step(where, off):
    from ssm_b200 import _lib

    a = _lib.GatedDeltaStepArgs()
    a.batch, a.heads, a.key_heads, a.kdim, a.vdim, a.io_dtype = 1, 2, 1, 8, 8, 1
    for name in ("state", "q", "k", "v", "g", "beta", "o"):
        _point(a, name, 4096)
    _point(a, where, 4096 + off)
    assert _lib.load().ssm_gated_delta_step(ctypes.byref(a), None) == ALIGN


@pytest.mark.parametrize("where,off", [("fwd.logits", 1), ("fwd.targets", 4), ("fwd.logp", 2), ("fwd.entropy", 2), ("fwd.top_logp", 2), ("fwd.top_ids", 4), ("fwd.stats", 8), ("dlogp", 2),
                                       ("dentropy", 2), ("dtop_logp", 2), ("dlogits", 1)])
def test_token_log_probs(where, off):
    from ssm_b200 import _lib

    lib = _lib.load()
    g = _lib.TokenLogpBwdArgs()
    a = g.fwd
    a.rows, a.row_stride, a.vocab, a.io_dtype, a.top_k, a.temperature = 2, 8, 8, 1, 2, 1.0
    for name in ("logits", "targets", "logp", "entropy", "top_logp", "top_ids", "stats"):
        _point(a, name, 4096)
    for name in ("dlogp", "dentropy", "dtop_logp", "dlogits"):
        _point(g, name, 4096)
    _point(g, where, 4096 + off)
    if where.startswith("fwd."):
        assert lib.ssm_token_logp(ctypes.byref(a), None) == ALIGN
    assert lib.ssm_token_logp_bwd(ctypes.byref(g), None) == ALIGN


@pytest.mark.parametrize("where,off", [("fwd.logits", 1), ("fwd.teacher", 2), ("fwd.ids", 4), ("fwd.loss", 2), ("fwd.stats", 8), ("dloss", 2), ("dlogits", 1)])
def test_distillation(where, off):
    from ssm_b200 import _lib

    lib = _lib.load()
    g = _lib.TopkDistillBwdArgs()
    a = g.fwd
    a.rows, a.row_stride, a.vocab, a.io_dtype, a.top_k, a.teacher_dtype, a.temperature = 2, 8, 8, 1, 2, 0, 1.0
    for name in ("logits", "teacher", "ids", "loss", "stats"):
        _point(a, name, 4096)
    for name in ("dloss", "dlogits"):
        _point(g, name, 4096)
    _point(g, where, 4096 + off)
    if where.startswith("fwd."):
        assert lib.ssm_topk_distill(ctypes.byref(a), None) == ALIGN
    assert lib.ssm_topk_distill_bwd(ctypes.byref(g), None) == ALIGN
