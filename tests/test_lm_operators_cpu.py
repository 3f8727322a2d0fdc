"""The operators beside the state-space ones, without a GPU: their definitions against differences, the C structs' layout, refusals."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import lm_oracle

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "ssm_b200_lm.h"


def _delta_inputs(nb, nl, nk, nh, kd, vd, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    return [unit(rn(nb, nl, nk, kd)), unit(rn(nb, nl, nk, kd)), rn(nb, nl, nh, vd), -rn(nb, nl, nh).abs(), torch.sigmoid(rn(nb, nl, nh))]


def test_gradients_of_the_definitions_are_those_of_differences():
    leaves = [t.requires_grad_(True) for t in _delta_inputs(2, 5, 1, 2, 3, 2)]
    init = torch.randn(2, 2, 2, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *a: lm_oracle.gated_delta(*a[:5], None, a[5]), (*leaves, init))
    gen = torch.Generator().manual_seed(2)
    logits = (2 * torch.randn(3, 7, generator=gen, dtype=torch.float64)).requires_grad_(True)
    targets = torch.tensor([2, -100, 6])
    assert torch.autograd.gradcheck(lambda x: lm_oracle.token_log_probs(x, targets, 0.7, 3)[:3], (logits,))
    ids = torch.tensor([[0, 3, 3], [1, -1, 2], [-1, -1, -1]])
    teacher = torch.randn(3, 3, generator=gen, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda x: lm_oracle.topk_distill_loss(x, teacher, ids, 2.0), (logits,))


def test_the_chunk_form_of_the_backward_is_the_recurrence_s():
    """The sums over pairs of tokens that the gradient kernel forms, for one chunk, against autograd through the recurrence."""
    nl, kd, vd = 9, 4, 3
    q, k, v, g, beta = [t.requires_grad_(True) for t in _delta_inputs(1, nl, 1, 1, kd, vd, 3)]
    gen = torch.Generator().manual_seed(4)
    s0 = torch.randn(1, 1, vd, kd, dtype=torch.float64, generator=gen).requires_grad_(True)
    do, ds = torch.randn(1, nl, 1, vd, dtype=torch.float64, generator=gen), torch.randn(1, 1, vd, kd, dtype=torch.float64, generator=gen)
    with torch.no_grad():
        g[0, 4] = -float("inf")  # a reset inside the chunk
    o, s1 = lm_oracle.gated_delta(q, k, v, g, beta, 0.5, s0)
    want = torch.autograd.grad([o, s1], [q, k, v, g, beta, s0], [do, ds])
    Q, K, V, B, D, S0, DS = 0.5 * q[0, :, 0], k[0, :, 0], v[0, :, 0], beta[0, :, 0], do[0, :, 0], s0[0, 0], ds[0, 0]
    a = torch.exp(g[0, :, 0])
    G = torch.stack([torch.stack([torch.prod(a[j + 1:i + 1]) if i >= j else a.new_zeros(()) for j in range(nl)]) for i in range(nl)])
    gam, suf = torch.cumprod(a, 0), G[-1]
    low = torch.tril(torch.ones(nl, nl, dtype=torch.float64))
    strict = torch.tril(low, -1)
    X = torch.linalg.inv(torch.eye(nl, dtype=torch.float64) + strict * G * (K @ K.T) * B[None, :])
    R = X @ (V - gam[:, None] * (K @ S0.T))
    W = X.T @ (B[:, None] * ((low * G * (Q @ K.T)).T @ D + suf[:, None] * (K @ DS.T)))
    N1, N2 = D @ R.T, W @ R.T
    D1, D2, Z = D @ S0, W @ S0, R @ DS
    dq = 0.5 * (gam[:, None] * D1 + (low * G * N1 * B) @ K)
    y = (low * G * N1).T @ Q - (strict * G * N2).T @ K + suf[:, None] * Z
    dk = B[:, None] * y - gam[:, None] * D2 - (strict * G * N2 * B) @ K
    M = strict * G * B * (N1 * (Q @ K.T) - N2 * (K @ K.T))
    dg = torch.stack([M[t:, :t].sum() + (gam * ((Q * D1).sum(-1) - (K * D2).sum(-1)))[t:].sum() + (B * suf * (K * Z).sum(-1))[:t].sum() + gam[-1] * (S0 * DS).sum()
                      for t in range(nl)])
    dinit = gam[-1] * DS + (gam[:, None] * D).T @ Q - (gam[:, None] * W).T @ K
    for got, ref in zip((dq, dk, W, dg, (K * y).sum(-1), dinit), (t.reshape(x) for t, x in zip(want, ((nl, kd), (nl, kd), (nl, vd), (nl,), (nl,), (vd, kd))))):
        finite = torch.isfinite(ref)  # autograd's own derivative of exp at -inf is 0, of the products NaN nowhere
        assert finite.all() and torch.allclose(got, ref, rtol=1e-10, atol=1e-12)


def test_header_and_ctypes_mirrors_agree(tmp_path):
    from ssm_b200 import _lib

    lib = _lib.load()
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(ssm_[a-z0-9_]+)\s*\(", text)))
    assert len(names) >= 9
    for name in names:
        assert hasattr(lib, name) and name in _lib.ENTRY_POINTS, name
    assert lib.ssm_b200_lm_abi_version() == _lib.LM_ABI_VERSION == int(re.search(r"#define SSM_B200_LM_ABI_VERSION (\d+)", text).group(1))
    pairs = {
        "ssm_gated_delta_args": _lib.GatedDeltaArgs, "ssm_gated_delta_bwd_args": _lib.GatedDeltaBwdArgs, "ssm_gated_delta_step_args": _lib.GatedDeltaStepArgs,
        "ssm_token_logp_args": _lib.TokenLogpArgs, "ssm_token_logp_bwd_args": _lib.TokenLogpBwdArgs, "ssm_topk_distill_args": _lib.TopkDistillArgs,
        "ssm_topk_distill_bwd_args": _lib.TopkDistillBwdArgs,
    }
    body = "".join(f'  printf("{n} %zu\\n", sizeof({n}));\n' for n in pairs)
    src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    src.write_text(f'#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{\n{body}  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size = line.split()
        assert ctypes.sizeof(pairs[name]) == int(size), name


def _delta_args(**kw):
    from ssm_b200 import _lib

    a = _lib.GatedDeltaArgs()
    a.batch, a.len, a.heads, a.key_heads, a.kdim, a.vdim = 1, 4, 2, 1, 8, 8
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("code,kw", [
    (-1, {}), (-2, {"heads": 3, "key_heads": 2}), (-2, {"kdim": 0}), (-6, {"kdim": 257}), (-3, {"io_dtype": 3}), (-3, {"g_dtype": 9}), (-2, {"batch": -1}),
    (-2, {"batch": 2, "num_seqs": 1}), (-1, {"num_seqs": 2}), (-6, {"num_seqs": 70000}), (0, {"batch": 0})])
def test_gated_delta_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    a = _delta_args(**kw)
    assert lib.ssm_gated_delta_fwd(ctypes.byref(a), None) == code
    g = _lib.GatedDeltaBwdArgs()
    g.fwd = a
    assert lib.ssm_gated_delta_bwd(ctypes.byref(g), None) == code
    assert lib.ssm_gated_delta_fwd(None, None) == lib.ssm_gated_delta_bwd(None, None) == lib.ssm_gated_delta_step(None, None) == -1


def test_sizes_of_gated_delta_scratch():
    from ssm_b200 import _lib

    lib = _lib.load()
    assert lib.ssm_gated_delta_chunks(3, 33, 0) == 6 and lib.ssm_gated_delta_chunks(1, 0, 0) == 0
    for nl in (0, 1, 31, 32, 33, 1000):  # any cut of nl rows into sequences and a rest has no more chunks than this
        for seqs in (1, 2, 7):
            bound = lib.ssm_gated_delta_chunks(1, nl, seqs)
            gen = torch.Generator().manual_seed(nl + seqs)
            for _ in range(50):
                cu = torch.sort(torch.randint(0, nl + 1, (seqs,), generator=gen)).values.tolist()
                cu = [0] + cu
                used = sum(-(-(b - a) // 32) for a, b in zip(cu, cu[1:])) + -(-(nl - cu[-1]) // 32)
                assert used <= bound
            assert lib.ssm_gated_delta_table_ints(1, nl, seqs) == 3 * seqs + 3 * bound


@pytest.mark.parametrize("code,kw", [(-2, {"vocab": 0}), (-3, {"io_dtype": 3}), (-2, {"temperature": 0.0}), (-2, {"temperature": float("nan")}), (-2, {"top_k": 9}),
                                     (-6, {"vocab": 500, "top_k": 129}), (-2, {"top_k": -1}), (-1, {}), (0, {"rows": 0}), (-6, {"rows": 1 << 29})])
def test_token_logp_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    a = _lib.TokenLogpArgs()
    a.rows, a.row_stride, a.vocab, a.temperature = 2, 8, 8, 1.0
    for name, value in kw.items():
        setattr(a, name, value)
    assert lib.ssm_token_logp(ctypes.byref(a), None) == code
    g = _lib.TokenLogpBwdArgs()
    g.fwd = a
    assert lib.ssm_token_logp_bwd(ctypes.byref(g), None) == code


@pytest.mark.parametrize("code,kw", [(-2, {"top_k": 0}), (-6, {"top_k": 1025}), (-3, {"teacher_dtype": 5}), (-1, {}), (0, {"rows": 0})])
def test_topk_distill_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    a = _lib.TopkDistillArgs()
    a.rows, a.row_stride, a.vocab, a.temperature, a.top_k = 2, 8, 8, 1.0, 2
    for name, value in kw.items():
        setattr(a, name, value)
    assert lib.ssm_topk_distill(ctypes.byref(a), None) == code


@pytest.mark.parametrize("code,kw", [
    (-1, {}), (-2, {"heads": 3, "key_heads": 2}), (-2, {"kdim": 0}), (-3, {"io_dtype": 9}), (-2, {"batch": 2, "num_seqs": 1})])
def test_chunked_gated_delta_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    g = _lib.GatedDeltaBwdArgs()
    g.fwd = _delta_args(io_dtype=1, **{k: x for k, x in kw.items() if k != "io_dtype"})
    if "io_dtype" in kw:
        g.fwd.io_dtype = kw["io_dtype"]
    assert lib.ssm_gated_delta_chunked_fwd(ctypes.byref(g.fwd), None, None, 0, None, None) == code
    assert lib.ssm_gated_delta_chunked_bwd(ctypes.byref(g), None, None, None, None) == code
    assert lib.ssm_gated_delta_chunked_fwd(None, None, None, 0, None, None) == lib.ssm_gated_delta_chunked_bwd(None, None, None, None, None) == -1


def test_what_goes_to_the_tensor_cores():
    """Pointers are looked at for their alignment alone here."""
    from ssm_b200 import _lib

    lib = _lib.load()

    def supported(**kw):
        a = _delta_args(io_dtype=1)
        a.q = a.k = a.v = a.o = 4096
        a.q_sh = a.k_sh = a.v_sh = 8
        a.q_st = a.k_st = a.v_st = 16
        a.q_sb = a.k_sb = a.v_sb = 64
        for name, value in kw.items():
            setattr(a, name, value)
        return lib.ssm_gated_delta_chunked_supported(ctypes.byref(a))

    assert supported() == supported(io_dtype=2) == supported(kdim=128) == supported(vdim=1024) == 1
    for kw in ({"io_dtype": 0}, {"kdim": 12}, {"kdim": 136}, {"kdim": 0}, {"vdim": 4}, {"vdim": 100}, {"len": 0}, {"q": 4098}, {"k": 4104}, {"v": 4100}, {"o": 4104},
               {"initial_state": 4100}, {"q_st": 12}, {"k_st": 0}, {"v_st": -16}, {"v_sh": 4}, {"heads": 0}, {"key_heads": 0}):
        assert supported(**kw) == 0, kw
    assert lib.ssm_gated_delta_chunked_supported(None) == 0


def test_sizes_beyond_32_bits_are_refused_before_they_are_cut():
    from ssm_b200 import ops

    wide = torch.zeros(1).expand(2, (1 << 32) + 5)
    with pytest.raises(ValueError, match="columns"):
        ops.token_log_probs(wide, torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="columns"):
        ops.topk_distill_loss(wide, torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.long))
    one = torch.zeros(1)
    big = (1 << 32) + 8
    for kd, vd, nh in ((big, 8, 2), (8, big, 2), (8, 8, 1 << 17)):
        q, v, b = one.expand(1, 3, 1, kd), one.expand(1, 3, nh, vd), one.expand(1, 3, nh)
        with pytest.raises(ValueError, match="at most"):
            ops.gated_delta_scan(q, q, v, b, b)
        with pytest.raises(ValueError, match="at most"):
            ops.gated_delta_step(one.expand(1, nh, vd, kd), q[:, 0], q[:, 0], v[:, 0], b[:, 0], b[:, 0])


def test_operators_refuse_wrong_shapes_and_cpu_tensors():
    from ssm_b200 import ops

    q, k, v, g, beta = _delta_inputs(1, 4, 1, 2, 8, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_delta_scan(q, k, v, g, beta)
    for bad in ((q[:, :3], k, v, g, beta), (q, k[..., :7], v, g, beta), (q, k, v[0], g, beta), (q, k, v, g[..., :1], beta), (q, k, v, g, beta[0]),
                (torch.cat([q] * 3, 2), torch.cat([k] * 3, 2), v, g, beta)):
        with pytest.raises(ValueError):
            ops.gated_delta_scan(*bad)
    with pytest.raises(ValueError, match="batch of one"):
        ops.gated_delta_scan(*(torch.cat([t, t]) for t in (q, k, v, g, beta)), cu_seqlens=torch.tensor([0, 4]))
    with pytest.raises(ValueError, match="initial_state"):
        ops.gated_delta_scan(q, k, v, g, beta, initial_state=torch.zeros(1, 2, 8, 7))
    with pytest.raises(ValueError, match="scale"):
        ops.gated_delta_scan(q, k, v, g, beta, scale=float("inf"))
    with pytest.raises(ValueError):
        ops.gated_delta_step(torch.zeros(1, 2, 8, 8), q[:, 0], k[:, 0], v[:, 0, :1], g[:, 0], beta[:, 0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_delta_step(torch.zeros(1, 2, 8, 8), q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.token_log_probs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long))
    for kw in ({"temperature": 0.0}, {"temperature": -1.0}, {"temperature": float("inf")}):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_log_probs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long), **kw)
        with pytest.raises(ValueError, match="temperature"):
            ops.topk_distill_loss(torch.zeros(2, 8), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.long), **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.topk_distill_loss(torch.zeros(2, 8), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.long))
