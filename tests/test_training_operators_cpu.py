"""What a training step runs around the mixers, without a GPU: the definitions against differences and torch's own, the C structs' layout,
refusals, and the model's side of it on the CPU oracle."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import training_oracle as oracle

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "ssm_b200_lm.h"


def _rn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_gradients_of_the_definitions_are_those_of_differences():
    for rms in (True, False):
        for gate in (None, _rn(4), _rn(2, 4), _rn(2, 3, 4)):
            leaves = [t.requires_grad_(True) for t in (_rn(2, 3, 4, seed=1), _rn(2, 3, 4, seed=2), _rn(4, seed=3), _rn(4, seed=4), _rn(4, seed=5), _rn(4, seed=6))]
            gate = None if gate is None else gate.requires_grad_(True)
            f = lambda x, r, pw, w, pb, b, *g: oracle.fused_block_norm(x, r, pw, w, pb, b, g[0] if g else None, 0.7, rms, 1e-2, 1e-3)  # noqa: E731
            assert torch.autograd.gradcheck(f, (*leaves, *([] if gate is None else [gate])))
    t = torch.tensor([2, -100, 6])
    h, w = _rn(3, 5).requires_grad_(True), _rn(7, 5, seed=1).requires_grad_(True)
    for reduction in ("none", "sum", "mean"):
        assert torch.autograd.gradcheck(lambda a, b: oracle.linear_cross_entropy(a, b, t, reduction=reduction, return_log_z=True), (h, w))


def test_the_definitions_are_torch_s():
    h, w, t = _rn(6, 5), _rn(7, 5, seed=1), torch.tensor([0, 6, -100, 3, 3, -100])
    for reduction in ("none", "sum", "mean"):
        torch.testing.assert_close(oracle.linear_cross_entropy(h, w, t, reduction=reduction), torch.nn.functional.cross_entropy(h @ w.t(), t, reduction=reduction))
    assert float(oracle.linear_cross_entropy(h, w, torch.full_like(t, -100), reduction="mean")) == 0
    tensors = [_rn(5, 3), _rn(7, seed=1)]
    params = [torch.nn.Parameter(t.clone()) for t in tensors]
    for p in params:
        p.grad = p.detach().clone()
    want = torch.nn.utils.clip_grad_norm_(params, 0.5)
    got = oracle.clip_global_norm_(tensors, 0.5)
    torch.testing.assert_close(got.double(), want, rtol=1e-6, atol=0)
    for a, b in zip(tensors, params):
        torch.testing.assert_close(a, b.grad)
    x, res = _rn(2, 3, 8), _rn(2, 3, 8, seed=1)
    y, r = oracle.fused_block_norm(x, res, torch.ones(8).double(), torch.ones(8).double(), is_rms=False, post_eps=1e-3)
    want = res + torch.nn.functional.layer_norm(x, (8,), eps=1e-3)
    torch.testing.assert_close(r, want)
    torch.testing.assert_close(y, torch.nn.functional.layer_norm(want, (8,), eps=1e-5))


def test_ctypes_structs_match_c_layout(tmp_path):
    from ssm_b200 import _lib

    pairs = {"ssm_block_norm_args": _lib.BlockNormArgs, "ssm_block_norm_bwd_args": _lib.BlockNormBwdArgs, "ssm_linear_ce_args": _lib.LinearCeArgs,
             "ssm_linear_ce_bwd_args": _lib.LinearCeBwdArgs, "ssm_tensor_ref": _lib.TensorRef}
    fields = [(n, f[0]) for n, c in pairs.items() for f in c._fields_]
    src = tmp_path / "sizes.c"
    body = "".join(f'  printf("{n} %zu\\n", sizeof({n}));\n' for n in pairs) + "".join(f'  printf("{n}.{f} %zu\\n", offsetof({n}, {f}));\n' for n, f in fields)
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{\n{body}  return 0;\n}}\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size = line.split()
        struct, _, field = name.partition(".")
        assert (getattr(pairs[struct], field).offset if field else ctypes.sizeof(pairs[struct])) == int(size), name


def _norm_args(**kw):
    from ssm_b200 import _lib

    a = _lib.BlockNormArgs()
    a.rows, a.len, a.dim, a.x, a.post_weight, a.weight, a.y, a.residual_out = 4, 2, 64, 4096, 4096, 4096, 4096, 4096
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("code,kw", [(-2, {"dim": 0}), (-2, {"rows": -1}), (-2, {"len": 0}), (-6, {"dim": 8193}), (-6, {"rows": 1 << 31}), (-3, {"io_dtype": 5}), (-3, {"gate_dtype": -1}),
                                     (-2, {"gate_kind": 4}), (-2, {"gate_kind": 2, "len": 3, "gate": 4096}), (-1, {"x": None}), (-1, {"gate_kind": 1}), (-1, {"bias": 4096}), (-1, {"y": None}),
                                     (-4, {"x": 4098}), (-4, {"stats": 4104}), (0, {"rows": 0})])
def test_block_norm_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    assert lib.ssm_block_norm_fwd(ctypes.byref(_norm_args(**kw)), None) == code
    assert lib.ssm_block_norm_fwd(None, None) == lib.ssm_block_norm_bwd(None, None) == -1
    g = _lib.BlockNormBwdArgs()
    g.fwd = _norm_args(**{"stats": 4096, **kw})
    if kw != {"y": None}:
        assert lib.ssm_block_norm_bwd(ctypes.byref(g), None) == (code or (0 if kw == {"rows": 0} else -1))


def _ce_args(**kw):
    from ssm_b200 import _lib

    a = _lib.LinearCeArgs()
    a.rows, a.hidden_stride, a.weight_stride, a.ignore_index, a.dim, a.vocab, a.io_dtype = 4, 64, 64, -100, 64, 100, 1
    for name in ("hidden", "weight", "targets", "row_loss", "log_z", "loss", "stats", "packs", "scratch", "status"):
        setattr(a, name, 4096)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("code,kw", [(-2, {"dim": 0}), (-2, {"vocab": 0}), (-2, {"rows": -1}), (-2, {"hidden_stride": -1}), (-6, {"vocab": (1 << 28) + 1}), (-6, {"dim": (1 << 20) + 1}),
                                     (-6, {"rows": (1 << 28) + 1}), (-3, {"io_dtype": 3}), (-2, {"reduction": 3}), (-1, {"weight": None}), (-1, {"hidden": None}), (-1, {"scratch": None}),
                                     (-1, {"packs": None}), (-1, {"status": None}), (-4, {"hidden": 4097}), (-4, {"scratch": 4096 + 64}), (-4, {"stats": 4104})])
def test_linear_ce_refuses_without_a_gpu(code, kw):
    from ssm_b200 import _lib

    lib = _lib.load()
    assert lib.ssm_linear_ce_fwd(ctypes.byref(_ce_args(**kw)), None) == code
    g = _lib.LinearCeBwdArgs()
    g.fwd, g.dloss = _ce_args(**kw), 4096
    assert lib.ssm_linear_ce_bwd(ctypes.byref(g), None) == code
    assert lib.ssm_linear_ce_train(ctypes.byref(_ce_args(**kw)), None, None, None, None) == code
    assert lib.ssm_linear_ce_fwd(None, None) == lib.ssm_linear_ce_bwd(None, None) == lib.ssm_linear_ce_train(None, None, None, None, None) == -1


def test_linear_ce_refuses_missing_outputs_and_what_one_pass_is_not_built_for():
    from ssm_b200 import _lib

    lib = _lib.load()
    for kw in ({"row_loss": None}, {"log_z": None}, {"reduction": 1, "loss": None}):
        assert lib.ssm_linear_ce_fwd(ctypes.byref(_ce_args(**kw)), None) == -1
    g = _lib.LinearCeBwdArgs()
    g.fwd = _ce_args()
    assert lib.ssm_linear_ce_bwd(ctypes.byref(g), None) == -1
    g.dloss, g.dweight_dtype = 4096, 7
    assert lib.ssm_linear_ce_bwd(ctypes.byref(g), None) == -3
    for kw in ({}, {"reduction": 1, "io_dtype": 0}, {"reduction": 2, "io_dtype": 2}, {"reduction": 1, "rows": 0}):
        assert lib.ssm_linear_ce_train(ctypes.byref(_ce_args(**kw)), None, None, 4096, None) == -5
    assert lib.ssm_linear_ce_train(ctypes.byref(_ce_args(reduction=1)), None, None, None, None) == -1
    assert lib.ssm_linear_ce_scale(None, 8, 2, 8, None, None, None, 0, None) == -1
    assert lib.ssm_linear_ce_scale(None, 8, 2, 9, None, None, None, 0, None) == -2
    assert lib.ssm_linear_ce_scale(None, 8, 0, 8, None, None, None, 0, None) == 0


@pytest.mark.parametrize("io", [0, 1, 2])
@pytest.mark.parametrize("rows,dim,vocab", [(0, 1, 1), (1, 1, 1), (8192, 2560, 50280), (100000, 64, 1 << 20), (1 << 28, 1, 1)])
def test_linear_ce_scratch_has_a_size_for_every_call(io, rows, dim, vocab):
    from ssm_b200 import _lib

    lib = _lib.load()
    a = _ce_args(rows=rows, dim=dim, vocab=vocab, io_dtype=io, hidden_stride=dim, weight_stride=dim)
    sizes = [lib.ssm_linear_ce_scratch_bytes(ctypes.byref(a), p) for p in range(3)]
    assert all(s >= 16 * rows for s in sizes) and lib.ssm_linear_ce_packs_bytes(ctypes.byref(a)) >= rows * (8 + 2 * dim)
    # 512 MB of the logits' gradient (three planes of it in fp32) and 256 rows at least, never the whole matrix of a long batch
    if (rows, dim, vocab) == (8192, 2560, 50280):
        assert sizes[1] < (512 << 20) + 4 * vocab * dim + (512 << 20)
    assert lib.ssm_linear_ce_scratch_bytes(None, 0) == lib.ssm_linear_ce_packs_bytes(None) == 0


@pytest.mark.parametrize("code,ref", [(-1, (None, 4, 0)), (-2, (4096, -1, 0)), (-3, (4096, 4, 4)), (-4, (4097, 4, 1)), (-6, (4096, (1 << 40) + 1, 0))])
def test_global_norm_refuses_without_a_gpu(code, ref):
    from ssm_b200 import _lib

    lib = _lib.load()
    one = (_lib.TensorRef * 1)(_lib.TensorRef(*ref, 0))
    assert lib.ssm_global_norm(one, 1, 0, 4096, 4096, None) == code
    assert lib.ssm_clip_global_norm(one, 1, 0, 1.0, 4096, 4096, None) == code
    good = (_lib.TensorRef * 1)(_lib.TensorRef(4096, 4, 0, 0))
    assert lib.ssm_global_norm(good, 1, 0, None, 4096, None) == lib.ssm_global_norm(good, 1, 0, 4096, None, None) == lib.ssm_global_norm(None, 1, 0, 4096, 4096, None) == -1
    assert lib.ssm_global_norm(good, -1, 0, 4096, 4096, None) == -2 and lib.ssm_global_norm(good, 1, 0, 4100, 4096, None) == -4
    assert lib.ssm_clip_global_norm(good, 1, 0, -1.0, 4096, 4096, None) == lib.ssm_clip_global_norm(good, 1, 0, math.nan, 4096, 4096, None) == -2
    assert lib.ssm_global_norm_scratch_bytes(0) == lib.ssm_global_norm_scratch_bytes(1024) < lib.ssm_global_norm_scratch_bytes(1025)


def test_operators_refuse_wrong_shapes_and_cpu_tensors():
    from ssm_b200 import ops

    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fused_block_norm(x, x, w, w)
    for args, kw in (((x[0], x[0], w, w), {}), ((x, x[:1], w, w), {}), ((x, x, w[:7], w), {}), ((x, x, w, w[None]), {}), ((x, x, w, w), {"gate": torch.zeros(3, 8)}),
                     ((x, x, w, w), {"gate": torch.zeros(2, 3, 1)}), ((x, x, w, w), {"gate": torch.zeros(2)}), ((x, x, w, w), {"bias": w[:1]}), ((x, x, w, w), {"post_bias": x}),
                     ((x, x, w, w), {"residual_scale": math.inf}), ((x, x, w, w), {"residual_scale": math.nan}), ((x, x, w, w), {"eps": -1.0}), ((x, x, w, w), {"post_eps": math.nan}),
                     ((torch.zeros(1, 1, 8193), None, torch.ones(8193), torch.ones(8193)), {})):
        with pytest.raises(ValueError):
            ops.fused_block_norm(*args, **kw)
    h, wt, t = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_cross_entropy(h, wt, t)
    for args, kw in (((h, wt[:, :7], t), {}), ((h, wt[0], t), {}), ((h, wt, t[:3]), {}), ((h, wt, t[None]), {}), ((h, wt, t.float()), {}), ((h, wt[:0], t), {}), ((h[:, :0], wt[:, :0], t), {}),
                     ((h, wt, t), {"reduction": "average"})):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy(*args, **kw)
    with pytest.raises(ValueError, match="at most"):
        ops.linear_cross_entropy(h, torch.zeros(1, 1).expand((1 << 28) + 1, 8), t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.global_norm([h])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.clip_global_norm_([h], 1.0)
    for bad in (1.0, 0.0, -2.0, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            ops.global_norm([h], bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_global_norm_([h], bad)
    for bad in ([1.0], [h, None], ["x"]):
        with pytest.raises(TypeError, match="tensors"):
            ops.global_norm(bad)
    with pytest.raises(ValueError, match="sparse"):
        ops.global_norm([torch.zeros(3).to_sparse()])


# ---- the model's side --------------------------------------------------------------------------------------------------------

KINDS = [("Mamba1", dict(d_state=8)), ("Mamba2", dict(d_state=16, headdim=8)), ("GatedDelta", dict(d_state=8, headdim=8))]


def _model(kind, extra, rms=True, **cfg):
    from ssm_b200.lm import MambaConfig, MambaLMHeadModel

    torch.manual_seed(0)
    model = MambaLMHeadModel(MambaConfig(d_model=32, n_layer=3, vocab_size=50, rms_norm=rms, ssm_cfg=dict(layer=kind, **extra), **cfg), ops=oracle.namespace())
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "post_" in n or "norm" in n:
                p += 0.1 * torch.randn_like(p)
    return model


@pytest.mark.parametrize("kind,extra", KINDS, ids=[k for k, _ in KINDS])
@pytest.mark.parametrize("gate", [True, False])
def test_decode_reproduces_the_full_forward_with_post_norms(kind, extra, gate):
    model = _model(kind, dict(extra, post_norm=True, post_gate=gate, residual_scale=0.5))
    ids = torch.randint(0, 50, (2, 7))
    with torch.no_grad():
        full = model(ids).logits
        cache = model.allocate_inference_cache(2)
        steps = torch.cat([model(ids[:, t:t + 1], inference_params=cache).logits for t in range(7)], dim=1)
    torch.testing.assert_close(steps, full, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("fp32", [True, False])
def test_post_norms_are_those_of_the_formula(rms, fp32):
    model = _model("Mamba1", dict(d_state=4, post_norm=True, post_gate=True, residual_scale=0.25), rms, residual_in_fp32=fp32).backbone
    ids = torch.randint(0, 50, (2, 5))

    def norm(x, w, b):
        x = x if rms else x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w
        return x if b is None else x + b

    with torch.no_grad():
        stream = model.embedding(ids)
        for layer in model.layers:
            out = layer.mixer_forward(norm(stream, layer.norm_w, getattr(layer, "norm_b", None)))
            stream = stream + 0.25 * layer.post_gate * norm(out, layer.post_norm_w, getattr(layer, "post_norm_b", None))
        torch.testing.assert_close(model(ids), norm(stream, model.norm_f_weight, model.norm_f_bias), rtol=1e-4, atol=1e-5)


def test_post_norm_options_stand_together():
    for extra in ({"post_gate": True}, {"residual_scale": 0.5}):
        with pytest.raises(ValueError, match="post_norm"):
            _model("Mamba1", extra)


def test_loss_is_that_of_the_logits():
    model = _model("Mamba2", dict(d_state=16, headdim=8))
    ids = torch.randint(0, 50, (2, 7))
    labels = torch.where(torch.rand(2, 7) < 0.3, torch.full_like(ids, -1), ids)
    want = -model.score(ids)
    torch.testing.assert_close(model.loss(ids, reduction="none"), want)
    torch.testing.assert_close(model.loss(ids), want.mean())
    torch.testing.assert_close(model.loss(ids, reduction="sum"), want.sum())
    want = -model.score(ids, labels, ignore_index=-1)
    loss, log_z = model.loss(ids, labels, ignore_index=-1, return_log_z=True)
    torch.testing.assert_close(loss, want.sum() / (labels[:, 1:] != -1).sum())
    torch.testing.assert_close(log_z, torch.logsumexp(model(ids).logits, -1)[:, :-1] * (labels[:, 1:] != -1))
    got = torch.autograd.grad(model.loss(ids), list(model.parameters()), allow_unused=True)
    want = torch.autograd.grad(-model.score(ids).mean(), list(model.parameters()), allow_unused=True)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)
    for kw in ({"sharded": True}, {"inference_params": model.allocate_inference_cache(2)}, {"num_last_tokens": 1}):
        with pytest.raises(ValueError, match="loss"):
            model.loss(ids, **kw)
    with pytest.raises(ValueError, match="2D"):
        model.loss(ids[0])


def test_clipping_scales_all_gradients_once():
    model = _model("Mamba1", dict(d_state=4))
    model.loss(torch.randint(0, 50, (2, 7))).backward()
    grads = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    want = torch.sqrt(sum(g.double().pow(2).sum() for g in grads))
    norm = model.clip_grad_norm_(0.01)
    assert abs(float(norm) - float(want)) < 1e-6 * float(want)
    for p, g in zip((p for p in model.parameters() if p.grad is not None), grads):
        torch.testing.assert_close(p.grad, g * (0.01 / (float(want) + 1e-6)), rtol=1e-5, atol=1e-9)
