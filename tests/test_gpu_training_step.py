"""A training step of a language model with norms after its mixers on the CUDA operators (loss without the logits, backward pass, clipping), as a program runs
it, against the same model on the CPU oracle."""

from __future__ import annotations

import copy

import pytest
import torch

from oracle import training_oracle as oracle
from tests.gpu_util import close

pytestmark = pytest.mark.gpu

TOL = dict(rtol=1e-4, atol=1e-5)  # as the other models' in fp32
KINDS = [("Mamba1", dict(d_state=8)), ("GatedDelta", dict(d_state=32, headdim=32))]


def pair(kind, extra, rms=True, dtype=torch.float32, **cfg):
    from ssm_b200.lm import MambaConfig, MambaLMHeadModel

    torch.manual_seed(5)
    config = MambaConfig(d_model=64, n_layer=2, vocab_size=90, rms_norm=rms, ssm_cfg=dict(layer=kind, post_norm=True, post_gate=True, residual_scale=0.5, **extra), **cfg)
    cpu = MambaLMHeadModel(config, ops=oracle.namespace())
    with torch.no_grad():
        for n, p in cpu.named_parameters():
            if "post_" in n or "norm" in n:
                p += 0.1 * torch.randn_like(p)
            if "embedding" in n:
                p *= 20
    gpu = MambaLMHeadModel(config)
    gpu.load_state_dict(copy.deepcopy(cpu.state_dict()))
    return cpu, gpu.cuda().to(dtype)


@pytest.mark.parametrize("kind,extra", KINDS, ids=[k for k, _ in KINDS])
@pytest.mark.parametrize("rms", [True, False])
def test_loss_gradients_and_clipping(kind, extra, rms):
    cpu, gpu = pair(kind, extra, rms)
    ids = torch.randint(0, 90, (3, 33))
    labels = torch.where(torch.rand(3, 33) < 0.2, torch.full_like(ids, -100), ids)
    for kw in ({}, {"reduction": "sum"}):
        for m, dev in ((cpu, "cpu"), (gpu, "cuda")):
            m.zero_grad()
            m.loss(ids.to(dev), labels.to(dev), **kw).backward()
        close(gpu.loss(ids.cuda(), labels.cuda(), **kw), cpu.loss(ids, labels, **kw), **TOL, what="loss", reduced=True)
        norms = [m.clip_grad_norm_(0.1) for m in (cpu, gpu)]
        close(norms[1], norms[0], **TOL, what="norm", reduced=True)
        for (n, p), q in zip(cpu.named_parameters(), gpu.parameters()):
            close(q.grad, p.grad, **TOL, what=n, reduced=True)
    close(gpu.loss(ids.cuda(), reduction="none"), cpu.loss(ids, reduction="none"), **TOL, what="losses", reduced=True)


@pytest.mark.parametrize("kind,extra", KINDS + [("Mamba2", dict(d_state=16, headdim=16))], ids=["Mamba1", "GatedDelta", "Mamba2"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_loss_is_that_of_the_scores(kind, extra, dtype):
    """The same hidden states, once through the head's logits.  Those are rounded: half a step each, relative to the largest, two to a loss (log Z and the target's)."""
    _, gpu = pair(kind, extra, dtype=dtype)
    ids = torch.randint(0, 90, (2, 40), device="cuda")
    with torch.no_grad():
        got, want = gpu.loss(ids, reduction="none"), -gpu.score(ids)
        assert float((got - want).abs().max()) < 1e-4 + 2 * torch.finfo(dtype).eps / 2 * float(gpu(ids).logits.abs().max())
        assert abs(float(gpu.loss(ids)) - float(got.mean())) < 1e-5 * float(got.mean())
    one = torch.autograd.grad(gpu.loss(ids), [p for p in gpu.parameters()])
    assert all(g.isfinite().all() for g in one)


def test_decode_with_post_norms():
    cpu, gpu = pair("GatedDelta", dict(d_state=32, headdim=32))
    ids = torch.randint(0, 90, (2, 6))
    want = cpu.generate(ids, 12)
    assert torch.equal(gpu.generate(ids.cuda(), 12).cpu(), want)
    assert torch.equal(gpu.generate(ids.cuda(), 12, cuda_graph=True).cpu(), want)


def test_a_step_in_a_graph_repeats_the_eager_one():
    _, gpu = pair("Mamba2", dict(d_state=16, headdim=16), dtype=torch.bfloat16)
    from ssm_b200 import ops

    ids = torch.randint(0, 90, (2, 64), device="cuda")
    params = list(gpu.parameters())

    def step():
        loss = gpu.loss(ids)
        grads = list(torch.autograd.grad(loss, params))
        norm = ops.clip_global_norm_(grads, 0.05)
        return [loss.detach(), norm, *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_traced_calls_are_made_again():
    from ssm_b200 import ops

    def f(x, res, w, head, t):
        y, r = ops.fused_block_norm(x, res, w, w, gate=w, residual_scale=0.5)
        return ops.linear_cross_entropy(y, head, t, reduction="mean"), r

    def inputs(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        return rn(2, 9, 64).bfloat16(), rn(2, 9, 64), rn(64).bfloat16(), rn(100, 64).bfloat16(), torch.randint(0, 100, (2, 9), device="cuda", generator=gen)

    with torch.no_grad():
        traced = torch.jit.trace(f, inputs(0), check_trace=False)
        for a, b in zip(traced(*inputs(1)), f(*inputs(1))):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="not traced"):
            torch.jit.trace(lambda x: ops.global_norm([x]), (inputs(0)[0],), check_trace=False)
