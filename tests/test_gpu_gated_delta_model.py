"""A gated delta language model on the CUDA operators against the same model on the CPU oracle: logits, decode, scores, distillation and their
gradients, as a program runs them one after the other."""

from __future__ import annotations

import copy

import pytest
import torch

from oracle import lm_oracle
from tests.gpu_util import close

pytestmark = pytest.mark.gpu

# chains of two layers of 16-bit operands end in tensors whose values are held relative to the largest, as for the other models
TOL = {torch.float32: dict(rtol=1e-4, atol=1e-5), torch.bfloat16: dict(rtol=2e-2, atol=2e-2)}


def near(got, want, dtype, what):
    """Logits.  In 16 bits each token passes 22 roundings (ten a layer: norm, projection, convolution, norm of q and k, answer, norm of the heads, gate, its
    product, out projection, sum; last norm and head), each at most 2^-8 and of either sign: sqrt(22) 2^-8 = 1.8e-2 in norm.  Single values have
    no such bound: the norm over a head divides by the answer's length, which has no lower bound (o = sum_j (q.k_j) u_j; keys and queries
    rounded by 2^-8 each move every q.k_j by up to 2^-7, and a query that happens to lie across all keys so far, as early tokens' do, has them all of that size)."""
    if dtype == torch.float32:
        return close(got, want, **TOL[dtype], what=what, reduced=True)
    got, want = got.double().cpu(), want.double().cpu()
    off = float((got - want).norm() / want.norm())
    assert off <= 22 ** 0.5 * 2.0 ** -8, (what, off)


def _pair(dtype, **extra):
    from ssm_b200.lm import MambaConfig, MambaLMHeadModel

    torch.manual_seed(5)
    cfg = MambaConfig(d_model=128, n_layer=2, vocab_size=96, ssm_cfg=dict(layer="GatedDelta", **extra))
    cpu = MambaLMHeadModel(cfg, ops=lm_oracle.namespace())
    gpu = MambaLMHeadModel(cfg)
    gpu.load_state_dict(copy.deepcopy(cpu.state_dict()))
    gpu = gpu.cuda()
    if dtype != torch.float32:
        for (name, pc), (_, pg) in zip(cpu.named_parameters(), gpu.named_parameters()):
            if not any(k in name for k in ("dt_bias", "A_log")):
                pg.data = pg.data.to(dtype)
            pc.data = pg.data.float().cpu()
    return cpu, gpu


@pytest.mark.parametrize("dtype,extra", [(torch.float32, dict(d_state=64, headdim=64, key_heads=2)), (torch.bfloat16, dict(d_state=128, headdim=128)),
                                         (torch.bfloat16, dict(d_state=64, headdim=64, key_heads=1))])
def test_model_matches_the_oracle(dtype, extra):
    cpu, gpu = _pair(dtype, **extra)
    tol = TOL[dtype]
    ids = torch.randint(0, 96, (2, 150), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        want = cpu(ids).logits
        got = gpu(ids.cuda()).logits
        near(got, want, dtype, "logits")
        cache = gpu.allocate_inference_cache(2)
        steps = torch.cat([gpu(ids[:, t:t + 1].cuda(), inference_params=cache).logits for t in range(20)], 1)
        near(steps, got[:, :20], dtype, "decode vs prefill")
        eager = gpu.generate(ids[:, :5].cuda(), 14)
        assert torch.equal(eager, gpu.generate(ids[:, :5].cuda(), 14, cuda_graph=True))
    teacher, tid = torch.topk(torch.randn(2, 150, 96, generator=torch.Generator().manual_seed(1)), 6)

    def losses(m, dev):
        logp, entropy = m.score(ids.to(dev), return_entropy=True)
        return logp, m.distill_loss(ids.to(dev), teacher.to(dev), tid.to(dev), 2.0), (logp.sum() + 0.1 * entropy.sum()) / 300

    a, b = losses(cpu, "cpu"), losses(gpu, "cuda")
    close(b[0], a[0], **tol, what="scores", reduced=True)
    close(b[1], a[1], **tol, what="distillation", reduced=True)
    (a[2] + a[1].mean()).backward()
    (b[2] + b[1].mean()).backward()
    for (name, pc), (_, pg) in zip(cpu.named_parameters(), gpu.named_parameters()):
        off = float((pg.grad.double().cpu() - pc.grad.double()).norm() / pc.grad.double().norm())
        assert off <= (1e-4 if dtype == torch.float32 else 3e-2), (name, off)
