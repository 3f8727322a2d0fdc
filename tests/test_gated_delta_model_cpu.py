"""The gated delta mixer and the head's losses in `ssm_b200.lm`, on the CPU oracle's operators."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from oracle import lm_oracle
from ssm_b200.lm import MambaConfig, MambaLMHeadModel
from ssm_b200.mixer import GatedDeltaBlock


def _model(**extra):
    torch.manual_seed(0)
    cfg = MambaConfig(d_model=32, n_layer=2, vocab_size=50, ssm_cfg=dict(layer="GatedDelta", d_state=16, headdim=16, **extra))
    return MambaLMHeadModel(cfg, ops=lm_oracle.namespace())


@pytest.mark.parametrize("extra", [{}, {"key_heads": 2}])
def test_decode_reproduces_the_forward_and_gradients_reach_every_weight(extra):
    model = _model(**extra)
    ids = torch.randint(0, 50, (2, 9))
    with torch.no_grad():
        full = model(ids).logits
        cache = model.allocate_inference_cache(2)
        steps = torch.cat([model(ids[:, t:t + 1], inference_params=cache).logits for t in range(9)], 1)
        torch.testing.assert_close(steps, full, rtol=1e-4, atol=1e-5)
        assert model.generate(ids[:, :4], 7).shape == (2, 7)
    model.score(ids).sum().backward()
    for layer in model.backbone.layers:
        for name, p in layer.named_parameters():
            assert p.grad is not None and float(p.grad.abs().max()) > 0, name


def test_block_equals_a_restatement():
    torch.manual_seed(1)
    m = GatedDeltaBlock(16, d_state=8, headdim=8, key_heads=2, ops=lm_oracle.namespace())
    x = torch.randn(2, 16, 16)  # as many steps as the q and k convolutions have channels
    out, res = m(x, None)
    u = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * m.pre_norm_w

    def conv(n):
        t = (u @ getattr(m, "in_" + n).t()).transpose(1, 2)
        w = getattr(m, "conv_" + n)
        return F.silu(F.conv1d(F.pad(t, (3, 0)), w[:, None], getattr(m, f"conv_{n}_b"), groups=w.shape[0])).transpose(1, 2)

    unit = lambda t: t * torch.rsqrt(t.square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    q, k, v = unit(conv("q").reshape(2, 16, 2, 8)), unit(conv("k").reshape(2, 16, 2, 8)), conv("v").reshape(2, 16, 4, 8)
    g = -torch.exp(m.A_log) * F.softplus(u @ m.in_a.t() + m.dt_bias)
    o, _ = lm_oracle.gated_delta(q, k, v, g, torch.sigmoid(u @ m.in_b.t()))
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-5) * m.norm_w
    want = (o.reshape(2, 16, 32) * F.silu(u @ m.in_z.t())) @ m.out_proj.t()
    torch.testing.assert_close(out, want, rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(res, x)
    for bad in (dict(headdim=7), dict(headdim=8, key_heads=3)):
        with pytest.raises(ValueError):
            GatedDeltaBlock(16, d_state=8, **bad)


def test_scores_and_distillation_of_a_model():
    model = _model()
    ids = torch.randint(0, 50, (2, 7))
    logp = torch.log_softmax(model(ids).logits, -1)
    want = torch.gather(logp[:, :-1], 2, ids[:, 1:, None])[..., 0]
    torch.testing.assert_close(model.score(ids), want)
    got, entropy, top, at = model.score(ids, top_k=3, return_entropy=True)
    assert entropy.shape == (2, 6) and top.shape == at.shape == (2, 6, 3)
    torch.testing.assert_close(top, torch.topk(logp[:, :-1], 3).values)
    labels = ids.clone()
    labels[:, :4] = -100
    assert not model.score(ids, labels=labels)[:, :3].any()
    teacher, tid = torch.topk(torch.randn(2, 7, 50), 5)
    loss = model.distill_loss(ids, teacher, tid, 2.0)
    t = torch.log_softmax(teacher / 2, -1)
    torch.testing.assert_close(loss, (t.exp() * (t - torch.gather(torch.log_softmax(model(ids).logits / 2, -1), 2, tid))).sum(-1))
