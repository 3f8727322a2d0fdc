"""Losses of rows whose logits, over the temperature, are large: masked with a finite value, or sampled at next to no temperature.

Tolerances.  The definition is taken on the rounded logits.  A log probability is a difference of two logits over the temperature (the temperature, its
inverse, the difference, the product: eight half steps of 2^-24 at most, relative to it), less the logarithm of a sum of V terms: V / 512 + 32 additions in a row
and 64 for the exponentials, whose arguments of 2^6 and below are rounded relative to themselves.  The inputs' differences are zero or beyond
what a sum of 32 bits holds beside its largest term, or their sizes are below 32.  Entropies weigh each exponent with its size, up to log V + 8 below 20.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import lm_oracle

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
INF = float("inf")


def near(got, want, atol, rtol=0.0, what=""):
    got, want = got.detach().double().cpu(), want.detach().float().double()  # beyond the numbers of 32 bits: infinite
    assert got.shape == want.shape, what
    same = got == want
    bad = ~(same | ((got - want).abs() <= atol + rtol * want.abs()))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, got {got[bad][:4].tolist()}, wanted {want[bad][:4].tolist()}"


def saturated(t, dtype):
    """A gradient over a small temperature can be beyond its type's numbers: infinite there (their largest and half a step)."""
    return torch.where(t.abs() >= torch.finfo(dtype).max * (1 + HALF_STEP[dtype] / 2), t.sign() * INF, t)


def check(x, dtype, temperature, targets, top=5):
    """Log probabilities, entropy, alternatives and gradients of rows, and distillation onto them, against 64 bits."""
    from ssm_b200 import ops

    rows, vocab = x.shape
    x = x.to(dtype)
    leaf = x.cuda().requires_grad_(True)
    x = x.double()
    # differences before quotients: neither overflows
    d = (x - x.amax(-1, keepdim=True)) / temperature
    want = lm_oracle.token_log_probs(d, targets, 1.0, top)
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
    logp = torch.log_softmax(d, -1)
    tol, rel = (vocab / 512 + 96) * 2.0 ** -24, 8 * 2.0 ** -24
    got = ops.token_log_probs(leaf, targets.cuda(), temperature, top_k=top, return_entropy=True)
    near(got[0], want[0], tol, rel, "log probability")
    near(got[1], want[1], 20 * tol, what="entropy")
    assert torch.equal(got[3].cpu(), ids)
    near(got[2], torch.gather(logp, 1, ids), tol, rel, "top")
    w = torch.linspace(0.5, 1.5, rows, dtype=torch.float64)
    p = torch.exp(logp)
    kept = targets >= 0
    wl = torch.where(kept, w, torch.zeros_like(w))
    ref = -wl[:, None] * p - 2 * w[:, None] * p * (logp.clamp_min(-1e300) + want[1][:, None])
    ref[torch.arange(rows), targets.clamp_min(0)] += wl
    grad, = torch.autograd.grad([got[0], got[1]], leaf, [w.float().cuda(), 2 * w.float().cuda()])
    least = 2.0 ** -24 if dtype == torch.float16 else 0  # fp16: smallest values
    near(grad, saturated(ref / temperature, dtype), 200 * tol / temperature + least, HALF_STEP[dtype] + rel, "gradient")
    if temperature >= 1e-4:  # a teacher of the same size, over the same temperature
        at = torch.stack([torch.arange(3) * 7 + r for r in range(rows)]) % vocab
        teacher = torch.tensor([[0.0, 1.0, -0.5]]).repeat(rows, 1) * temperature
        t = torch.log_softmax(teacher.double() / temperature, -1)
        logq = torch.gather(logp, 1, at)
        live = torch.isfinite(logq).all(-1)
        loss = ops.topk_distill_loss(leaf, teacher.cuda(), at.cuda(), temperature)
        near(loss[live], (t.exp() * (t - logq)).sum(-1)[live], 4 * tol, 2 * rel, "distillation")
        grad, = torch.autograd.grad(loss.sum(), leaf)
        near(grad.double() * temperature, p.scatter_add(1, at, -t.exp()), 8 * tol + least * temperature, HALF_STEP[dtype] + rel, "gradient of the distillation")


SIZES = {torch.float32: [-1e10, 1e10, -1e12, 1e12, -1e15, -1e30, -1e32, 1e32, -1e36, 3e38, -3e38], torch.bfloat16: [-1e10, 1e10, -1e15, -1e30, -1e32, -1e36, 3e38, -3e38],
         torch.float16: [-65504.0, 65504.0, -3e4]}


@pytest.mark.parametrize("dtype", list(SIZES))
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_rows_of_one_value(dtype, vocab):
    """All logits masked by the same finite value, or all but a few: the distribution is even over what is left."""
    rows = []
    for v in SIZES[dtype]:
        a = torch.full((vocab,), v, dtype=torch.float64)
        b = a.clone()
        b[11:31] = v * (0.5 if v < 0 else 1.0)  # twenty above the others
        if v > 0:
            b[40:] *= 0.5
        rows += [a, b]
    x = torch.stack(rows)
    targets = torch.arange(len(rows)) % 31
    targets[3] = -100
    check(x, dtype, 1.0, targets)


@pytest.mark.parametrize("dtype", list(SIZES))
@pytest.mark.parametrize("vocab", [1000, 40000])
@pytest.mark.parametrize("temperature", [1e-6, 1e-8, 1e-20, 1e-36, 1e4, 1e30])
def test_temperatures_next_to_zero_and_beyond_all_logits(dtype, vocab, temperature):
    x = torch.round(30 * torch.rand(6, vocab, generator=torch.Generator().manual_seed(vocab), dtype=torch.float64))  # ties, differences of one or more
    x[1] -= 60
    x[2, 5] = 31.0
    x[3, 4:] = -INF
    x[4] = -INF
    x[4, [7, vocab - 1]] = -20.0
    x[5] = torch.finfo(dtype).min
    x[5, 3] = -5.0
    check(x, dtype, temperature, torch.tensor([3, 2, 5, 0, 7, 3]), top=2)


def test_masked_rows_between_ordinary_ones_keep_their_neighbours():
    """Rows of live logits beside fully masked ones, many rows: each as on its own."""
    from ssm_b200 import ops

    rows, vocab = 700, 3001
    x = 3 * torch.randn(rows, vocab, generator=torch.Generator().manual_seed(0))
    clean = x.clone()
    x[::3] = -1e30
    targets = torch.arange(rows) % vocab
    got, entropy, top, ids = ops.token_log_probs(x.cuda(), targets.cuda(), top_k=3, return_entropy=True)
    want = ops.token_log_probs(clean.cuda(), targets.cuda(), top_k=3, return_entropy=True)
    live = torch.arange(rows) % 3 != 0
    for a, b in zip((got, entropy, top, ids), want):
        assert torch.equal(a[live.cuda()], b[live.cuda()])
    dead = ~live.cuda()
    near(got[dead], torch.full((int(dead.sum()),), -math.log(vocab), dtype=torch.float64), 110 * 2.0 ** -24)
    near(entropy[dead], torch.full((int(dead.sum()),), math.log(vocab), dtype=torch.float64), 200 * 2.0 ** -24)
    assert torch.equal(ids[dead].cpu(), torch.arange(3).expand(int(dead.sum()), 3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_and_infinity_among_large_logits(dtype):
    """They show wherever they lie, beside any size of the others."""
    from ssm_b200 import ops

    x = torch.full((6, 40000), -1e30)
    x[1, 17] = float("nan")
    x[2, 39999] = INF
    x[3] = -INF
    x[3, 5] = float("nan")
    x[4] = -3e38
    x[4, 39990] = float("nan")
    x[5] = 1e30
    targets = torch.full((6,), 3).cuda()
    leaf = x.to(dtype).cuda().requires_grad_(True)
    logp, entropy = ops.token_log_probs(leaf, targets, return_entropy=True)
    bad = torch.tensor([False, True, True, True, True, False])
    for t in (logp, entropy):
        assert torch.equal(torch.isnan(t).cpu(), bad)
    d, = torch.autograd.grad(logp.sum() + entropy.sum(), leaf)
    assert torch.isnan(d[bad.cuda()]).all() and torch.isfinite(d[~bad.cuda()]).all()


def test_a_target_outside_the_vocabulary_reaches_masked_columns():
    """The row's gradient is NaN everywhere, where the probability is zero too."""
    from ssm_b200 import ops

    x = torch.zeros(2, 900, device="cuda")
    x[:, 50:] = -INF
    x.requires_grad_(True)
    logp, entropy = ops.token_log_probs(x, torch.tensor([900, 3]).cuda(), return_entropy=True)
    d, = torch.autograd.grad(logp.sum() + entropy.sum(), x)
    assert torch.isnan(logp[0]) and torch.isnan(d[0]).all() and torch.isfinite(d[1]).all()
