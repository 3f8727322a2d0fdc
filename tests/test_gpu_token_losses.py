"""Log probabilities of given tokens and distillation on the GPU against their definitions in 64 bits.

Tolerances.  A log probability is x - m, less the logarithm of a sum of V positive terms: its error is that of a difference and a product of
values of the size of the logits (three half steps of 2^-24) plus the sum's relative error; each thread adds V / 512 + 32 terms or
fewer in a row, with a 2^-21 relative error in every exponential (its argument, of size up to 2^6, is rounded: 2^6 2^-24 at most, plus
the instruction's own 2^-22).  Together under (V / 512 + 96) 2^-24 + 4 2^-24 |x|.  A gradient is a product of such probabilities, relative
error four times that, plus half a step of its own type.
"""

from __future__ import annotations

import pytest
import torch

from oracle import lm_oracle

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


def bar(vocab, size):
    return (vocab / 512 + 96 + 4 * size) * 2.0 ** -24


def near(got, want, atol, rtol=0.0, what=""):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, what
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(same | (off <= atol + rtol * want.abs()))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {off[bad].max().item():.3e}, allowed {atol:.3e}"


def logits_of(shape, dtype, seed=0, spread=3.0):
    return (spread * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)).to(dtype).double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top,temperature", [(1, 1, 1, 1.0), (3, 2, 2, 0.5), (5, 129, 7, 1.0), (2, 128, 128, 3.0), (300, 1000, 5, 1.0), (1, 50277, 20, 1.0),
                                                       (8, 50280, 20, 0.7), (9, 8193, 64, 1.0), (40, 4099, 0, 1.0), (2, 151937, 3, 1.3), (600, 333, 1, 1.0)])
def test_log_probs_entropy_top_and_gradients(rows, vocab, top, temperature, dtype):
    from ssm_b200 import ops

    x = logits_of((rows, vocab), dtype, seed=vocab).requires_grad_(True)
    gen = torch.Generator().manual_seed(rows)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    if rows > 2:
        targets[1] = -100
    want = lm_oracle.token_log_probs(x, targets, temperature, top)
    w = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in want[:3]]
    ref, = torch.autograd.grad(sum((a * b).sum() for a, b in zip(want[:3], w)), x)
    leaf = x.detach().to(dtype).cuda().requires_grad_(True)
    got = ops.token_log_probs(leaf, targets.cuda(), temperature, top_k=top, return_entropy=True)
    size = x.abs().max().item() / temperature
    tol = bar(vocab, size)
    near(got[0], want[0], tol, what="log probability")
    near(got[1], want[1], tol * (1 + size), what="entropy")  # each exponent weighs in with its own size
    outs, gs = [got[0], got[1]], [w[0], w[1]]
    if top:
        near(got[2], want[2], tol, what="top log probabilities")
        assert torch.equal(got[3].cpu(), want[3])
        outs, gs = outs + [got[2]], gs + [w[2]]
    d, = torch.autograd.grad(outs, leaf, [t.float().cuda() for t in gs])
    assert d.dtype == dtype and d.shape == leaf.shape
    scale = (1 + size) * (1 + sum(float(t.abs().max()) for t in gs if t.numel()) + (float(w[2].abs().sum(-1).max()) if top else 0)) / temperature
    near(d, ref, 4 * tol * scale + (2.0 ** -24 if dtype == torch.float16 else 0), HALF_STEP[dtype], "gradient")  # fp16: smallest values are 2^-24 apart


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_id(dtype):
    from ssm_b200 import ops

    for vocab in (700, 5000, 40000):
        x = torch.zeros(3, vocab, dtype=torch.float64)
        x[1] = torch.randint(-2, 3, (vocab,), generator=torch.Generator().manual_seed(vocab)).double()  # thousands of equal largest
        x[2, ::7] = -0.0
        x[2, 5:9] = 1.5
        want = lm_oracle.token_log_probs(x, torch.zeros(3, dtype=torch.long), top_k=40)
        got = ops.token_log_probs(x.to(dtype).cuda(), torch.zeros(3, dtype=torch.long).cuda(), top_k=40)
        assert torch.equal(got[2].cpu(), want[3])
        near(got[1], want[2], bar(vocab, 3))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(dtype):
    """-inf and the type's lowest value in masked places, rows with fewer live tokens than alternatives, rows with none."""
    from ssm_b200 import ops

    vocab, low = 9000, torch.finfo(dtype).min
    x = logits_of((6, vocab), dtype)
    x[0, 100:] = -INF
    x[1, torch.arange(vocab) % 1000 != 3] = -INF
    x[2] = -INF
    x[3, 10:] = low
    x[4] = low
    x[5, 1:] = -INF
    x.requires_grad_(True)
    targets = torch.tensor([5, 3, 7, 2, 8, 0])
    live = [0, 1, 3, 4, 5]
    want = lm_oracle.token_log_probs(x[live], targets[live], 1.0, 12)
    w = torch.linspace(0.5, 1.5, 6, dtype=torch.float64)
    # the definition's derivative, written out: autograd's has 0 * inf in masked places
    logp = torch.log_softmax(x.detach(), -1)
    p = torch.exp(logp)
    H = torch.zeros(6, dtype=torch.float64)
    H[live] = want[1].detach()
    plogp = torch.where(p > 0, p * logp.clamp_min(-1e300), torch.zeros_like(p))
    ref = -w[:, None] * p - 2 * w[:, None] * (plogp + p * H[:, None])
    ref[torch.arange(6), targets] += w
    ref[2] = 0
    leaf = x.detach().to(dtype).cuda().requires_grad_(True)
    got = ops.token_log_probs(leaf, targets.cuda(), top_k=12, return_entropy=True)
    near(got[0][live], want[0], bar(vocab, 12), what="log probability")
    near(got[1][live], want[1], 20 * bar(vocab, 12), what="entropy")
    # row 3's last two alternatives are the type's lowest value: |x| is 65504 there in fp16, where fp32 values are 2^-8 apart, and the
    # 4 2^-24 |x| of the tolerance is relative to it, not to the 12 of the other logits
    near(got[2][live], want[2], bar(vocab, 12), 4 * 2.0 ** -24, what="top")
    assert torch.equal(got[3][live].cpu(), want[3])
    assert got[0][2] == -INF and got[1][2] == 0 and (got[2][2] == -INF).all() and torch.equal(got[3][2].cpu(), torch.arange(12))
    d, = torch.autograd.grad([got[0], got[1]], leaf, [w.float().cuda(), 2 * w.float().cuda()])
    near(d, ref, 100 * bar(vocab, 12) + 2.0 ** -24, HALF_STEP[dtype], "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 40000])
def test_few_live_logits_among_masked_ones(dtype, vocab):
    """Fewer live logits than alternatives: the rest of the alternatives are the first masked ones.  One thread holding most of the largest."""
    from ssm_b200 import ops

    x = torch.full((6, vocab), -INF, dtype=torch.float64)
    x[0, [3, 5, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0], dtype=torch.float64)
    x[1] = torch.finfo(dtype).min
    x[1, [8, vocab // 2]] = torch.tensor([-1.0, 4.0], dtype=torch.float64)
    x[2, ::2] = torch.finfo(dtype).min
    x[3, vocab - 40:] = 1.0
    x[4] = 0.5 * torch.arange(vocab).remainder(8)
    x[5] = torch.finfo(dtype).min
    targets = torch.tensor([5, 8, 0, vocab - 1, 7, 3])
    want = lm_oracle.token_log_probs(x, targets, 1.0, 30)
    got = ops.token_log_probs(x.to(dtype).cuda(), targets.cuda(), top_k=30, return_entropy=True)
    near(got[0], want[0], bar(vocab, 4))
    near(got[1], want[1], 20 * bar(vocab, 4))
    near(got[2], want[2], bar(vocab, 4), 4 * 2.0 ** -24)
    assert torch.equal(got[3].cpu(), want[3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_inf_and_targets_outside(dtype):
    from ssm_b200 import ops

    x = logits_of((7, 600), dtype)
    x[1, 17], x[2, 18], x[3, 500] = NAN, INF, NAN
    targets = torch.tensor([3, 3, 3, -100, 600, -1, 599])
    leaf = x.to(dtype).cuda().requires_grad_(True)
    logp, entropy, top, ids = ops.token_log_probs(leaf, targets.cuda(), top_k=2, return_entropy=True)
    want = lm_oracle.token_log_probs(x[[0, 6]], targets[[0, 6]], 1.0, 2)
    near(logp[[0, 6]], want[0], bar(600, 12))
    assert torch.isnan(logp[[1, 2, 4, 5]]).all() and logp[3] == 0
    assert torch.isnan(entropy[[1, 2, 3]]).all() and torch.isfinite(entropy[[0, 4, 5, 6]]).all()
    assert ids[1, 0] == 17 and ids[2, 0] == 18 and torch.isnan(top[[1, 2, 3]]).all() and torch.isfinite(top[[4, 5]]).all()
    d, = torch.autograd.grad(logp[[0, 1, 2, 4, 6]].sum(), leaf)
    assert torch.isnan(d[[1, 2, 4]]).all() and torch.isfinite(d[[0, 6]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k,temperature", [(1, 1, 1, 1.0), (4, 50, 3, 2.0), (60, 50277, 32, 1.0), (3, 2000, 1024, 0.5), (700, 300, 20, 4.0), (2, 151937, 64, 1.0)])
def test_distillation_and_its_gradient(rows, vocab, k, temperature, dtype):
    from ssm_b200 import ops

    gen = torch.Generator().manual_seed(k)
    x = logits_of((rows, vocab), dtype, seed=1).requires_grad_(True)
    teacher = logits_of((rows, k), dtype, seed=2)
    ids = torch.stack([torch.randperm(max(vocab, k), generator=gen)[:k] % vocab for _ in range(rows)])
    if rows > 2 and k > 2:
        ids[0, 1] = -1          # left out
        ids[1, 2] = ids[1, 0]   # twice
        ids[2] = -5             # none
        teacher[0, 0] = -INF
    loss = lm_oracle.topk_distill_loss(x, teacher, ids, temperature)
    w = torch.randn(rows, generator=gen, dtype=torch.float64)
    ref, = torch.autograd.grad(loss, x, w)
    leaf = x.detach().to(dtype).cuda().requires_grad_(True)
    got = ops.topk_distill_loss(leaf, teacher.to(dtype).cuda(), ids.cuda(), temperature)
    size = max(x.abs().max().item(), teacher[torch.isfinite(teacher)].abs().max().item()) / temperature
    tol = bar(vocab, size) + bar(16 * k, size)
    near(got, loss, tol * (1 + size), what="loss")
    d, = torch.autograd.grad(got, leaf, w.float().cuda())
    near(d, ref, 4 * tol * (1 + float(w.abs().max())) / temperature + (2.0 ** -24 if dtype == torch.float16 else 0), HALF_STEP[dtype], "gradient")
    if rows > 2 and k > 2:
        assert got[2] == 0 and not d[2].any()


def test_distillation_of_masked_students_and_bad_ids():
    from ssm_b200 import ops

    x = logits_of((5, 900), torch.float32).float().cuda()
    x[0, 4] = -INF   # the teacher wants it
    x[1] = -INF
    x[2, 1] = NAN
    ids = torch.tensor([[4, 5], [4, 5], [4, 5], [4, 900], [4, 5]]).cuda()
    teacher = torch.tensor([[0.0, 1.0]]).repeat(5, 1).cuda()
    leaf = x.requires_grad_(True)
    loss = ops.topk_distill_loss(leaf, teacher, ids)
    assert loss[0] == INF and loss[1] == INF and torch.isnan(loss[2]) and torch.isnan(loss[3]) and torch.isfinite(loss[4])
    d, = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
    assert torch.isfinite(d[[0, 1, 4]]).all() and not d[1].any() and torch.isnan(d[2]).all()
    with pytest.raises(ValueError, match="detach"):
        ops.topk_distill_loss(leaf, teacher.requires_grad_(True), ids)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_leading_axes_and_integer_types(dtype):
    from ssm_b200 import ops

    x = logits_of((3, 5, 601), dtype).to(dtype).cuda()
    targets = torch.randint(0, 601, (3, 5), generator=torch.Generator().manual_seed(0)).cuda()
    ids = torch.randint(0, 601, (3, 5, 4), generator=torch.Generator().manual_seed(1)).cuda()
    teacher = torch.randn(3, 5, 4, generator=torch.Generator().manual_seed(2)).cuda()

    def both(t, a=targets, b=ids):
        t = t.detach().requires_grad_(True)
        out = [*ops.token_log_probs(t, a, top_k=3, return_entropy=True), ops.topk_distill_loss(t, teacher, b)]
        return out + [torch.autograd.grad(out[0].sum() + out[1].sum() + out[2].sum() + out[4].sum(), t)[0]]

    want = both(x)
    assert want[0].shape == (3, 5) and want[2].shape == want[3].shape == (3, 5, 3) and want[5].shape == x.shape
    wide = torch.full((3, 5, 700), NAN, dtype=dtype, device="cuda")
    for at in (0, 1, 8, 13):  # a padded row: slices at any offset
        view = wide[..., at:at + 601].copy_(x)
        for a, b in zip(both(view), want):  # other sums, both rounded: half a step each, so neighbours of a border lie a whole step apart
            near(a, b.cpu(), 1e-6, 2 * HALF_STEP[dtype])
    for view in (x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2)):
        assert all(torch.equal(a, b) for a, b in zip(both(view), want))
    assert all(torch.equal(a, b) for a, b in zip(both(x, targets.int(), ids.int()), want))
    one = ops.token_log_probs(x[0, 0], targets[0, 0])
    assert one.shape == () and torch.equal(one, want[0][0, 0])
    empty = x[:0].requires_grad_(True)
    got = ops.token_log_probs(empty, targets[:0], top_k=2)
    assert got[0].shape == (0, 5) and got[1].shape == (0, 5, 2)
    got[0].sum().backward()
    assert ops.topk_distill_loss(x[:0], teacher[:0], ids[:0]).shape == (0, 5)


def test_gradients_against_differences():
    """fp32, h = 2^-5 along directions of norm one; the loss is a sum of 6 terms of size 10 with errors of 1e-6 each: 1e-4 of 2h."""
    from ssm_b200 import ops

    x = logits_of((6, 200), torch.float32).float().cuda().requires_grad_(True)
    gen = torch.Generator().manual_seed(1)
    targets, ids = torch.randint(0, 200, (6,), generator=gen).cuda(), torch.randint(0, 200, (6, 5), generator=gen).cuda()
    teacher = torch.randn(6, 5, generator=gen).cuda()

    def f(t):
        logp, entropy, top, _ = ops.token_log_probs(t, targets, 0.8, top_k=2, return_entropy=True)
        return (logp + 0.5 * entropy).double().sum() + 0.3 * top.double().sum() + ops.topk_distill_loss(t, teacher, ids, 1.5).double().sum()

    grad, = torch.autograd.grad(f(x), x)
    h = 2.0 ** -5
    for _ in range(4):
        d = torch.randn(x.shape, generator=gen).cuda()
        d /= d.norm()
        diff = float((f(x.detach() + h * d) - f(x.detach() - h * d)) / (2 * h))
        assert abs(diff - float((grad * d).sum())) <= 1e-3 + h * h * 5


def test_streams_graphs_edits_and_second_derivatives():
    from ssm_b200 import ops

    x = logits_of((20, 5000), torch.bfloat16).bfloat16().cuda().requires_grad_(True)
    gen = torch.Generator().manual_seed(1)
    targets, ids = torch.randint(0, 5000, (20,), generator=gen).cuda(), torch.randint(0, 5000, (20, 5), generator=gen).cuda()
    teacher = torch.randn(20, 5, generator=gen).bfloat16().cuda()

    def go(t):
        logp, entropy, top, idx = ops.token_log_probs(t, targets, top_k=4, return_entropy=True)
        loss = ops.topk_distill_loss(t, teacher, ids, 2.0)
        return [logp, entropy, top, idx, loss, torch.autograd.grad([logp, entropy, top, loss], t, [torch.ones_like(s) for s in (logp, entropy, top, loss)])[0]]

    want = [t.detach().clone() for t in go(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    fresh = x.detach().clone().requires_grad_(True)
    with torch.cuda.stream(side):
        again = go(fresh)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept = go(fresh)
    with torch.no_grad():
        fresh.zero_()
    graph.replay()
    with torch.no_grad():
        fresh.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))
    logp, top, idx = ops.token_log_probs(x, targets, top_k=4)
    idx.fill_(-7)  # the caller's own
    got, = torch.autograd.grad(top.sum(), x)
    assert torch.isfinite(got).all()
    logits = x * 1.0
    logp = ops.token_log_probs(logits, targets)
    logits.add_(1.0)
    with pytest.raises(RuntimeError, match="modified in place"):
        logp.sum().backward()
    loss = ops.topk_distill_loss(x, teacher, ids)
    g, = torch.autograd.grad(loss.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), x)


def test_refusals_on_the_gpu():
    from ssm_b200 import ops

    x, t = torch.zeros(2, 200, device="cuda"), torch.zeros(2, dtype=torch.long, device="cuda")
    for kw in ({"top_k": 201}, {"top_k": 129}, {"top_k": -1}, {"temperature": 0.0}):
        with pytest.raises(ValueError):
            ops.token_log_probs(x, t, **kw)
    with pytest.raises(ValueError):
        ops.token_log_probs(x, t[:1])
    with pytest.raises(ValueError, match="integers"):
        ops.token_log_probs(x, t.float())
    with pytest.raises(ValueError, match="not built"):
        ops.token_log_probs(x.double(), t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.token_log_probs(x, t.cpu())
    ids = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for teacher, i in ((x[:, :2], ids), (x[:1, :3], ids[:1]), (x[:, :0], ids[:, :0]), (x[:, :3], ids.float())):
        with pytest.raises(ValueError):
            ops.topk_distill_loss(x, teacher, i)


def test_rows_beyond_32_bit_offsets():
    """A row that begins behind 2^31 elements: 45000 rows of 50280 bf16 logits, of which only the last few are looked at closely."""
    from ssm_b200 import ops

    rows, vocab = 45000, 50280
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-3:] = logits_of((3, vocab), torch.bfloat16).bfloat16().cuda()
    targets = torch.full((rows,), 11, device="cuda")
    x.requires_grad_(True)
    logp, entropy = ops.token_log_probs(x, targets, return_entropy=True)
    want = lm_oracle.token_log_probs(x[-3:].detach().double().cpu(), targets[-3:].cpu())
    near(logp[-3:], want[0], bar(vocab, 15))
    near(entropy[-3:], want[1], 16 * bar(vocab, 15))
    d, = torch.autograd.grad(logp.sum(), x)
    ref = -torch.softmax(x[-3:].detach().double().cpu(), -1)
    ref[:, 11] += 1
    near(d[-3:], ref, 8 * bar(vocab, 15), 2.0 ** -8)
    assert torch.isfinite(d[::997]).all()
