"""``ops.linear_cross_entropy`` against its definition in 64 bits.

Tolerances.  A logit is a sum of D products, each exact to 2^-24 or better, added in fp32 a few at a time: off by at most (D / 4 + 8) 2^-23 of the sum of the products' sizes, `dz`.  log Z is off by
no more than the largest of these, and by the exponentials' 2^-22 and the sums' 2^-18; the loss by twice that.  An element of the logits' gradient is then off by
p (2 dz + 2^-18) |w| and by half a step of the type it is rounded to (fp16: at least 2^-25 of 2^-13 of the largest weight; fp32: 2^-24), and its products with W and h carry that as sums of
sizes, with (terms / 4 + 8) 2^-23 of the sums for the additions; half a step of the result's type ends it (2^-25 at least in fp16, whose numbers below 2^-14 are 2^-24 apart)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training_oracle as oracle
from ssm_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(n, d, v, dtype, seed=0, left_out=0.1, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    h, w = rn(n, d).to(dtype), (spread / math.sqrt(d) * rn(v, d)).to(dtype)
    t = torch.randint(0, v, (n,), device="cuda", generator=gen)
    t = torch.where(torch.rand(n, device="cuda", generator=gen) < left_out, torch.full_like(t, -100), t)
    return h, w, t, torch.rand(n, device="cuda", generator=gen) + 0.1, 0.3 * rn(n)


def half(t):
    return torch.finfo(t).eps / 2


def bounds(h, w, t, wl, wz):
    """Values in 64 bits with how far each may be off: loss, log_z, dh, dw."""
    dtype = h.dtype
    kept = t != -100
    h, w = h.detach().double(), w.detach().double()
    h = torch.where(kept[:, None], h, torch.zeros((), dtype=torch.float64, device="cuda"))
    wl, wz = wl.double() * kept, wz.double() * kept
    at = torch.where(kept, t, torch.zeros_like(t))[:, None]
    z = h @ w.t()
    log_z = torch.logsumexp(z, -1)
    loss = (log_z - torch.gather(z, 1, at)[:, 0]) * kept
    d = h.shape[1]
    dz = (d / 4 + 8) * 2.0 ** -23 * (h.abs() @ w.abs().t())
    far = dz.amax(-1)
    e_z = far + 2.0 ** -18 + 2.0 ** -23 * log_z.abs()
    p = torch.exp(z - log_z[:, None])
    g = p * (wl + wz)[:, None]
    e = g.abs() * (2 * far + 2.0 ** -18)[:, None]
    g.scatter_add_(1, at, -wl[:, None])
    step = 2.0 ** -24 if dtype == torch.float32 else half(dtype)
    e = e + step * (g.abs() + e)
    if dtype == torch.float16:
        e = e + 2.0 ** -38 * float(torch.maximum(wl.abs(), (wl + wz).abs()).amax()) * kept[:, None]
    v, n = w.shape[0], h.shape[0]
    out = []
    for a, ea, b, terms in ((g, e, w, v), (g.t(), e.t(), h, n)):
        val = a @ b
        out.append((val, (ea + (terms / 4 + 8) * 2.0 ** -23 * a.abs()) @ b.abs() + half(dtype) * val.abs() + 1e-30))
    return (loss, 2 * e_z * kept), (log_z * kept, e_z * kept), *out


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    tol = tol + torch.finfo(got.dtype).smallest_normal * half(got.dtype)
    beyond = (want.abs() + tol >= torch.finfo(got.dtype).max) & got.isinf() & (got.double().sign() == want.sign())  # the type holds no more
    err = torch.where(beyond, torch.zeros_like(err), err)
    assert (err <= tol).all(), f"{what}: {float((err / tol.clamp(min=1e-30)).max())} of the tolerance"


def check(h, w, t, wl, wz, **kw):
    h, w = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, log_z = ops.linear_cross_entropy(h, w, t, return_log_z=True, **kw)
    dh, dw = torch.autograd.grad([loss, log_z], [h, w], [wl, wz])
    want = bounds(h, w, t, wl, wz)
    for got, (val, tol), what in zip((loss.detach(), log_z.detach(), dh, dw), want, ("loss", "log_z", "dh", "dw")):
        near(got, val, tol, what)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype and loss.dtype == log_z.dtype == torch.float32
    assert not dh[t == -100].any() and not loss[t == -100].any() and not log_z[t == -100].any()
    with torch.no_grad():
        assert torch.equal(ops.linear_cross_entropy(h, w, t, **kw), loss)
    return dh, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(1, 64, 256), (300, 64, 256), (256, 128, 512), (128, 1, 1), (7, 3, 5), (130, 100, 1000), (257, 65, 257), (1000, 320, 5003), (1, 768, 50277), (513, 260, 2049)])
def test_sizes(dtype, n, d, v):
    check(*make(n, d, v, dtype, left_out=0.0 if n == 1 else 0.1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 31, 32, 33, 63, 64, 65])
def test_up_to_64_rows_with_targets_all_over_a_warps_rows(n, dtype):
    """Up to 64 rows are columns of a product of the weight's rows: a target is a lane of one warp."""
    h, w, t, wl, wz = make(n, 96, 1001, dtype, left_out=0.0)
    for first, step in ((0, 1), (31, 32), (990, 0)):
        t = (first + step * torch.arange(n, device="cuda")).clamp(max=1000)
        t[n // 2] = 1000
        if step == 32:
            t[n // 3] = -100
        check(h, w, t, wl, wz)


@pytest.mark.parametrize("dtype", TYPES)
def test_an_odd_width_with_few_and_with_many_rows(dtype):
    check(*make(20, 1219, 700, dtype))
    check(*make(300, 517, 333, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_backward_pass(dtype):
    v = 151936  # 512 MB hold 1766 such rows in 16 bits
    check(*make(2000 if dtype != torch.float32 else 600, 64, v, dtype))


def test_more_rows_than_one_piece_of_the_forward_pass():
    check(*make(16384 + 300, 32, 300, torch.bfloat16))


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("dtype", TYPES)
def test_reductions(reduction, dtype):
    h, w, t, _, wz = make(500, 96, 700, dtype)
    share = 3.0 / (1 if reduction == "sum" else int((t != -100).sum()))
    want = bounds(h, w, t, torch.full((500,), share, device="cuda"), wz)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss, log_z = ops.linear_cross_entropy(h, w, t, reduction=reduction, return_log_z=True)
    dh, dw = torch.autograd.grad([loss, log_z], [h, w], [torch.full((), 3.0, device="cuda"), wz])
    total, tol = want[0][0].sum() * share / 3, want[0][1].sum() * share / 3
    near(loss.detach(), total, tol + 2.0 ** -24 * total.abs(), "loss")
    # the row's weight is one fp32 division more
    near(dh, want[2][0], want[2][1] + 2.0 ** -23 * want[2][0].abs(), "dh")
    near(dw, want[3][0], want[3][1] + 2.0 ** -23 * want[3][0].abs(), "dw")


def one_pass(h, w, t, reduction="mean", scale=3.0):
    """bf16 sums and means form the gradients with the loss: values against the definition.  There the rows' 1 / sum is rounded into h once more (2^-9) for dw."""
    n = h.shape[0]
    share = scale / (1 if reduction == "sum" else max(1, int((t != -100).sum())))
    want = bounds(h, w, t, torch.full((n,), share, device="cuda"), torch.zeros(n, device="cuda"))
    h, w = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = ops.linear_cross_entropy(h, w, t, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, [h, w], torch.full((), scale, device="cuda"))
    total, tol = want[0][0].sum() * share / scale, want[0][1].sum() * share / scale
    near(loss.detach(), total, tol + 2.0 ** -24 * total.abs(), "loss")
    near(dh, want[2][0], want[2][1] + 2.0 ** -23 * want[2][0].abs(), "dh")
    hd, wd = h.detach().double(), w.detach().double()
    kept = (t != -100).double()[:, None]
    p = torch.softmax(hd @ wd.t(), -1) * share * kept
    near(dw, want[3][0], want[3][1] + 2.0 ** -9 * (p.t() @ hd.abs()) * 1.01 + 2.0 ** -23 * want[3][0].abs(), "dw")
    return dh, dw


@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("n,d,v", [(1, 64, 256), (300, 64, 256), (7, 3, 5), (130, 100, 1000), (257, 65, 257), (1000, 320, 5003), (1, 768, 50277), (2000, 64, 151936), (9000, 40, 300)])
def test_loss_and_gradient_in_one_pass(n, d, v, reduction):
    one_pass(*make(n, d, v, torch.bfloat16, left_out=0.0 if n == 1 else 0.1)[:3], reduction)


@pytest.mark.parametrize("spread", [0.0, 40.0, 3000.0])
def test_one_pass_with_targets_far_below_the_maximum(spread):
    h, w, t, _, _ = make(700, 128, 900, torch.bfloat16, spread=spread)
    one_pass(h, w, t)
    one_pass(h, w, (h @ w.t()).float().argmax(-1))
    one_pass(h, w, (h @ w.t()).float().argmin(-1))


def test_one_pass_takes_the_targets_logit_from_the_product():
    """A loss near zero is a difference of two numbers that share the product's errors; only the exponentials, their sum and its logarithm differ between the forms: 2^-18 a row, as in
    `bounds` (a target's logit summed apart was off by 2^-20 of logits of 64 and more)."""
    h, w, _, _, _ = make(200, 1024, 700, torch.bfloat16, left_out=0.0)
    h = h * 16
    t = (h.float() @ w.float().t()).argmax(-1)
    loss = ops.linear_cross_entropy(h.requires_grad_(True), w, t, reduction="sum").detach()
    with torch.no_grad():
        want = ops.linear_cross_entropy(h, w, t, reduction="sum")
    assert (loss - want).abs() <= 200 * 2.0 ** -18 + 2.0 ** -22 * want


def test_one_pass_where_one_tile_of_rows_is_formed_again():
    h, w, t, _, _ = make(1000, 64, 700, torch.bfloat16, left_out=0.0)
    h[300] *= 100
    t[300] = (h[300] @ w.t()).float().argmin()
    one_pass(h, w, t)


def test_one_pass_with_common_targets():
    h, w, t, _, _ = make(3000, 64, 700, torch.bfloat16)
    one_pass(h, w, torch.where(torch.arange(3000, device="cuda") % 3 == 0, torch.full_like(t, 17), t))
    one_pass(h, w, torch.full_like(t, 699))


def test_one_pass_with_values_that_are_not_finite():
    h, w, t, _, _ = make(600, 64, 400, torch.bfloat16)
    want = one_pass(h, w, t)
    h2 = torch.where((t == -100)[:, None], torch.full_like(h, math.nan), h)
    for a, b in zip(torch.autograd.grad(ops.linear_cross_entropy(h2.requires_grad_(True), w.requires_grad_(True), t, reduction="mean"), [h2, w], torch.full((), 3.0, device="cuda")), want):
        assert torch.equal(a, b)
    for kind in ("target", math.nan, math.inf):
        h3, t3 = h.detach().clone(), t.clone()
        if kind == "target":
            t3[5] = 400
        else:
            h3[5, 7], t3[5] = kind, 3
        h3.requires_grad_(True)
        loss = ops.linear_cross_entropy(h3, w, t3, reduction="sum")
        dh, dw = torch.autograd.grad(loss, [h3, w])
        assert loss.isnan() and dh[5].isnan().all() and dw.isnan().all()
        assert dh[torch.arange(600, device="cuda") != 5].isfinite().all()


@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("factor", [math.inf, math.nan])
def test_one_pass_with_a_factor_that_is_not_finite_keeps_rows_left_out_at_zero(factor, d):
    h, w, t, _, _ = make(300, d, 400, torch.bfloat16)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, reduction="sum"), [h, w], torch.full((), factor, device="cuda"))
    out = t == -100
    assert out.any() and torch.equal(dh[out], torch.zeros_like(dh[out])) and not dh[~out].isfinite().any() and not dw.isfinite().any()


def test_one_pass_may_be_walked_twice():
    h, w, t, _, _ = make(300, 64, 400, torch.bfloat16)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    loss = ops.linear_cross_entropy(h, w, t, reduction="mean")
    a = torch.autograd.grad(loss, [h, w], retain_graph=True)
    a[0].zero_()
    b = torch.autograd.grad(2 * loss, [h, w])
    assert b[0].any() and torch.equal(b[1], 2 * a[1])
    only = torch.autograd.grad(ops.linear_cross_entropy(h, w.detach(), t, reduction="mean"), h)[0]
    assert torch.equal(2 * only, b[0])
    only = torch.autograd.grad(ops.linear_cross_entropy(h.detach(), w, t, reduction="mean"), w)[0]
    assert torch.equal(only, a[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_left_out_may_hold_anything(dtype):
    h, w, t, wl, wz = make(400, 96, 600, dtype, left_out=0.5)
    want = check(h, w, t, wl, wz)
    h = torch.where((t == -100)[:, None], torch.full_like(h, math.nan), h)
    h[(t == -100).nonzero()[0, 0]] = math.inf
    got = check(h, w, t, wl, wz)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rows", [0, 5, 300])
def test_nothing_counts(rows):
    h, w, t, _, _ = make(max(rows, 1), 64, 300, torch.bfloat16)
    h, t = h[:rows].requires_grad_(True), torch.full((rows,), -100, device="cuda")
    w.requires_grad_(True)
    for reduction in ("none", "sum", "mean"):
        loss = ops.linear_cross_entropy(h, w, t, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, [h, w], torch.ones_like(loss))
        assert not loss.detach().any() and not dh.any() and not dw.any() and dh.shape == h.shape


def test_the_first_and_last_row_and_column():
    h, w, t, wl, wz = make(512, 64, 513, torch.bfloat16, left_out=0.0)
    t[0], t[1], t[255], t[256], t[511] = 0, 512, 511, 256, 255
    check(h, w, t, wl, wz)
    t[1:] = -100
    check(h, w, t, wl, wz)
    t[:], t[511] = -100, 512
    check(h, w, t, wl, wz)


def test_other_ignore_index_and_integer_types():
    h, w, t, wl, wz = make(100, 64, 300, torch.float16)
    want = ops.linear_cross_entropy(h, w, t)
    for kind in (torch.int32, torch.int16):
        assert torch.equal(ops.linear_cross_entropy(h, w, t.to(kind)), want)
    moved = torch.where(t == -100, torch.full_like(t, 7), torch.where(t == 7, torch.full_like(t, 8), t))
    got = ops.linear_cross_entropy(h, w, moved, ignore_index=7)
    assert not got[t == -100].any() and torch.equal(got[(t != -100) & (t != 7)], want[(t != -100) & (t != 7)])


def test_targets_outside_and_values_that_are_not_finite():
    h, w, t, wl, wz = make(300, 64, 400, torch.bfloat16, left_out=0.0)
    clean = ops.linear_cross_entropy(h, w, t)
    t2 = t.clone()
    t2[5], t2[6], t2[7] = 400, -1, 2 ** 40
    h2 = h.clone()
    h2[9, 3], h2[10, 0] = math.nan, math.inf
    hl = h2.requires_grad_(True)
    loss = ops.linear_cross_entropy(hl, w, t2)
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[[5, 6, 7, 9, 10]] = True
    assert loss[bad].isnan().all() and torch.equal(loss[~bad], clean[~bad])
    dh = torch.autograd.grad(loss, hl, wl)[0]
    assert dh[bad].isnan().all() and dh[~bad].isfinite().all()


@pytest.mark.parametrize("spread", [0.0, 40.0, 3000.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_flat_and_steep_distributions(spread, dtype):
    check(*make(200, 128, 900, dtype, spread=spread))


@pytest.mark.parametrize("scale", [1e-4, 1.0, 65536.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_and_large_weights_of_rows(scale, dtype):
    h, w, t, wl, wz = make(200, 64, 300, dtype)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    dh = torch.autograd.grad(ops.linear_cross_entropy(h, w, t), h, scale * wl)[0]
    val, tol = bounds(h, w, t, scale * wl, 0 * wz)[2]
    near(dh, val, tol + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps, "dh")


def test_strides_and_shapes():
    h, w, t, _, _ = make(60, 72, 500, torch.bfloat16)
    want = ops.linear_cross_entropy(h, w, t)
    assert torch.equal(ops.linear_cross_entropy(h.view(4, 15, 72), w, t.view(4, 15)), want.view(4, 15))
    wide = torch.randn(60, 200, device="cuda").to(torch.bfloat16)
    wide[:, 5:77] = h
    assert torch.equal(ops.linear_cross_entropy(wide[:, 5:77], w, t), want)
    odd = torch.empty(500, 75, device="cuda", dtype=torch.bfloat16)
    odd[:, 1:73] = w
    assert torch.equal(ops.linear_cross_entropy(h, odd[:, 1:73], t), want)
    assert torch.equal(ops.linear_cross_entropy(h.t().contiguous().t(), w.t().contiguous().t(), t), want)
    same = ops.linear_cross_entropy(h[:1].expand(60, 72), w, t)
    assert torch.equal(same, ops.linear_cross_entropy(h[:1].repeat(60, 1), w, t))
    one = ops.linear_cross_entropy(h[0], w, t[0])
    assert one.shape == () and torch.equal(one, want[0])
    for shape in ((3, 20), (2, 3, 10)):
        hl = h.view(*shape, 72).requires_grad_(True)
        g = torch.autograd.grad(ops.linear_cross_entropy(hl, w, t.view(shape), reduction="sum"), hl)[0]
        assert g.shape == hl.shape


@pytest.mark.parametrize("wt", TYPES)
def test_a_weight_of_another_type(wt):
    h, w, t, wl, wz = make(150, 64, 300, torch.bfloat16)
    w = w.to(wt).requires_grad_(True)
    h = h.requires_grad_(True)
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, t), [h, w], wl)
    assert dw.dtype == wt
    val, tol = bounds(h, w.to(torch.bfloat16), t, wl, 0 * wz)[3]
    near(dw, val, tol + half(wt) * val.abs(), "dw")


def test_only_one_gradient_is_wanted():
    h, w, t, wl, _ = make(150, 64, 300, torch.bfloat16)
    both = torch.autograd.grad(ops.linear_cross_entropy(h.requires_grad_(True), w.requires_grad_(True), t), [h, w], wl)
    only_h = torch.autograd.grad(ops.linear_cross_entropy(h, w.detach(), t), h, wl)[0]
    only_w = torch.autograd.grad(ops.linear_cross_entropy(h.detach(), w, t), w, wl)[0]
    assert torch.equal(only_h, both[0]) and torch.equal(only_w, both[1])
    loss, log_z = ops.linear_cross_entropy(h, w, t, reduction="mean", return_log_z=True)
    g = torch.autograd.grad(log_z, h, wl)[0]
    want = bounds(h, w, t, 0 * wl, wl)[2]
    near(g, *want, "dh of log_z alone")


def test_gradients_against_differences():
    """Central differences of the 64-bit definition, in random directions."""
    h, w, t, wl, _ = make(20, 24, 50, torch.float32)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    dh, dw = torch.autograd.grad((ops.linear_cross_entropy(h, w, t) * wl).sum(), [h, w])
    f = lambda a, b: (oracle.linear_cross_entropy(a, b, t) * wl.double()).sum()  # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i, g in ((0, dh), (1, dw)):
        x = [h.detach().double(), w.detach().double()]
        dir = torch.randn(x[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-5 * dir, x[i] - 1e-5 * dir
        want = float((f(*up) - f(*down)) / 2e-5)
        assert abs(float((g.double() * dir).sum()) - want) < 1e-4 * (1 + abs(want))


def test_repeats_streams_and_graphs_give_the_same_bits():
    h, w, t, wl, _ = make(700, 128, 1500, torch.bfloat16)
    h, w = h.requires_grad_(True), w.requires_grad_(True)

    def once():
        loss = ops.linear_cross_entropy(h, w, t, reduction="mean")
        return [loss.detach(), *torch.autograd.grad(loss, [h, w])]

    want = once()
    for a, b in zip(once(), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
        once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for _ in range(2):
        for o in out:
            o.zero_()
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    t.copy_(torch.where(torch.arange(700, device="cuda") < 400, torch.full_like(t, -100), t))  # other rows count now
    graph.replay()
    for a, b in zip(out, once()):
        assert torch.equal(a, b)


def test_an_edit_between_the_passes_and_second_derivatives_are_errors():
    h, w, t, wl, _ = make(50, 64, 100, torch.bfloat16)
    h.requires_grad_(True)
    loss = ops.linear_cross_entropy(h, w, t)
    w.mul_(2)
    with pytest.raises(RuntimeError, match="modified in place"):
        loss.sum().backward()
    # what is not read again may be edited: targets, and everything where the gradients came with the loss
    for reduction in ("none", "mean"):
        want = torch.autograd.grad(ops.linear_cross_entropy(h, w, t, reduction=reduction).sum(), h)[0]
        t2, w2 = t.clone(), w.clone()
        loss = ops.linear_cross_entropy(h, w2, t2, reduction=reduction)
        t2.fill_(3)
        if reduction == "mean":
            w2.zero_()
        assert torch.equal(torch.autograd.grad(loss.sum(), h)[0], want)
    g = torch.autograd.grad(ops.linear_cross_entropy(h, w, t).sum(), h, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_last_piece_without_rows(dtype):
    """Pieces of 512 MB: nothing, or nothing in the last of them, counts."""
    h, w, t, wl, wz = make(2000 if dtype != torch.float32 else 600, 40, 151936, dtype)
    t[300:] = -100
    check(h, w, t, wl, wz)
    if dtype == torch.bfloat16:
        one_pass(h, w, t)
    t[:] = -100
    dh, dw = check(h, w, t, wl, wz)
    assert not dh.any() and not dw.any()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("d", [33, 36, 40, 64, 264])
def test_odd_widths_of_every_type_of_weight(wt, d):
    h, w, t, wl, wz = make(400, d, 700, torch.bfloat16)
    t[:200] = 3  # a common one
    w = w.to(wt).requires_grad_(True)
    h = h.requires_grad_(True)
    val, tol = bounds(h, w.to(torch.bfloat16), t, wl, 0 * wz)[3]
    near(torch.autograd.grad(ops.linear_cross_entropy(h, w, t), w, wl)[0], val, tol + half(wt) * val.abs(), "dw")
    one_pass(h.detach(), w.detach().to(torch.bfloat16), t)


@pytest.mark.parametrize("scale", [1e5, 1e7, 1e9])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_very_large_logits(scale, dtype):
    """The products' rounding is all that counts then: the loss is the largest logit's distance, to 2^-18 of the sums of the products' sizes; from 2^28 on NaN."""
    h, w, t, wl, _ = make(100, 64, 300, dtype)
    h = (h.float() * scale).to(dtype).requires_grad_(True)
    w.requires_grad_(True)
    z = h.detach().double() @ w.detach().double().t()
    kept = t != -100
    want = (torch.logsumexp(z, -1) - torch.gather(z, 1, t.clamp(min=0)[:, None])[:, 0]) * kept
    far = z.abs().amax(-1) * 1.4427 > 2.0 ** 28
    for reduction in ("none", "sum"):
        loss = ops.linear_cross_entropy(h, w, t, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, [h, w], torch.ones_like(loss))
        if reduction == "none":
            tol = 2.0 ** -18 * (h.detach().double().abs() @ w.detach().double().abs().t()).amax(-1)
            ok = kept & ~far
            assert ((loss.detach().double() - want).abs()[ok] <= tol[ok]).all()
            assert (loss.isnan() | (loss.detach().double() - want).abs().le(tol)).all() and not dh[~kept].any()
        if not far.any():
            assert dh.isfinite().all() and dw.isfinite().all() and loss.isfinite().all()


def test_a_long_batch_in_many_pieces():
    check(*make(40000, 24, 200, torch.bfloat16))
    one_pass(*make(40000, 24, 200, torch.bfloat16)[:3])


@pytest.mark.parametrize("kind", ["one pass", "two passes", "fp32"])
def test_a_walk_gives_back_what_the_call_held(kind):
    """The gradients that came with the loss, or the rows (and an fp32 weight) as the products read them, go with the walk, not with the loss."""
    n, d, v = 512, 256, 20000
    h, w, t, wl, _ = make(n, d, v, torch.float32 if kind == "fp32" else torch.bfloat16)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    one = torch.ones((), device="cuda")
    kw, g = ({"reduction": "mean"}, one) if kind == "one pass" else ({}, wl)
    least = (n + v) * d * 4 if kind == "one pass" else n * d * 2 if kind == "two passes" else 3 * (n + v) * d * 2
    loss = ops.linear_cross_entropy(h, w, t, **kw)
    want = torch.autograd.grad(loss, [h, w], g, retain_graph=True)
    before = torch.cuda.memory_allocated()
    got = torch.autograd.grad(loss, [h, w], g)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del got, a, b
    assert before - torch.cuda.memory_allocated() >= least
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, [h, w], g)


@pytest.mark.parametrize("n,v", [(50, 4000), (400, 4000)])
@pytest.mark.parametrize("by", ["loss", "log_z"])
def test_weights_of_rows_that_lie_far_apart_in_fp16(by, n, v):
    """Each row's gradient is as exact as its own weight asks, 2^12 down to 2^-12; dW where light rows alone reach is too.  A row's weight moves nothing but a power of two (`bounds`
    for weights of 1, times the row's own); for dW it goes to h, whose step is then 2^-25 of 2^13 of the largest product of a weight and a row's largest h at the worst, so
    2^-37 of that largest product for each row, times p."""
    h, w, t, _, _ = make(n, 64, v, torch.float16, left_out=0.1)
    size = torch.exp2((12 - 24 * torch.arange(n, device="cuda") // (n - 1)).float())
    light = torch.arange(n, device="cuda") >= n // 2  # these rows' distributions lie in the second half of the vocabulary
    h[:, 0], h[:, 1] = torch.where(light, -4.0, 4.0), torch.where(light, 4.0, -4.0)
    w[:, :2] = 0
    w[: v // 2, 0], w[v // 2:, 1] = 5.0, 5.0
    t = torch.where(t == -100, t, t % (v // 2) + (v // 2) * light)
    zero, one = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    unit = (one, zero) if by == "loss" else (zero, one)
    kept = t != -100
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    dh, dw = torch.autograd.grad(list(ops.linear_cross_entropy(hl, wl, t, return_log_z=True)), [hl, wl], [size * u for u in unit])
    (val, tol) = bounds(h, w, t, *unit)[2]
    near(dh, val * size[:, None].double(), tol * size[:, None], "dh")
    hd, wd, s = h.detach().double() * kept[:, None], w.detach().double(), size.double() * kept
    z = hd @ wd.t()
    p = torch.softmax(z, -1) * s[:, None]
    far = ((64 / 4 + 8) * 2.0 ** -23 * (hd.abs() @ wd.abs().t())).amax(-1)
    g = p.clone()
    if by == "loss":
        g.scatter_add_(1, t.clamp(min=0)[:, None], -s[:, None])
    e = p * (2 * far + 2.0 ** -18)[:, None] + half(torch.float16) * g.abs() + 2.0 ** -38 * s[:, None]
    val = g.t() @ hd
    tol = (e.t() + (n / 4 + 8) * 2.0 ** -23 * g.abs().t()) @ hd.abs() + half(torch.float16) * val.abs()
    tol = tol + 2.0 ** -37 * float((s * hd.abs().amax(-1)).max()) * (p / s.clamp(min=1e-30)[:, None]).sum(0)[:, None]
    near(dw, val, tol, "dw")


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_that_cancel(dtype):
    """dloss and dlog_z that add up to nothing, or to little, leave the target's part alone."""
    h, w, t, wl, _ = make(300, 64, 500, dtype)
    check(h, w, t, wl, -wl)
    check(h, w, t, wl, -wl * (1 - 2.0 ** -20))
    check(h, w, t, wl, torch.where(torch.arange(300, device="cuda") % 2 == 0, -wl, wl))
    check(h, w, t, 0 * wl, 0 * wl)


@pytest.mark.parametrize("n", [20, 100])
@pytest.mark.parametrize("v", [1, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_logits_are_all_far_below_zero(dtype, v, n):
    """As in `test_very_large_logits`: logits of one sign, around -1e8 to -3.6e8, within 2^29 ln 2 = 3.72e8; beyond it NaN, not an infinite loss."""
    h, w, t, _, _ = make(n, 64, v, dtype, left_out=0.0)
    h = (1 + 0.2 * h.float().abs().clamp(max=2.0)) / 64
    w = -(1 + 0.2 * w.float().abs().clamp(max=2.0))
    for size, reach in ((1e8, True), (1.85e8, True), (4e8, False)):
        hl, wl = (size * h).to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
        z = hl.detach().double() @ wl.detach().double().t()
        assert z.amax() * 1.4427 > -2.0 ** 29 if reach else z.amax() < -3.8e8
        want = torch.logsumexp(z, -1) - torch.gather(z, 1, t[:, None])[:, 0]
        tol = 2.0 ** -18 * z.abs().amax(-1)
        loss, log_z = ops.linear_cross_entropy(hl, wl, t, return_log_z=True)
        total = ops.linear_cross_entropy(hl, wl, t, reduction="sum")
        for out, g in ((loss, torch.ones(n, device="cuda")), (total, torch.ones((), device="cuda"))):
            assert all(x.isfinite().all() if reach else x.isnan().all() for x in (out, *torch.autograd.grad(out, [hl, wl], g)))
        if reach:
            assert ((loss.detach().double() - want).abs() <= tol).all() and ((log_z.detach().double() - torch.logsumexp(z, -1)).abs() <= tol).all()
            assert (total.detach().double() - want.sum()).abs() <= tol.sum()
        else:
            assert log_z.isnan().all()


@pytest.mark.parametrize("v", [2 ** 19 - 1, 2 ** 19, 2 ** 19 + 1])
def test_vocabularies_around_2_to_the_19(v):
    """From 2^19 on a target and its row's place take 64 bits where the targets are sorted."""
    h, w, t, wl, wz = make(70, 8, v, torch.bfloat16)
    t[0], t[1], t[2], t[3:9], t[68] = v - 1, v - 2, 0, v // 2, v - 1
    check(h, w, t, wl, wz)
    one_pass(h, w, t)


@pytest.mark.parametrize("wt", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,d,v", [(20, 96, 1001), (500, 64, 700), (300, 33, 400)])
def test_one_pass_with_a_weight_of_another_type(n, d, v, wt):
    """A model's fp32 (or fp16) weight beside bf16 hidden states: read in bf16, its gradient leaves in its own type."""
    h, w, t, _, _ = make(n, d, v, torch.bfloat16)
    w = torch.where(w.abs() < 2.0 ** -10, torch.zeros_like(w), w).to(wt)  # numbers that both types hold
    for reduction in ("mean", "sum"):
        dh, dw = one_pass(h, w, t, reduction)
        assert dh.dtype == torch.bfloat16 and dw.dtype == wt


def test_fp16_weights_of_rows_in_a_graph():
    """The rows' powers of two and dW's scale are found on the device: a replay goes by the weights of that moment, and two runs give the same bits."""
    h, w, t, wl, wz = make(700, 96, 1500, torch.float16)
    h, w, wl = h.requires_grad_(True), w.requires_grad_(True), wl * torch.exp2(-(torch.arange(700, device="cuda") % 20).float())

    def once():
        loss, log_z = ops.linear_cross_entropy(h, w, t, return_log_z=True)
        return torch.autograd.grad([loss, log_z], [h, w], [wl, wz])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for factor in (1.0, 2.0 ** -9, 3000.0):
        wl.mul_(factor), wz.mul_(factor)
        graph.replay()
        got = [o.clone() for o in out]
        for a, b in zip(got, once()):
            assert torch.equal(a, b)
        for a, (val, tol) in zip(got, bounds(h, w, t, wl, wz)[2:]):
            near(a, val, tol, "gradient")
