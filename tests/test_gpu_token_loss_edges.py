"""Token losses at the border of what their documents say: ids outside the vocabulary that carry no weight, rows of NaN, rows without a teacher."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_id_outside_the_vocabulary_counts_by_its_weight_in_both_directions(dtype):
    """Lists padded with an id of V and a logit of -inf, or with one whose weight is nothing: as if left out; with any weight NaN, loss and gradient."""
    from ssm_b200 import ops

    vocab = 700
    x = torch.randn(6, vocab, generator=torch.Generator().manual_seed(0)).to(dtype).cuda().requires_grad_(True)
    ids = torch.tensor([[4, 5, vocab], [4, 5, vocab + 9], [vocab, vocab, vocab], [4, 5, -1], [4, 5, vocab], [vocab, -1, 4]]).cuda()
    teacher = torch.tensor([[0.0, 1.0, -INF], [0.0, 1.0, -30000.0], [-INF, -INF, -INF], [0.0, 1.0, 7.0], [0.0, 1.0, 0.5], [-INF, 3.0, -INF]]).to(dtype).cuda()
    loss = ops.topk_distill_loss(x, teacher, ids)
    d, = torch.autograd.grad(loss.sum(), x)
    left = ids.masked_fill(ids >= vocab, -1)
    left[4, 2] = 6
    want = ops.topk_distill_loss(x, teacher, left)
    ref, = torch.autograd.grad(want.sum(), x)
    for row in (0, 1, 2, 3, 5):
        assert torch.equal(loss[row], want[row]) and torch.equal(d[row], ref[row]), row
    assert torch.isnan(loss[4]) and torch.isnan(d[4]).all()
    assert loss[2] == 0 and not d[2].any() and loss[5] == 0 and not d[5].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_teacher_have_no_gradient_whatever_the_student_says(dtype):
    from ssm_b200 import ops

    x = torch.randn(3, 500, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, 7], x[1, 8] = NAN, INF
    x = x.cuda().requires_grad_(True)
    ids = torch.tensor([[-1, -1], [3, 4], [3, 4]]).cuda()
    teacher = torch.tensor([[1.0, 2.0], [-INF, -INF], [0.0, 1.0]]).cuda()
    loss = ops.topk_distill_loss(x, teacher, ids)
    d, = torch.autograd.grad(loss.sum(), x)
    assert loss[0] == 0 and loss[1] == 0 and not d[:2].any() and torch.isfinite(d[2]).all() and d[2].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 5000), (3, 40000), (400, 3000)])
def test_alternatives_of_rows_of_nan_start_at_the_first(rows, vocab, dtype):
    """More values of NaN than are kept as candidates, the first column among them; and one at the first column before thousands of ties."""
    from ssm_b200 import ops

    x = torch.zeros(rows, vocab)
    x[0] = NAN
    if rows > 1:
        x[1, ::2] = NAN
        x[2, 0] = NAN
        x[2, 1:2500] = torch.arange(2499).remainder(3).float()
    k = 20
    ids = ops.token_log_probs(x.to(dtype).cuda(), torch.zeros(rows, dtype=torch.long).cuda(), top_k=k)[2].cpu()
    assert torch.equal(ids[0], torch.arange(k))
    if rows > 1:
        assert torch.equal(ids[1], 2 * torch.arange(k))
        assert torch.equal(ids[2], torch.cat([torch.tensor([0]), torch.arange(k - 1) * 3 + 3]))


@pytest.mark.parametrize("value", [NAN, INF])
def test_a_teacher_that_is_not_finite_shows_in_loss_and_gradient(value):
    """Its weights are NaN, and with them every column of the row's gradient; the other rows as without it."""
    from ssm_b200 import ops

    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(True)
    ids = torch.tensor([[1, 2, 3], [3, 4, 5], [5, 6, -1]]).cuda()
    teacher = torch.tensor([[0.5, 0.0, 1.0], [0.0, value, 1.0], [0.0, 1.0, value]]).cuda()
    loss = ops.topk_distill_loss(x, teacher, ids)
    d, = torch.autograd.grad(loss.sum(), x)
    assert torch.isnan(loss[1]) and torch.isnan(d[1]).all()
    assert torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(d[[0, 2]]).all()  # an entry left out counts for nothing
