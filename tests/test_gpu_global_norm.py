"""``ops.global_norm`` and ``ops.clip_global_norm_`` against 64 bits.

Tolerances.  Sixteen bytes' squares are added in fp32, four such sums too: at most 16 roundings of 2^-24 on terms of one sign, 1e-6 of the sum, half of that of its
root; the rest is fp64, and the root is rounded to fp32: 6e-7 in all.  A clipped element is off by that, the roundings of the factor (three of 2^-24) and
half a step of its type."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import training_oracle as oracle
from ssm_b200 import ops

pytestmark = pytest.mark.gpu
REL = 6e-7


def rn(*shape, dtype=torch.float32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=gen)).to(dtype)


def same(got, want):
    assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
    assert float(got) == float(want) or abs(float(got) - float(want)) <= REL * float(want), (float(got), float(want))  # equal where beyond 32 bits


def clip(tensors, limit, **kw):
    before = [t.detach().double() for t in tensors]
    want = oracle.global_norm([t.cpu() for t in tensors], **kw)
    got = ops.clip_global_norm_(tensors, limit, **kw)
    same(got, want)
    c = min(1.0, limit / (float(want) + 1e-6))
    for t, b in zip(tensors, before):
        eps = torch.finfo(t.dtype).eps / 2
        tiny = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps / 2
        assert ((t.double() - b * c).abs() <= (eps + REL + 4e-7) * (b * c).abs() + tiny).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 255, 4096, 8191, 8192, 8193, 100003, 3000001])
def test_sizes(dtype, n):
    t = rn(n, dtype=dtype)
    same(ops.global_norm([t]), oracle.global_norm(t.cpu()))
    same(ops.global_norm(t, math.inf), oracle.global_norm(t.cpu(), math.inf))
    clip([t], 0.25 * float(t.double().norm()))


@pytest.mark.parametrize("count", [2, 37, 1024, 1025, 2600])
def test_many_tensors_of_mixed_types(count):
    types = [torch.float32, torch.bfloat16, torch.float16]
    tensors = [rn(1 + (i * 37) % 501, dtype=types[i % 3], seed=i, scale=10.0 ** (i % 5 - 2)) for i in range(count)]
    same(ops.global_norm(tensors), oracle.global_norm([t.cpu() for t in tensors]))
    same(ops.global_norm(tensors, math.inf), oracle.global_norm([t.cpu() for t in tensors], math.inf))
    clip(tensors, 1.5)
    clip(tensors, 0.5, norm_type=math.inf)


@pytest.mark.parametrize("offset", range(9))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_places_that_are_not_aligned_and_what_lies_around_them(offset, dtype):
    for n in (1, 3, 6, 50, 9000):
        whole = rn(n + 20, dtype=dtype, seed=offset)
        kept = whole.clone()
        t = whole[offset:offset + n]
        clip([t], 1e-3)
        assert torch.equal(whole[:offset], kept[:offset]) and torch.equal(whole[offset + n:], kept[offset + n:])


def test_nothing_is_written_where_nothing_is_clipped():
    tensors = [rn(1000, seed=1), rn(500, dtype=torch.bfloat16, seed=2)]
    kept = [t.clone() for t in tensors]
    norm = float(ops.global_norm(tensors))
    for limit in (2 * norm, math.inf, norm * 1.001):
        same(ops.clip_global_norm_(tensors, limit), norm)
        assert all(torch.equal(a, b) for a, b in zip(tensors, kept))
    ops.clip_global_norm_(tensors, 0.0)
    assert not any(t.any() for t in tensors)


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e-19, 3e18, 1e25, 2e37])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_whose_squares_32_bits_cannot_hold(scale, dtype):
    t = rn(50, dtype=dtype, scale=scale)
    mixed = [rn(5000, dtype=dtype, scale=scale), torch.zeros(3000, device="cuda"), rn(3, scale=scale)]
    same(ops.global_norm([t]), oracle.global_norm(t.cpu()))
    same(ops.global_norm(mixed), oracle.global_norm([x.cpu() for x in mixed]))


def test_values_that_are_not_finite():
    for bad in (math.inf, -math.inf):
        t = [rn(5000, seed=3), rn(100, seed=4)]
        t[0][77] = bad
        assert float(ops.global_norm(t)) == math.inf and float(ops.global_norm(t, math.inf)) == math.inf
        assert float(ops.clip_global_norm_(t, math.inf)) == math.inf and t[1].any()
        assert float(ops.clip_global_norm_(t, 1.0)) == math.inf
        assert t[0][77].isnan() and not t[0][:77].any() and not t[1].any()
    t = [rn(5000, seed=3), rn(100, seed=4)]
    t[0][4999], t[0][3] = math.nan, math.inf
    for kind in (2.0, math.inf):
        assert ops.global_norm(t, kind).isnan() and ops.global_norm(t[::-1], kind).isnan()
    ops.clip_global_norm_(t, 1.0)
    assert t[0].isnan().all() and t[1].isnan().all()


def test_layouts():
    base = rn(64, 33)
    clip([base.t()], 1.0)  # dense in another order
    wide = rn(40, 64, seed=1)
    kept = wide.clone()
    clip([wide[:, ::2]], 1.0)  # gaps
    assert torch.equal(wide[:, 1::2], kept[:, 1::2])
    same(ops.global_norm([wide[0].expand(5, 64)]), float(wide[0].double().norm()) * math.sqrt(5))
    same(ops.global_norm([base, base]), float(base.double().norm()) * math.sqrt(2))
    same(ops.global_norm([torch.empty(0, 4, device="cuda"), base]), oracle.global_norm(base.cpu()))
    assert float(ops.global_norm([])) == 0.0 and float(ops.clip_global_norm_([], 1.0)) == 0.0
    assert float(ops.global_norm([torch.empty(0, device="cuda")])) == 0.0


def test_refusals_on_the_gpu():
    a = rn(10, 10)
    for bad in ([a, a], [a, a[3]], [a[:6], a[5:]]):
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_global_norm_(bad, 1.0)
    ops.clip_global_norm_([a[:5], a[5:]], 1.0)
    with pytest.raises(ValueError, match="broadcast"):
        ops.clip_global_norm_([a[0].expand(4, 10)], 1.0)
    with pytest.raises(ValueError, match="no gradient flows"):
        ops.global_norm([a.clone().requires_grad_(True)])
    with torch.no_grad():
        ops.global_norm([a.clone().requires_grad_(True)])
    with pytest.raises(ValueError, match="not built"):
        ops.global_norm([a.double()])
    with pytest.raises((ValueError, RuntimeError)):
        ops.global_norm([a, a.cpu()])


def test_a_graph_notices_that_its_tensor_was_clipped():
    w = rn(8).requires_grad_(True)
    loss = (w * w).sum()
    with torch.no_grad():
        ops.clip_global_norm_([w], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_repeats_streams_and_graphs_give_the_same_bits():
    fresh = [rn(70001, seed=5), rn(333, 77, dtype=torch.bfloat16, seed=6), rn(5, seed=7)]
    work = [t.clone() for t in fresh]

    def once():
        for w, f in zip(work, fresh):
            w.copy_(f)
        return ops.clip_global_norm_(work, 1.0)

    norm, want = once(), [w.clone() for w in work]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert float(once()) == float(norm)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(work, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for _ in range(3):
        held.zero_()
        graph.replay()
        assert torch.equal(held, norm) and all(torch.equal(a, b) for a, b in zip(work, want))
    fresh[0].mul_(100)
    graph.replay()
    same(held, oracle.global_norm([t.cpu() for t in fresh]))


def test_views_of_one_buffer_that_lie_between_one_another():
    """Columns of one matrix, every second element, planes of the last axis: their spans overlap, their elements do not."""
    def pieces(kind):
        m = rn(64, 40, seed=3)
        return m, {"columns": [m[:, :13], m[:, 13:20], m[:, 20:]], "every second": [m[:, 1::2], m[:, ::2]], "rows and columns": [m[:32, :8], m[32:], m[:32, 8:]],
                   "planes": [m.view(64, 8, 5)[..., i] for i in range(5)], "blocks": [m.view(16, 4, 40)[:, :1, :7], m.view(16, 4, 40)[:, 1:, :7], m[:, 7:]],
                   "turned": [m.t()[:13], m.t()[13:]], "one column": [m[:, 0], m[:, 1:]]}[kind]

    for kind in ("columns", "every second", "rows and columns", "planes", "blocks", "turned", "one column"):
        m, parts = pieces(kind)
        kept = m.clone()
        clip(parts, 1.0)
        c = min(1.0, 1.0 / (float(torch.cat([p.reshape(-1) for p in pieces(kind)[1]]).double().norm()) + 1e-6))
        assert torch.allclose(m, kept * c, rtol=2e-6, atol=0), kind


def test_views_of_one_buffer_that_share_elements_are_refused():
    m = rn(64, 40, seed=3)
    kept = m.clone()
    for bad in ([m[:, :20], m[:, 19:]], [m[:, ::2], m[:, ::4]], [m[:, 3:], m[5]], [m[5], m[9, 2:7], m[:, 3:]], [m.t()[:5], m[:, 4:]], [m[:, 0], m[:, 5], m[40:, :6]], [m[::2], m[2::4]]):
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_global_norm_(bad, 1.0)
    assert torch.equal(m, kept)
