"""GPU tests of the lists that the gradient norm and clipping take: views that overlap in memory,
refused calls, sequences that make their items, copies on write, and factors below fp32's range.

Tolerances as in test_gpu_grad_clip.py."""

import math
import random

import pytest
import torch

import genie_tk
from gpu_util import require_gpu
from test_gpu_grad_clip import U, _check_scaled, _make, _norm

pytestmark = pytest.mark.gpu


def test_strided_gradients_that_overlap_are_refused():
    """A view that is neither contiguous nor dense is clipped through a copy; what counts is the
    memory it stands for."""
    dev = require_gpu()
    from genie_tk import ops
    a = _make([(12, 10)], [torch.float32], 1, dev)[0]
    kept = a.clone()
    flat = a.view(-1)
    for bad in ([a[:, ::2], a[:, ::2]], [a, a[:, ::2]], [a[:, 3:6], a[:, 5:8]], [a[2:5, 1:9], a[4:, 8:]],
                [a[::2, :3], flat[40:42]], [a[:, ::3], a[:, 1::2]], [a[3:7].t()[::3], a[5]],
                [a[:6, :5], a[6:, :5], a[5:7, 4:]]):
        for order in (bad, bad[::-1]):
            with pytest.raises(RuntimeError, match="overlap"):
                ops.clip_grad_norm(order, 1e-3)
    # windows that share elements with one another
    for windows in (flat.as_strided((20, 4), (2, 1)), flat.as_strided((5, 3, 4), (20, 6, 2))):
        with pytest.raises(ValueError, match="more than once"):
            ops.clip_grad_norm([windows], 1e-3)
    # outputs on a strided gradient: on its own, on another's, in the gaps of none
    other = torch.zeros(12, 5, device=dev)
    for grads, outs in (([a[:, ::2]], [flat[:60].view(12, 5)]), ([a[:, ::2], other], [torch.empty_like(other), flat[30:90].view(12, 5)]),
                        ([a[:, :5], other], [torch.empty_like(other), a[6:, :].view(12, 5)])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_grad_norm(grads, 1e-3, out=outs)
    torch.cuda.synchronize()
    assert torch.equal(a, kept) and not other.any()
    # read only, they may
    n = math.sqrt(2) * float(a[:, ::2].double().norm())
    assert abs(float(ops.grad_norm([a[:, ::2], a[:, ::2]])) - n) <= 10 * U * n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_gradients_beside_one_another(dtype):
    """Views that share a buffer and no element: columns and rows in turn, blocks, planes."""
    dev = require_gpu()
    from genie_tk import ops
    a = _make([(24, 30)], [dtype], 2, dev)[0]
    b = _make([(6, 8, 10)], [dtype], 3, dev)[0]
    e = _make([(4, 6, 6, 5)], [dtype], 4, dev)[0]
    lists = [[a[:, ::2], a[:, 1::2]], [a[:, :7], a[:, 7:20], a[:, 20:]], [a[::3, 4:9], a[1::3, 2:11], a[2::3, :30:4]],
             [a[:11, 13:], a[11:, :13], a[:11, :13], a[11:, 13:]], [b[:, :2, :2], b[:, 2:, 1:]],
             [b[:, 1::2].transpose(0, 1), b[:, ::2]], [e[:, :, ::2, 1:], e[:, :, 1::2, 1:], e[:, ::2, :, 0], e[:, 1::2, :, 0]],
             [a[:, c] for c in range(30)], [a.view(-1).as_strided((4, 5), (31, 7)), a[20:]],
             [a.view(-1).as_strided((4, 5), (3, 4)), a[1:]]]  # 3 i + 4 j: a number twice would take four rows apart
    for views in lists:
        base = views[0]._base
        before, kept, n = base.clone(), [v.clone() for v in views], _norm(views)
        k = min(1.0, 0.25 * n / (n + 1e-6))
        outs = [torch.empty_like(v, memory_format=torch.contiguous_format) for v in views]
        ops.clip_grad_norm(views, 0.25 * n, out=outs)
        assert torch.equal(base, before)
        got = ops.clip_grad_norm(views, 0.25 * n)
        assert abs(float(got) - n) <= 10 * U * n
        touched = torch.zeros_like(base)
        for v, c, o in zip(views, kept, outs):
            _check_scaled(v, c, k)
            _check_scaled(o, c, k)
            assert torch.equal(v, o)
            touched.as_strided(v.shape, v.stride(), v.storage_offset() - base.storage_offset()).fill_(1)
        assert torch.equal(base[touched == 0], before[touched == 0])
        base.copy_(before)


def test_many_columns_of_one_buffer():
    """Some hundred interleaved views: the check of their memory goes by pairs that span the same
    addresses, and stays short."""
    dev = require_gpu()
    from genie_tk import ops
    a = torch.ones(3000, 300, device=dev)
    ops.clip_grad_norm([a[:, c] for c in range(300)], 3.0)
    assert abs(float(a.double().norm()) - 3.0) <= 1e-5
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm([a[:, c] for c in range(300)] + [a[2999, 299:]], 3.0)
    b = torch.ones(3, 1700, device=dev)  # 1.4 million pairs
    ops.clip_grad_norm([b[:, c] for c in range(1700)], 3.0)
    assert abs(float(b.double().norm()) - 3.0) <= 1e-5


def test_refused_calls_leave_the_versions():
    """A refused call has written nothing, and autograd must not think that it had."""
    dev = require_gpu()
    from genie_tk import ops
    g = [torch.randn(6, 5, device=dev) for _ in range(3)]
    o = [torch.empty(6, 5, device=dev) for _ in range(3)]
    s = torch.randn(6, 10, device=dev)
    before = [t._version for t in g + o + [s]]
    calls = [lambda: ops.clip_grad_norm([g[0], s[:, ::2], g[1].double()], 1.0), lambda: ops.clip_grad_norm([g[0], g[0]], 1.0),
             lambda: ops.clip_grad_norm([g[0], 1.0], 1.0), lambda: ops.clip_grad_norm(g[:2], 1.0, out=[o[0], o[1].half()]),
             lambda: ops.clip_grad_norm(g[:2], 1.0, out=[o[0], o[0]]), lambda: ops.clip_grad_norm(g[:2], 1.0, out=[o[0], s[:, ::2]])]
    for call in calls:
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            call()
        assert [t._version for t in g + o + [s]] == before
    ops.clip_grad_norm(g[:2] + [s[:, ::2]], 1.0)
    assert all(t._version > v for t, v in zip(g[:2] + [s], before[:2] + before[-1:])) and g[2]._version == before[2]
    ops.clip_grad_norm(g, 1.0, out=o)
    assert all(t._version > v for t, v in zip(o, before[3:])) and g[2]._version == before[2]
    # the same through autograd: a saved tensor that a refused call named is as it was
    x = torch.randn(7, device=dev, requires_grad=True)
    y = x.detach().clone()
    loss = (x * y).sum()
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm([y, y], 1.0)
    loss.backward()
    assert torch.equal(x.grad, y)


class _Made:
    """A sequence that makes each item when it is asked for and keeps none."""

    def __init__(self, base):
        self.base = base

    def __len__(self):
        return len(self.base)

    def __getitem__(self, i):
        if i >= len(self.base):
            raise IndexError(i)
        return self.base[i].clone()


@pytest.mark.parametrize("n", [100, 2432, 5000])
def test_sequences_that_make_their_items(n):
    """The gradients of such a sequence live until the call has been queued: 2432 fp32 elements are
    as many bytes as the workspace, which would otherwise be given their memory."""
    dev = require_gpu()
    from genie_tk import ops
    base = _make([(n,), (n,)], [torch.float32], 5, dev)
    for grads in (base[:1], base):
        total = _norm(grads)
        torch.cuda.synchronize()
        outs = [torch.empty_like(g) for g in grads]
        got = ops.clip_grad_norm(_Made(grads), 0.5 * total, out=outs)
        assert abs(float(got) - total) <= 10 * U * total
        for o, g in zip(outs, grads):
            _check_scaled(o, g, 0.5 * total / (total + 1e-6))
        assert abs(float(ops.grad_norm(_Made(grads))) - total) <= 10 * U * total


def test_copies_on_write():
    """Clipping a lazy clone leaves its source, and two lazy clones are two tensors."""
    dev = require_gpu()
    from genie_tk import ops
    src = torch.randn(1000, device=dev)
    kept = src.clone()
    a, b = torch._lazy_clone(src), torch._lazy_clone(src)
    n = _norm([a, b])
    ops.clip_grad_norm([a, b], 0.5 * n)
    assert torch.equal(src, kept)
    for t in (a, b):
        _check_scaled(t, kept, 0.5 * n / (n + 1e-6))


@pytest.mark.parametrize("out", [None, torch.float32, "same"])
@pytest.mark.parametrize("n", [1003, 2100007])
def test_factors_below_the_fp32_range(n, out):
    """Values near fp32's largest under a small limit: the factor is below 2^-126, where fp32 has
    fewer bits, or below 2^-150, where it has none; the scaled values are ordinary numbers."""
    dev = require_gpu()
    from genie_tk import ops
    for dtype in (torch.float32, torch.bfloat16):
        for limit in (1e3, 1e-1, 1e-5):
            gen = torch.Generator(device=dev).manual_seed(n)
            g = ((torch.rand(n, generator=gen, device=dev) + 1) * 1.2e38).to(dtype)[1:]
            kept = g.clone()
            norm = _norm([g])
            if out is None:
                ops.clip_grad_norm([g], limit)
                got = g
            else:
                got = torch.empty(n - 1, device=dev, dtype=dtype if out == "same" else out)
                ops.clip_grad_norm([g], limit, out=[got])
                assert torch.equal(g, kept)
            _check_scaled(got, kept, limit / norm)


def test_random_views_against_their_elements():
    """Random views of one buffer: refused exactly where two share an element, or one holds an element
    twice."""
    dev = require_gpu()
    from genie_tk import ops
    rng = random.Random(1)
    base = torch.zeros(400, device=dev)
    number = torch.arange(400)
    seen = {"apart": 0, "overlap": 0, "twice": 0}
    for _ in range(600):
        views, places = [], []
        for _ in range(rng.choice([1, 2, 2])):
            while True:
                dims = rng.randint(1, 3)
                size, stride = [rng.randint(1, 6) for _ in range(dims)], [rng.randint(1, 40) for _ in range(dims)]
                at = rng.randint(0, 60)
                if at + sum((n - 1) * s for n, s in zip(size, stride)) < 400:
                    break
            views.append(base.as_strided(size, stride, at))
            places.append(number.as_strided(size, stride, at).reshape(-1).tolist())
        twice = any(len(set(p)) < len(p) for p in places)
        overlap = len(places) > 1 and set(places[0]) & set(places[1])
        if twice:
            with pytest.raises(ValueError, match="more than once"):
                ops.clip_grad_norm(views, 1.0)
        elif overlap:
            with pytest.raises(RuntimeError, match="overlap"):
                ops.clip_grad_norm(views, 1.0)
        else:
            ops.clip_grad_norm(views, 1.0)
        seen["twice" if twice else "overlap" if overlap else "apart"] += 1
    assert min(seen.values()) > 50, seen
