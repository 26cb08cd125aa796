"""GPU tests of the global gradient norm and clipping (gtk_grad_norm / gtk_clip_grad_norm)
against sums in 64 bits.

Tolerances, with u = 2^-24: sixteen squares are summed in fp32 (each rounded, at most 16 further
roundings), everything above in 64 bits; the root halves the relative error: the norm is off by
at most 9 u, and by 10 u after its own rounding. The factor adds one rounding, a scaled element
two, and a 16-bit result its half step."""

import math

import pytest
import torch

import genie_tk
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _make(shapes, dtypes, seed, dev, scale=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(s, generator=gen, device=dev) * scale).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(shapes)]


def _norm(grads, kind=2.0):
    if kind == math.inf:
        return max(float(g.double().abs().max()) for g in grads if g.numel())
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check_scaled(out, grad, k):
    ref = grad.double() * k
    tol = 13 * U * ref.abs()
    if out.dtype != torch.float32:
        tol = tol + torch.finfo(out.dtype).eps / 2 * (ref.abs() + tol)
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[out.dtype]
    assert ((out.double() - ref).abs() <= tol + tiny).all()


def _run(grads, factor, kind=2.0, out_dtypes=None):
    """Clip to `factor` times the norm: in place, and into other tensors."""
    from genie_tk import ops
    n = _norm(grads, kind)
    max_norm = n * factor
    k = min(1.0, max_norm / (n + 1e-6))
    assert abs(float(ops.grad_norm(grads, kind)) - n) <= 10 * U * n
    kept = [g.clone() for g in grads]
    outs = [torch.full_like(g, 7.0, dtype=out_dtypes[i % len(out_dtypes)] if out_dtypes else g.dtype,
                            memory_format=torch.contiguous_format) for i, g in enumerate(grads)]
    got = ops.clip_grad_norm(grads, max_norm, kind, out=outs)
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - n) <= 10 * U * n
    for g, c, o in zip(grads, kept, outs):
        assert torch.equal(g, c)
        _check_scaled(o, c, k)
    got = ops.clip_grad_norm(grads, max_norm, kind)
    assert abs(float(got) - n) <= 10 * U * n
    for g, c in zip(grads, kept):
        _check_scaled(g, c, k)
        if factor > 1:
            assert torch.equal(g, c)


SHAPES = [(128,), (128, 128), (1,), (7,), (3, 5, 11), (8191,), (8192,), (8193,), (4, 128), (100003,), (0,), (33, 65)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("factor", [0.1, 2.0])
def test_one_type(dtype, factor):
    dev = require_gpu()
    _run(_make(SHAPES, [dtype], 1, dev), factor)
    if dtype != torch.float32:
        _run(_make(SHAPES, [dtype], 2, dev), factor, out_dtypes=[torch.float32])


def test_mixed_types_and_the_largest_magnitude():
    dev = require_gpu()
    dts = [torch.float32, torch.bfloat16, torch.float16]
    for kind in (2.0, math.inf):
        _run(_make(SHAPES * 3, dts, 3, dev), 0.25, kind)
        _run(_make(SHAPES * 3, dts, 4, dev), 1.5, kind, out_dtypes=[torch.float32])


@pytest.mark.parametrize("n", [1, 2, 64, 65, 256, 257, 1000, 1001, 2500])
def test_number_of_tensors(n):
    """The table's sizes, and several launches from 1001 tensors on."""
    dev = require_gpu()
    gen = torch.Generator().manual_seed(n)
    shapes = [(int(x),) for x in torch.randint(1, 3000, (n,), generator=gen)]
    _run(_make(shapes, [torch.float32], n, dev), 0.3)
    _run(_make(shapes, [torch.bfloat16, torch.float32], n, dev), 0.3)


def test_alignments_and_strides():
    dev = require_gpu()
    for dtype in (torch.float32, torch.bfloat16):
        flat = _make([(300000,)], [dtype], 6, dev)[0]
        out = torch.zeros(300000, device=dev)
        views, outs, at = [], [], 0
        for i, n in enumerate([1, 2, 3, 9000, 5, 17, 40000, 7, 8192, 16385, 12345]):
            at += i % 4
            views.append(flat[at:at + n])
            outs.append(out[at + i % 3:at + i % 3 + n] if i < 1 else out[at:at + n])
            at += n
        _run(views, 0.2)
        from genie_tk import ops
        kept = [v.clone() for v in views]
        n = _norm(views)
        ops.clip_grad_norm(views, 0.5 * n, out=outs)
        for o, c in zip(outs, kept):
            _check_scaled(o, c, 0.5 * n / (n + 1e-6))
        untouched = torch.ones(300000, dtype=torch.bool, device=dev)
        for o in outs:
            a = o.storage_offset()
            untouched[a:a + o.numel()] = False
        assert not out[untouched].any()  # nothing beside the tensors is written
        # transposed (dense), every other column and expanded rows
        t = _make([(60, 70), (50, 40), (30, 64)], [dtype], 7, dev)
        _run([t[0].t(), t[1][:, ::2], t[2][3:9, 5:60]], 0.3)
        rest = t[1][:, 1::2].clone()
        ops.clip_grad_norm([t[1][:, ::2]], 1e-3)
        assert torch.equal(t[1][:, 1::2], rest)


def test_extreme_values():
    dev = require_gpu()
    from genie_tk import ops
    for scale in (1e30, 1e-30, 3e37, 1e-38):  # squares over- and underflow in fp32
        g = _make([(10007,), (64, 33)], [torch.float32], 8, dev, scale)
        n = _norm(g)
        got = float(ops.grad_norm(g))
        # 12,119 values of 3e37 have a norm of 3.3e39, above the largest fp32 (3.4e38): it rounds to inf
        assert got == math.inf if n > torch.finfo(torch.float32).max else abs(got - n) <= 10 * U * n + 2.0 ** -149
    mixed = [torch.full((5000,), 1e-25, device=dev), torch.ones(3, device=dev)]
    assert abs(float(ops.grad_norm(mixed)) - math.sqrt(3)) <= 10 * U * 2
    _run(_make([(10007,), (64, 33)], [torch.float32], 8, dev, 1e28), 0.01)
    zeros = [torch.zeros(9000, device=dev), torch.zeros(3, device=dev, dtype=torch.float16)]
    assert float(ops.clip_grad_norm(zeros, 1.0)) == 0.0 and not zeros[0].any()
    assert float(ops.grad_norm([torch.zeros(0, device=dev)])) == 0.0
    assert float(ops.clip_grad_norm([torch.zeros(0, device=dev)], 1.0)) == 0.0
    # max_norm 0 zeroes; max_norm infinite keeps
    g = _make([(100,)], [torch.float32], 9, dev)
    c = g[0].clone()
    ops.clip_grad_norm(g, math.inf)
    assert torch.equal(g[0], c)
    ops.clip_grad_norm(g, 0.0)
    assert not g[0].any()
    for kind in (2.0, math.inf):
        for bad, want in ((float("nan"), "nan"), (float("inf"), "inf"), (-float("inf"), "inf")):
            for at in (0, 5, 9999):
                g = _make([(50,), (10000,)], [torch.float32], 10, dev)
                g[1][at] = bad
                ref = [t.clone() for t in g]
                n = ops.clip_grad_norm(g, 1.0, kind)
                assert str(abs(float(n))) == want
                if want == "nan":
                    assert g[0].isnan().all() and g[1].isnan().all()
                else:  # factor 0: finite elements become 0, inf * 0 is NaN
                    assert not g[0].any() and g[1][at].isnan() and int(g[1].isnan().sum()) == 1
                torch.nn.utils.clip_grad_norm_([_param(t) for t in ref], 1.0, kind)
                assert torch.equal(ref[0].isnan(), g[0].isnan())


def _param(g):
    p = torch.nn.Parameter(torch.zeros_like(g))
    p.grad = g
    return p


def test_beside_torch_on_a_module():
    dev = require_gpu()
    torch.manual_seed(1)
    net = genie_tk.PairTransformLayer(128).to(dev)
    grads = [torch.randn_like(p) for p in net.parameters()]
    for f in (0.05, 3.0):
        for kind in (2.0, math.inf):
            for p, g in zip(net.parameters(), grads):
                p.grad = g.clone()
            max_norm = f * _norm(grads, kind)
            ref = torch.nn.utils.clip_grad_norm_(net.parameters(), max_norm, kind)
            want = [p.grad for p in net.parameters()]
            for p, g in zip(net.parameters(), grads):
                p.grad = g.clone()
            got = genie_tk.clip_grad_norm_(net.parameters(), max_norm, kind)
            torch.testing.assert_close(got, ref, rtol=1e-5, atol=0)  # torch sums in fp32
            for p, w in zip(net.parameters(), want):
                torch.testing.assert_close(p.grad, w, rtol=1e-5, atol=0)
    p = next(net.parameters())
    before = p.grad.clone()
    v = p.grad._version
    genie_tk.clip_grad_norm_(p, 1e-3)
    assert p.grad._version > v
    p.grad = before.clone()
    p.grad.view(-1)[0] = float("inf")
    kept = p.grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        genie_tk.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad, kept)


def test_same_bits_on_streams_and_from_graphs():
    dev = require_gpu()
    from genie_tk import ops
    g1 = _make(SHAPES * 20, [torch.float32], 11, dev)
    g2 = _make(SHAPES * 20, [torch.bfloat16], 12, dev)
    o1, o2 = [torch.empty_like(g) for g in g1], [torch.empty_like(g) for g in g2]
    want1, want2 = ops.clip_grad_norm(g1, 3.0, out=o1), ops.clip_grad_norm(g2, 5.0, out=o2)
    r1, r2 = [o.clone() for o in o1], [o.clone() for o in o2]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    norms = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            norms.append((ops.clip_grad_norm(g1, 3.0, out=o1), want1))
        with torch.cuda.stream(s2):
            norms.append((ops.clip_grad_norm(g2, 5.0, out=o2), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in norms)
    assert all(torch.equal(a, b) for a, b in zip(o1 + o2, r1 + r2))
    graphs = []
    for g, o, m in ((g1, o1, 3.0), (g2, o2, 5.0)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            n = ops.clip_grad_norm(g, m, out=o)
        graphs.append((gr, n))
    for o in o1 + o2:
        o.zero_()
    for _ in range(2):
        for gr, _ in graphs:
            gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want1) and torch.equal(graphs[1][1], want2)
    assert all(torch.equal(a, b) for a, b in zip(o1 + o2, r1 + r2))


def test_more_than_2_31_elements():
    dev = require_gpu()
    from genie_tk import ops
    n = (1 << 31) + 5001
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    g[-3:] = 2.0
    g[: 1 << 20] = 0.5
    want = math.sqrt(12.0 + 0.25 * (1 << 20))
    got = ops.clip_grad_norm([g], want / 4)
    assert abs(float(got) - want) <= 10 * U * want
    assert (g[-3:] == 0.5).all() and (g[: 1 << 20] == 0.125).all() and not g[1 << 20:-3].any()


def test_refusals():
    dev = require_gpu()
    from genie_tk import ops
    g = torch.randn(100, device=dev)
    kept = g.clone()
    for bad in ([g, g], [g[:60], g[50:]], [g[50:], g[:60]]):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_grad_norm(bad, 1.0)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.clip_grad_norm([g[:50], g[50:]], 1.0, out=[g[50:], g[:50]])
    with pytest.raises(RuntimeError, match="one device"):
        ops.clip_grad_norm([g, torch.randn(3)], 1.0)
    with pytest.raises(TypeError):
        ops.clip_grad_norm([g.double()], 1.0)
    with pytest.raises(TypeError):
        ops.clip_grad_norm([g], 1.0, out=[g.half()])
    with pytest.raises(TypeError):
        ops.clip_grad_norm([g.to_sparse()], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grad_norm([g], 1.0, out=[])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([g], 1.0, out=[g[:50]])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([g.view(10, 10)], 1.0, out=[torch.empty(10, 20, device=dev)[:, ::2]])
    with pytest.raises(ValueError):
        ops.grad_norm([g], 1.0)
    with pytest.raises(ValueError, match="more than once"):
        ops.clip_grad_norm([g, torch.randn(1, 4, device=dev).expand(3, 4)], 1e-3)
    with pytest.raises(TypeError, match="dense"):  # a lazily negated view
        ops.grad_norm([torch.zeros(4, dtype=torch.complex64, device=dev).conj().imag])
    assert torch.equal(g, kept)
    # read only, an expanded gradient is as good as any
    e = torch.randn(1, 4, device=dev).expand(3, 4)
    torch.testing.assert_close(ops.grad_norm([e]), e.double().norm().float(), rtol=1e-6, atol=0)
