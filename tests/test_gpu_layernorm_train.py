"""GPU tests of LayerNorm's training form (gtk_layernorm_forward / gtk_layernorm_backward) against
the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and h the half step of the output's type:
a mean over D elements is summed 16 or 32 per thread and then in a tree of at most 9 + 16 steps,
so it is off by at most 60 u mean|x| (the wide rows: D / 512 + 25 steps, 120 u at the sizes here).
From it, xhat is off by e = N u (rstd mean|x| + rstd max|x - mean| + |xhat|) with N = 64 (128), and
the other bounds follow by counting each rounding once (see ``_bounds``). A 16-bit result adds
h |value|."""

import pytest
import torch

import genie_tk
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _reference(x, w, b, dy, eps=EPS):
    x, dy = x.double(), dy.double()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps) ** -0.5
    xh = (x - mean) * rstd
    g = dy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    lead = tuple(range(x.dim() - 1))
    return {"mean": mean.squeeze(-1), "rstd": rstd.squeeze(-1), "y": xh * w + b, "dx": rstd * (g - c1 - xh * c2),
            "dw": (dy * xh).sum(lead), "db": dy.sum(lead), "x": x, "xh": xh, "g": g, "c1": c1, "c2": c2, "w": w, "b": b,
            "dy": dy, "rs": rstd}


def _bounds(r, dtype, pdtype):
    D = r["x"].shape[-1]
    rows = max(1, r["x"].numel() // D)
    N = 64 if D <= 16384 else 128
    ax = r["x"].abs().mean(-1, keepdim=True)
    dev = (r["xh"].abs() / r["rs"]).amax(-1, keepdim=True)
    e = N * U * (r["rs"] * ax + r["rs"] * dev + r["xh"].abs())
    em = e.mean(-1, keepdim=True)
    ga, gx = r["g"].abs().mean(-1, keepdim=True), (r["g"] * r["xh"]).abs().mean(-1, keepdim=True)
    lead = tuple(range(r["x"].dim() - 1))
    tree = (64 + rows / 148) * U
    b = {
        "mean": (N * U * ax).squeeze(-1),
        "rstd": (r["rs"] * N * U * (1 + r["rs"] * ax)).squeeze(-1),
        "y": e * r["w"].abs() + 4 * U * (r["y"].abs() + r["b"].abs()),
        # g is off by u|g|, c1 by N u mean|g|, c2 by N u mean|g xh| + mean|g| e
        "dx": r["rs"] * (8 * U * r["g"].abs() + N * U * ga + r["xh"].abs() * (N * U * gx + ga * em.clamp_min(0)
                         + (r["g"].abs() * e).mean(-1, keepdim=True)) + 2 * e * r["c2"].abs())
              + N * U * (1 + r["rs"] * ax) * r["dx"].abs(),
        "dw": (r["dy"].abs() * e).sum(lead) + tree * (r["dy"] * r["xh"]).abs().sum(lead),
        "db": tree * r["dy"].abs().sum(lead),
    }
    for k, t in (("y", dtype), ("dx", dtype), ("dw", pdtype), ("db", pdtype)):
        b[k] = b[k] + _half(t) * (r[k].abs() + b[k])
        if t is torch.float16:
            b[k] = b[k] + 2.0 ** -25  # below 2^-14 fp16 has fixed steps of 2^-24
    return b


def _check(got, ref, bound, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - ref).abs() > bound
    assert not bad.any(), (what, float(((got - ref).abs() / bound.clamp_min(1e-300)).max()))


def _inputs(shape, dtype, pdtype, seed, dev):
    gen = torch.Generator(device=dev).manual_seed(seed)
    D = shape[-1]
    x = (torch.randn(shape, generator=gen, device=dev) * 1.5 + torch.randn(D, generator=gen, device=dev)).to(dtype)
    dy = torch.randn(shape, generator=gen, device=dev).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=gen, device=dev)).to(pdtype)
    b = torch.randn(D, generator=gen, device=dev).to(pdtype)
    return x, dy, w, b


def _run_and_check(x, dy, w, b, eps=EPS):
    from genie_tk import ops
    y, mean, rstd = ops.layernorm_forward(x, w, b, eps)
    dx, dw, db = ops.layernorm_backward(dy, x, w, mean, rstd)
    assert y.dtype == x.dtype and dx.dtype == x.dtype and y.is_contiguous() and dx.is_contiguous()
    pdtype = x.dtype if w is None else w.dtype
    assert dw.dtype == pdtype and db.dtype == pdtype
    r = _reference(x, w, b, dy, eps)
    bound = _bounds(r, x.dtype, pdtype)
    for k, t in (("y", y), ("mean", mean), ("rstd", rstd), ("dx", dx), ("dw", dw), ("db", db)):
        _check(t, r[k], bound[k], k)


@pytest.mark.parametrize("dtype,pdtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                          ("f16", "f32")])
@pytest.mark.parametrize("rows,D", [(1, 8), (2, 9), (1, 384), (5, 33), (37, 384), (300, 128), (2000, 16), (257, 1000),
                                    (65, 512), (66, 520), (64, 1024), (700, 2048), (9, 5003), (5, 8192), (3, 8193),
                                    (4, 8200), (4, 16384), (5, 8185), (5, 8191), (3, 16377), (3, 16379), (3, 16385), (2, 40000)])
def test_matches_the_formula(rows, D, dtype, pdtype):
    dev = require_gpu()
    x, dy, w, b = _inputs((rows, D), DT[dtype], DT[pdtype], rows * 7 + D, dev)
    _run_and_check(x, dy, w, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_many_rows(dtype):
    """More rows than the grid has groups, with a last turn that is not full."""
    dev = require_gpu()
    for rows, D in ((100003, 40), (20011, 128), (6007, 777), (50001, 37), (3001, 1001), (5000, 513), (2999, 2050)):
        _run_and_check(*_inputs((rows, D), DT[dtype], torch.float32, rows, dev))


@pytest.mark.parametrize("D", [1, 2, 3])
def test_shortest_rows(D):
    """One element: xhat is 0, y the bias and dx exactly 0. Two or three: the forward holds;
    their dx nearly cancels, which the bound takes in through c2."""
    dev = require_gpu()
    from genie_tk import ops
    x, dy, w, b = _inputs((50, D), torch.float32, torch.float32, D, dev)
    _run_and_check(x, dy, w, b)
    if D == 1:
        y, mean, rstd = ops.layernorm_forward(x, w, b)
        dx, dw, _ = ops.layernorm_backward(dy, x, w, mean, rstd)
        assert torch.equal(y, b.expand_as(y)) and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,D", [(1, 9, 128), (2, 7, 128), (3, 5, 33), (2, 6, 64), (1, 8, 128), (2, 37, 96),
                                   (1, 70, 600)])
def test_transposed_pair_axes_are_read_in_place(B, N, D, dtype):
    dev = require_gpu()
    x, dy, w, b = _inputs((B, N, N, D), DT[dtype], torch.float32, N, dev)
    _run_and_check(x.transpose(1, 2), dy.transpose(1, 2), w, b)
    _run_and_check(x.transpose(1, 2), dy, w, b)
    _run_and_check(x, dy.transpose(1, 2), w, b)


def test_other_strides_and_alignments():
    dev = require_gpu()
    for dtype in (torch.float32, torch.bfloat16):
        x, dy, w, b = _inputs((6, 5, 4, 3, 64), dtype, torch.float32, 3, dev)
        _run_and_check(x.permute(3, 1, 0, 2, 4), dy.permute(3, 1, 0, 2, 4), w, b)  # four levels: copied
        _run_and_check(x[:, ::2], dy[:, ::2], w, b)
        big, dbig, w, b = _inputs((40, 131), dtype, torch.float32, 5, dev)
        for a, n in ((0, 128), (1, 128), (2, 64), (3, 100)):  # rows at odd offsets
            _run_and_check(big[:, a:a + n], dbig[:, a:a + n], w[a:a + n], b[a:a + n])
        flat = big.reshape(-1)[1:1 + 39 * 128].view(39, 128)  # contiguous, base not on 16 bytes
        _run_and_check(flat, dbig[:39, :128], w[:128], b[:128])
        # gradient of a mean: every row's dy is the same memory, or one number
        _run_and_check(big[:, :128], dbig[:1, :128].expand(40, 128), w[:128], b[:128])
        _run_and_check(big[:, :128], dbig[:1, :1].expand(40, 128), w[:128], b[:128])


def test_without_parameters_and_parts_of_the_gradients():
    dev = require_gpu()
    from genie_tk import ops
    x, dy, w, b = _inputs((77, 128), torch.float32, torch.float32, 1, dev)
    _run_and_check(x, dy, None, None)
    _run_and_check(x, dy, w, None)
    _, mean, rstd = ops.layernorm_forward(x, w, b)
    full = ops.layernorm_backward(dy, x, w, mean, rstd)
    for nw in (True, False):
        for nb in (True, False):
            got = ops.layernorm_backward(dy, x, w, mean, rstd, nw, nb)
            assert torch.equal(got[0], full[0])
            assert (got[1] is None) == (not nw) and (got[2] is None) == (not nb)
            assert not nw or torch.equal(got[1], full[1])
            assert not nb or torch.equal(got[2], full[2])


def test_extreme_values():
    """A mean far above the deviation loses no more than the type's step of the mean; constant
    rows have rstd = eps^-1/2; a NaN or infinity stays in its row (and in dw, db)."""
    dev = require_gpu()
    from genie_tk import ops
    x, dy, w, b = _inputs((40, 256), torch.float32, torch.float32, 8, dev)
    _run_and_check(x + 1000.0, dy, w, b)
    _run_and_check(x * 1e-4, dy, w, b)
    _run_and_check(x * 1e6, dy * 1e-6, w, b)
    y, mean, rstd = ops.layernorm_forward(torch.full((3, 256), 7.0, device=dev), w, b)
    assert torch.equal(mean, torch.full_like(mean, 7.0)) and torch.equal(y, b.expand_as(y))
    torch.testing.assert_close(rstd, torch.full_like(rstd, EPS ** -0.5), rtol=1e-6, atol=0)
    bad = x.clone()
    bad[3, 5], bad[9, 0] = float("nan"), float("inf")
    y, mean, rstd = ops.layernorm_forward(bad, w, b)
    dx, dw, db = ops.layernorm_backward(dy, bad, w, mean, rstd)
    keep = torch.ones(40, dtype=torch.bool, device=dev)
    keep[3] = keep[9] = False
    clean = ops.layernorm_forward(x, w, b)
    cdx, _, cdb = ops.layernorm_backward(dy, x, w, *clean[1:])
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], cdx[keep])
    assert y[3].isnan().all() and dx[3].isnan().all() and y[9].isnan().any()
    assert dw.isnan().all() and torch.equal(db, cdb)


def test_empty_inputs():
    dev = require_gpu()
    from genie_tk import ops
    x = torch.empty(0, 5, 128, device=dev)
    w = torch.ones(128, device=dev)
    y, mean, rstd = ops.layernorm_forward(x, w, w)
    assert y.shape == x.shape and mean.shape == (0, 5)
    dx, dw, db = ops.layernorm_backward(x, x, w, mean, rstd)
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_same_bits_every_time_on_any_stream_and_from_graphs():
    dev = require_gpu()
    from genie_tk import ops
    x, dy, w, b = _inputs((3001, 384), torch.bfloat16, torch.float32, 4, dev)

    def step(x, dy):
        y, mean, rstd = ops.layernorm_forward(x, w, b)
        return (y, mean, rstd) + ops.layernorm_backward(dy, x, w, mean, rstd)

    want = step(x, dy)
    x2, dy2 = x.flip(0).contiguous(), dy.flip(1).contiguous()
    want2 = step(x2, dy2)
    torch.cuda.synchronize()
    # two streams at once
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s, args in ((s1, (x, dy)), (s2, (x2, dy2))) * 4:
        with torch.cuda.stream(s):
            got.append(step(*args))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b_) for a, b_ in zip(g, want2 if i % 2 else want))
    # two graphs, replayed in turn on inputs that change
    graphs = []
    for args in ((x, dy), (x2, dy2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(*args)
        graphs.append((gr, out))
    for _ in range(2):
        for gr, _ in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for (_, out), wnt in zip(graphs, (want, want2)):
        assert all(torch.equal(a, b_) for a, b_ in zip(out, wnt))
    x.copy_(x2)
    dy.copy_(dy2)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b_) for a, b_ in zip(graphs[0][1], want2))


@pytest.mark.parametrize("rows,D", [(1, 384), (37, 384), (64, 128), (8, 5000), (5, 5003), (7, 8185), (250, 16), (300, 33)])
def test_few_rows_join_in_one_cluster(rows, D):
    """Grids of up to eight blocks: one launch that joins the parameters' gradients itself, on two
    streams at once and from a graph; parts of the gradients only."""
    dev = require_gpu()
    from genie_tk import ops
    args = [_inputs((rows, D), torch.float32, torch.float32, s, dev) for s in (1, 2)]
    for a in args:
        _run_and_check(*a)

    def back(x, dy, w, b, *need):
        _, mean, rstd = ops.layernorm_forward(x, w, b)
        return ops.layernorm_backward(dy, x, w, mean, rstd, *need)

    want = [back(*a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in args], []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, back(*args[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for i, g in got for p, q in zip(g, want[i]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = back(*args[0])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(out, want[0]))
    dx, dw, db = back(*args[0], False, True)
    assert dw is None and torch.equal(db, want[0][2]) and torch.equal(dx, want[0][0])
    dx, dw, db = back(*args[0], True, False)
    assert db is None and torch.equal(dw, want[0][1])


def test_module_and_autograd():
    dev = require_gpu()
    torch.manual_seed(0)
    m = genie_tk.LayerNorm(96).to(dev)
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    x = torch.randn(4, 7, 96, device=dev, requires_grad=True)
    v = torch.randn(4, 7, 96, device=dev)
    (m(x) * v).sum().backward()
    r = _reference(x.detach(), m.weight.detach(), m.bias.detach(), v)
    bound = _bounds(r, torch.float32, torch.float32)
    for k, t in (("dx", x.grad), ("dw", m.weight.grad), ("db", m.bias.grad)):
        _check(t, r[k], bound[k], k)
    # against central differences of the 64-bit forward along random directions
    for leaf, grad in ((0, x.grad), (1, m.weight.grad), (2, m.bias.grad)):
        args = [x.detach().double(), m.weight.detach().double(), m.bias.detach().double()]
        d = torch.randn_like(args[leaf])
        h = 1e-5
        vals = []
        for s in (1, -1):
            a = [t + s * h * d if i == leaf else t for i, t in enumerate(args)]
            vals.append((torch.nn.functional.layer_norm(a[0], (96,), a[1], a[2], EPS) * v.double()).sum())
        diff = (vals[0] - vals[1]) / (2 * h)
        # h^2 of the third derivative and 2^-53 / h of the values are below 1e-6 of the norms
        assert abs(float(diff - (grad.double() * d).sum())) <= 1e-5 * float(grad.double().norm() * d.norm())
    # the gradient arrives in another type and layout (the output was cast and transposed)
    xb = x.detach().to(torch.bfloat16).requires_grad_(True)
    mb = genie_tk.LayerNorm(96).to(dev)
    (mb(xb).float().transpose(0, 1) * v.transpose(0, 1)).sum().backward()
    assert xb.grad.dtype == torch.bfloat16 and mb.weight.grad.dtype == torch.float32
    r = _reference(xb.detach(), mb.weight.detach(), mb.bias.detach(), v.to(torch.bfloat16))
    _check(xb.grad, r["dx"], _bounds(r, torch.bfloat16, torch.float32)["dx"], "dx")
    # several normalised axes, no parameters, no gradient asked for
    m2 = genie_tk.LayerNorm((7, 96)).to(dev)
    ref = torch.nn.functional.layer_norm(x.detach().double(), (7, 96), m2.weight.double(), m2.bias.double())
    torch.testing.assert_close(m2(x.detach()).double(), ref, rtol=1e-5, atol=1e-5)
    assert genie_tk.LayerNorm(96, elementwise_affine=False).to(dev)(x).requires_grad
    with torch.no_grad():
        assert not m(x).requires_grad
    g, = torch.autograd.grad((m(x) * v).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    dev = require_gpu()
    from genie_tk import ops
    x = torch.randn(4, 64, device=dev)
    w = torch.ones(64, device=dev)
    y, mean, rstd = ops.layernorm_forward(x, w, w)
    with pytest.raises(TypeError):
        ops.layernorm_forward(x.double(), w, w)
    with pytest.raises(TypeError):
        ops.layernorm_forward(x, w.half(), w.half())
    with pytest.raises(TypeError):
        ops.layernorm_forward(x.half(), w.half(), w)
    with pytest.raises(ValueError):
        ops.layernorm_forward(x, w[:63], None)
    with pytest.raises(RuntimeError):
        ops.layernorm_forward(x, w.cpu(), None)
    with pytest.raises(RuntimeError):
        ops.layernorm_forward(x, w, w, eps=-1.0)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x[:3], x, w, mean, rstd)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x.half(), x, w, mean, rstd)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x, x, w, mean[:3], rstd)
    with pytest.raises(TypeError):
        ops.layernorm_backward(x, x, w, mean.double(), rstd)
    with pytest.raises(ValueError):
        genie_tk.LayerNorm(32).to(dev)(x)
