"""GPU tests of the embedding lookup and its gradient by sorted tokens (gtk_embedding_forward /
gtk_embedding_backward) against sums in 64 bits.

Tolerances, with u = 2^-24 and h the half step of the result's type: the lookup rounds the
product once in fp32 and once in its type. In the gradient the n rows of a token are added in some
fixed order: at most n - 1 roundings, whatever the order, and never more than 300 one on another
(fours of at most 1024 rows, then trees): (min(n, 1024) + 8) u times the sum of magnitudes covers
both, and then come the product with the scale and the rounding."""

import pytest
import torch

import genie_tk
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _tokens(kind, n, V, dev, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=gen, device=dev)
    if kind == "one":
        return torch.full((n,), V - 1, device=dev, dtype=torch.int64)
    if kind == "down":
        return (V - 1 - torch.arange(n, device=dev) % V)
    if kind == "sorted":
        return torch.randint(0, V, (n,), generator=gen, device=dev).sort().values
    u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)  # zipf
    return ((V + 1.0) ** u - 1).long().clamp_(0, V - 1)


def _check_backward(dy, tok, V, scale=1.0, padding=None, dtype=None):
    from genie_tk import ops
    dw = ops.embedding_backward(dy, tok, V, scale, padding, dtype)
    D = dy.shape[-1]
    assert dw.shape == (V, D) and dw.dtype == (dtype or dy.dtype)
    t, g = tok.reshape(-1).long(), dy.reshape(-1, D).double()
    ok = (t >= 0) & (t < V)
    t, g = t[ok], g[ok]
    ref = torch.zeros(V, D, dtype=torch.float64, device=dy.device).index_add_(0, t, g)
    mag = torch.zeros_like(ref).index_add_(0, t, g.abs())
    if padding is not None:
        ref[padding], mag[padding] = 0, 0
    count = torch.bincount(t, minlength=V).clamp(max=1024).unsqueeze(1)
    tol = (count + 8) * U * mag * abs(scale) + 2 * U * (ref * scale).abs()
    tol = tol + _half(dw.dtype) * ((ref * scale).abs() + tol)
    if dw.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    tol[bincount_zero(t, V)] = 0
    err = (dw.double() - ref * scale).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    return dw


def bincount_zero(t, V):
    return torch.bincount(t, minlength=V) == 0


@pytest.mark.parametrize("dtype,wdtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                          ("f16", "f32")])
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 21, 384), (2, 2, 8), (31, 5, 33), (33, 66, 128), (300, 21, 384),
                                   (1000, 255, 64), (1000, 256, 64), (1000, 257, 100), (5000, 32000, 32),
                                   (8192, 1000, 128), (8193, 1000, 128), (20000, 70000, 24), (70000, 66, 128),
                                   (30000, 300, 1000)])
def test_gradient(T, V, D, dtype, wdtype):
    dev = require_gpu()
    gen = torch.Generator(device=dev).manual_seed(T + V + D)
    dy = torch.randn(T, D, generator=gen, device=dev).to(DT[dtype])
    for kind in ("uniform", "zipf"):
        for index in (torch.int64, torch.int32):
            _check_backward(dy, _tokens(kind, T, V, dev, T).to(index), V, 1.0 if kind == "zipf" else D ** 0.5, None,
                            DT[wdtype])


@pytest.mark.parametrize("D", [1, 2, 4, 7, 8, 15, 16, 17, 24, 31, 32, 40, 63, 64, 65, 96, 127, 129, 250, 256, 260, 515])
def test_widths(D):
    """Groups of 4 to 32 lanes, one slab of columns or several, vectors and single elements."""
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(D)
    for T, V in ((3, 5), (600, 7), (3000, 40), (9001, 5000)):
        tok = _tokens("zipf", T, V, dev, T)
        for dtype in (torch.float32, torch.bfloat16):
            dy = torch.randn(T, D, generator=gen, device=dev).to(dtype)
            _check_backward(dy, tok, V)
            _check_backward(dy, tok, V, 2.0, 1, torch.float32)
            w = torch.randn(V, D, generator=gen, device=dev).to(dtype)
            assert torch.equal(ops.embedding_forward(tok, w), w[tok])
            assert torch.equal(ops.embedding_forward(tok, w, 0.5), w[tok] * 0.5)


@pytest.mark.parametrize("kind", ["one", "down", "sorted"])
@pytest.mark.parametrize("T", [1, 32, 33, 512, 513, 700, 1024, 1025, 4097, 8192, 8193, 16385, 32768, 32769, 50001, 131073, 262145, 600001])
def test_orders_of_tokens(kind, T):
    dev = require_gpu()
    gen = torch.Generator(device=dev).manual_seed(T)
    dy = torch.randn(T, 72, generator=gen, device=dev)
    for V in (1, 7, 1023):
        _check_backward(dy, _tokens(kind, T, V, dev), V)
        _check_backward(dy, _tokens(kind, T, V, dev), V, 2.0, padding=V // 2)


def test_runs_that_end_at_chunk_borders():
    """Runs of 31, 32, 33, 64 ... tokens, so that they begin and end on either side of the chunks
    that the sorted list is cut into."""
    dev = require_gpu()
    gen = torch.Generator(device=dev).manual_seed(2)
    lengths = [31, 1, 32, 32, 33, 63, 64, 65, 1, 1, 30, 96, 128, 3, 29, 500, 12, 1024, 2048]
    tok = torch.cat([torch.full((n,), i, device=dev) for i, n in enumerate(lengths)])
    dy = torch.randn(len(tok), 40, generator=gen, device=dev)
    _check_backward(dy, tok, len(lengths))
    p = torch.randperm(len(tok), generator=gen, device=dev)
    _check_backward(dy, tok[p], len(lengths) + 3)
    # the same runs in a list long enough for longer chunks
    big = tok.repeat_interleave(40)
    dy = torch.randn(len(big), 129, generator=gen, device=dev)
    _check_backward(dy, big, len(lengths))


def test_relative_positions_of_a_pair_grid():
    dev = require_gpu()
    N, k = 300, 32
    i = torch.arange(N, device=dev)
    tok = (i[None] - i[:, None]).clamp(-k, k) + k
    tok[:, 200:] = 2 * k + 1
    gen = torch.Generator(device=dev).manual_seed(5)
    dy = torch.randn(1, N, N, 128, generator=gen, device=dev)
    _check_backward(dy, tok[None].int(), 2 * k + 2)
    _check_backward(dy.transpose(1, 2), tok[None], 2 * k + 2)  # a strided gradient
    _check_backward(dy[:, :1].expand(1, N, N, 128), tok[None], 2 * k + 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (7, 3, 5), (300, 21, 384), (1001, 500, 33), (4099, 32000, 128),
                                   (513, 64, 4096)])
def test_lookup(T, V, D, dtype):
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(T)
    w = torch.randn(V, D, generator=gen, device=dev).to(DT[dtype])
    tok = _tokens("uniform", T, V, dev, 3)
    assert torch.equal(ops.embedding_forward(tok, w), w[tok])
    s = 0.7 * D ** 0.5
    got = ops.embedding_forward(tok.int().view(1, T, 1), w, s)
    assert got.shape == (1, T, 1, D) and got.dtype == w.dtype
    s32 = float(torch.tensor(s, dtype=torch.float32))
    ref = (w[tok].double() * s32).view(1, T, 1, D)
    tol = (U + _half(w.dtype) * (1 + U)) * ref.abs() + (2.0 ** -25 if w.dtype == torch.float16 else 0)
    assert ((got.double() - ref).abs() <= tol).all()


def test_strides_and_alignment():
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(9)
    big = torch.randn(50, 131, generator=gen, device=dev)
    tok = _tokens("uniform", 60, 49, dev).view(6, 10)
    for w in (big[:49, :128], big[1:, 3:67], big.reshape(-1)[1:1 + 49 * 128].view(49, 128)):
        assert torch.equal(ops.embedding_forward(tok.t(), w), w[tok.t()])
    dyb = torch.randn(10, 6, 131, generator=gen, device=dev)
    _check_backward(dyb[..., 1:129], tok.t(), 49)
    flat = torch.randn(60 * 128 + 1, generator=gen, device=dev)[1:].view(10, 6, 128)
    _check_backward(flat, tok.t(), 49)
    _check_backward(flat.bfloat16(), tok.t(), 49, 3.0, 5, torch.float32)


def test_tokens_outside_the_table():
    dev = require_gpu()
    from genie_tk import ops
    ops.check_status(dev)
    w = torch.randn(10, 64, device=dev)
    tok = torch.tensor([3, -1, 10, 9, 2 ** 32 + 3, -2 ** 40, 0], device=dev)
    y = ops.embedding_forward(tok, w)
    assert ops.check_status(dev) == 0x80 and ops.check_status(dev) == 0
    ok = torch.tensor([True, False, False, True, False, False, True], device=dev)
    assert torch.equal(y[ok], w[tok[ok]]) and not y[~ok].any()
    dy = torch.randn(7, 64, device=dev)
    dw = _check_backward(dy, tok, 10)
    assert ops.check_status(dev) == 0x80
    assert torch.equal(dw[3], dy[0]) and torch.equal(dw[9], dy[3]) and torch.equal(dw[0], dy[6])
    for n in (5, 9000, 40000):  # none of them is in the table
        dw = ops.embedding_backward(torch.full((n, 64), float("nan"), device=dev), torch.full((n,), 77, device=dev), 10)
        assert not dw.any() and ops.check_status(dev) == 0x80
    _check_backward(torch.randn(40000, 8, device=dev), torch.arange(40000, device=dev) % 20 - 5, 10)
    assert ops.check_status(dev) == 0x80
    # rows at the padding token do not reach the sums, whatever they hold; the lookup reads the row
    dy = torch.randn(100, 64, device=dev)
    tok = torch.arange(100, device=dev) % 10
    dy[tok == 4] = float("nan")
    dw = ops.embedding_backward(dy, tok, 10, padding_idx=4)
    assert not dw[4].any() and torch.isfinite(dw).all() and ops.check_status(dev) == 0
    assert torch.equal(ops.embedding_forward(tok, w), w[tok])


def test_empty_calls():
    dev = require_gpu()
    from genie_tk import ops
    none = torch.empty(0, 3, dtype=torch.int64, device=dev)
    assert ops.embedding_forward(none, torch.randn(4, 8, device=dev)).shape == (0, 3, 8)
    dw = ops.embedding_backward(torch.empty(0, 3, 8, device=dev), none, 4)
    assert dw.shape == (4, 8) and not dw.any()


def test_module_and_autograd():
    dev = require_gpu()
    torch.manual_seed(0)
    m = genie_tk.Embedding(21, 96, padding_idx=20, scale=96 ** 0.5).to(dev)
    assert list(m.state_dict()) == ["weight"] and not m.weight[20].any()
    tok = torch.randint(0, 21, (2, 50), device=dev)
    y = m(tok)
    assert y.requires_grad and torch.equal(y, m.weight[tok] * torch.tensor(96 ** 0.5, device=dev))
    v = torch.randn(2, 50, 96, device=dev)
    (y * v).sum().backward()
    ref = torch.zeros(21, 96, dtype=torch.float64, device=dev).index_add_(0, tok.view(-1), v.view(-1, 96).double())
    ref *= 96 ** 0.5
    ref[20] = 0
    # at most 100 rows a token: (100 + 10) u of the magnitudes, which are below 60 * 10 here
    assert float((m.weight.grad - ref).abs().max()) <= 110 * U * 600
    # against differences of the forward, which is linear: exact up to rounding
    d = torch.randn(21, 96, dtype=torch.float64, device=dev)
    d[20] = 0
    diff = ((d[tok] * 96 ** 0.5) * v.double()).sum()
    got = (m.weight.grad.double() * d).sum()
    assert abs(float(diff - got)) <= 110 * U * 600 * 21 * 96
    with torch.no_grad():
        assert not m(tok).requires_grad
    mb = genie_tk.Embedding(21, 96).to(dev).bfloat16()
    mb(tok).float().sum().backward()
    assert mb.weight.grad.dtype == torch.bfloat16
    assert torch.equal(mb.weight.grad[:, 0].float(), torch.bincount(tok.view(-1), minlength=21).float())


def test_same_bits_on_streams_and_from_graphs():
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(1)
    cases = []
    for T, V in ((30000, 66), (5000, 32000), (20000, 70000)):
        cases.append((torch.randn(T, 136, generator=gen, device=dev), _tokens("zipf", T, V, dev, T), V))
    want = [ops.embedding_backward(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(4):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.embedding_backward(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))
    graphs = []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = (ops.embedding_backward(*c), ops.embedding_forward(c[1], want[0][:1].expand(c[2], 136).contiguous()))
        graphs.append((gr, out))
    for _ in range(2):
        for gr, _ in graphs:
            gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], w) for (_, o), w in zip(graphs, want))
    cases[0][1].copy_(cases[0][1].flip(0))
    want0 = ops.embedding_backward(*cases[0])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], want0)


def test_more_than_2_31_elements():
    dev = require_gpu()
    from genie_tk import ops
    T, D, V = (1 << 20) + 77, 2056, 5
    dy = torch.ones(T, D, dtype=torch.bfloat16, device=dev)
    tok = torch.zeros(T, dtype=torch.int32, device=dev)
    tok[-100:] = 3
    tok[1000] = 4
    dy[-1] = 3.0
    dw = ops.embedding_backward(dy, tok, V, dtype=torch.float32)
    assert (dw[3] == 102).all() and (dw[4] == 1).all() and (dw[0] == T - 101).all() and not dw[1:3].any()
    w = torch.randn(V, D, device=dev).bfloat16()
    y = ops.embedding_forward(tok, w)
    assert torch.equal(y[-101:], w[tok[-101:].long()]) and torch.equal(y[:2], w[:1].expand(2, D))


def test_refusals():
    dev = require_gpu()
    from genie_tk import ops
    w = torch.randn(10, 8, device=dev)
    tok = torch.tensor([1, 2], device=dev)
    dy = torch.randn(2, 8, device=dev)
    for e, call in ((TypeError, lambda: ops.embedding_forward(tok.short(), w)),
                    (TypeError, lambda: ops.embedding_forward(tok.float(), w)),
                    (TypeError, lambda: ops.embedding_forward(tok, w.double())),
                    (ValueError, lambda: ops.embedding_forward(tok, w[0])),
                    (RuntimeError, lambda: ops.embedding_forward(tok.cpu(), w)),
                    (ValueError, lambda: ops.embedding_backward(dy[:1], tok, 10)),
                    (ValueError, lambda: ops.embedding_backward(dy, tok, 0)),
                    (ValueError, lambda: ops.embedding_backward(dy, tok, 10, padding_idx=10)),
                    (ValueError, lambda: ops.embedding_backward(dy, tok, 10, padding_idx=-1)),
                    (TypeError, lambda: ops.embedding_backward(dy, tok, 10, dtype=torch.bfloat16)),
                    (RuntimeError, lambda: ops.embedding_backward(dy, tok.cpu(), 10))):
        with pytest.raises(e):
            call()
    from genie_tk import autograd
    for bad in (-1, 10):
        with pytest.raises(ValueError, match="padding_idx"):
            autograd.embedding(tok, w, 1.0, bad)
