"""GPU tests of the LayerNorm kernels that few calls reach: rows of more than 16384 elements in
numbers, rows that begin anywhere (element by element), and the statistics' shape.

Tolerances as in test_gpu_layernorm_train.py, unless a test says its own."""

import pytest
import torch

import genie_tk
from gpu_util import require_gpu
from test_gpu_layernorm_train import DT, EPS, U, _bounds, _check, _inputs, _reference, _run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(130, 16379), (130, 20000), (700, 16379), (700, 20000), (65, 40001)])
def test_wide_rows_in_numbers(rows, D, dtype):
    """More rows than the partial sums have slabs, and than four to an SM."""
    dev = require_gpu()
    _run_and_check(*_inputs((rows, D), DT[dtype], torch.float32, rows + D, dev))


@pytest.mark.parametrize("B,N,D", [(1, 9, 16379), (2, 11, 20000)])
def test_wide_rows_transposed(B, N, D):
    dev = require_gpu()
    x, dy, w, b = _inputs((B, N, N, D), torch.bfloat16, torch.float32, N, dev)
    _run_and_check(x.transpose(1, 2), dy.transpose(1, 2), w, b)
    _run_and_check(x, dy.transpose(1, 2), w, b)


def test_wide_rows_sum_their_columns_in_short_chains():
    """dw and db of many wide rows: a value of 1 in each 256 rows and 255 that half a step of 1 is
    more than (one after another onto it, they are all lost: 254 u of the sum). Sixteen rows are
    added in fp32 (15 u), the sixteens in 64 bits, stored (u), and 64 such sums are joined (four to a
    thread, two shuffles, five over the warps: 10 u): 32 u."""
    dev = require_gpu()
    from genie_tk import ops
    rows, D = 16384, 16385
    small = 2.0 ** -24 * (1 - 2.0 ** -8)
    column = torch.full((rows, 1), small, dtype=torch.float64, device=dev)
    column[::256] = 1.0
    dy = column.to(torch.bfloat16).expand(rows, D).contiguous()
    assert torch.equal(dy[:, :1].double(), column)
    x = torch.ones(rows, D, dtype=torch.bfloat16, device=dev)
    x[:, 1::2] = -1.0
    mean, rstd = torch.zeros(rows, device=dev), torch.ones(rows, device=dev)
    w = torch.ones(D, device=dev)
    _, dw, db = ops.layernorm_backward(dy, x, w, mean, rstd)
    want = float(column.sum())
    sign = x[0].double()
    assert float((db.double() - want).abs().max()) <= 32 * U * want
    assert float((dw.double() * sign - want).abs().max()) <= 32 * U * want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,D", [(9, 33), (40, 33), (9, 601), (40, 601), (10, 5003), (9, 9001), (13, 16377)])
def test_transposed_rows_that_begin_anywhere(N, D, dtype):
    """Odd widths at strides: no vectors. Tiles of rows from N = 8 on; groups in a warp, one group
    a block, and 32 elements a thread."""
    dev = require_gpu()
    x, dy, w, b = _inputs((1, N, N, D), DT[dtype], torch.float32, N + D, dev)
    _run_and_check(x.transpose(1, 2), dy.transpose(1, 2), w, b)
    _run_and_check(x.transpose(1, 2), dy, w, b)
    _run_and_check(x, dy.transpose(1, 2), w, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("D", [40, 600, 5003, 9001])
def test_bases_off_a_vector(rows, D, dtype):
    dev = require_gpu()
    x, dy, w, b = _inputs((rows * D + 5,), DT[dtype], torch.float32, rows + D, dev)
    w, b = w[:D].contiguous(), b[:D].contiguous()
    shift = lambda t, k: t[k:k + rows * D].view(rows, D)  # noqa: E731
    _run_and_check(shift(x, 1), shift(dy, 3), w, b)
    _run_and_check(shift(x, 0), shift(dy, 1), w, b)
    _run_and_check(shift(x, 1), shift(dy, 0), w, b)


def test_statistics_lie_as_the_rows_do():
    """mean and rstd have one element for each row in x's own axes (or in one axis, or with a last
    axis of one): statistics of the transposed tensor are refused, not read in another order."""
    dev = require_gpu()
    from genie_tk import ops
    x, dy, w, b = _inputs((3, 5, 7, 24), torch.float32, torch.float32, 1, dev)
    y, mean, rstd = ops.layernorm_forward(x, w, b)
    want = ops.layernorm_backward(dy, x, w, mean, rstd)
    for m, r in ((mean.reshape(-1), rstd.reshape(-1)), (mean.unsqueeze(-1), rstd.unsqueeze(-1)), (mean, rstd.reshape(-1))):
        assert all(torch.equal(p, q) for p, q in zip(ops.layernorm_backward(dy, x, w, m, r), want))
    xt, dyt = x.transpose(1, 2), dy.transpose(1, 2)
    with pytest.raises(ValueError, match="one element for each row"):
        ops.layernorm_backward(dyt, xt, w, mean, rstd)
    with pytest.raises(ValueError, match="one element for each row"):
        ops.layernorm_backward(dyt, xt, w, mean.transpose(1, 2), rstd)
    got = ops.layernorm_backward(dyt, xt, w, mean.transpose(1, 2), rstd.transpose(1, 2))
    torch.testing.assert_close(got[0], want[0].transpose(1, 2), rtol=0, atol=0)
    with pytest.raises(ValueError, match="one element for each row"):
        ops.layernorm_backward(dy, x, w, mean.reshape(15, 7), rstd)
    one = torch.randn(24, device=dev)
    _, m, r = ops.layernorm_forward(one, w, b)
    assert m.dim() == 0 and ops.layernorm_backward(one, one, w, m, r)[0].shape == (24,)


def _check_rows(x, dy, w, b, got, rows):
    """y, mean, rstd and dx of some rows (indices into the flattened leading axes)."""
    y, mean, rstd, dx = got
    D = x.shape[-1]
    pick = lambda t: torch.stack([t[tuple(i)] for i in rows])  # noqa: E731
    xs, gs = pick(x), pick(dy)
    r = _reference(xs, w, b, gs)
    bound = _bounds(r, x.dtype, w.dtype)
    for k, t in (("y", pick(y)), ("mean", pick(mean)), ("rstd", pick(rstd)), ("dx", pick(dx))):
        _check(t, r[k], bound[k], k)
    assert xs.shape[-1] == D


@pytest.mark.parametrize("shape,swap", [(((1 << 24) + 77, 130), False), ((4100, 4100, 128), True), ((4100, 4099, 129), True)])
def test_more_than_2_31_elements(shape, swap):
    """The last and some other rows against 64 bits, and the parameters' gradients against sums by
    parts: xhat is off by 64 u (3 + 2 |xhat|) at most for this data, and a sum of R rows by
    (64 + R / 148) u of its magnitudes."""
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
    dy = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
    D = shape[-1]
    w, b = 1 + 0.1 * torch.randn(D, generator=gen, device=dev), torch.randn(D, generator=gen, device=dev)
    if swap:
        x, dy = x.transpose(0, 1), dy.transpose(0, 1)
    y, mean, rstd = ops.layernorm_forward(x, w, b)
    dx, dw, db = ops.layernorm_backward(dy, x, w, mean, rstd)
    lead = x.shape[:-1]
    rows = [[n - 1 for n in lead], [0] * len(lead), [n // 2 for n in lead]]
    rows += [[lead[0] - 2 - i] + [n - 3 for n in lead[1:]] for i in range(40)]
    _check_rows(x, dy, w, b, (y, mean, rstd, dx), rows)
    del y, dx
    R = x.numel() // D
    want_w = torch.zeros(D, dtype=torch.float64, device=dev)
    want_b, mag_w, mag_b, part = (torch.zeros_like(want_w) for _ in range(4))
    step = 1 << 20 if not swap else 256
    for i in range(0, lead[0], step):
        xs, gs = x[i:i + step].double(), dy[i:i + step].double()
        xh = (xs - xs.mean(-1, keepdim=True)) * (xs.var(-1, correction=0, keepdim=True) + EPS) ** -0.5
        axes = tuple(range(xs.dim() - 1))
        want_w += (gs * xh).sum(axes)
        want_b += gs.sum(axes)
        mag_w += (gs * xh).abs().sum(axes)
        mag_b += gs.abs().sum(axes)
        part += (gs.abs() * (3 + 2 * xh.abs())).sum(axes)
    tree = (64 + R / 148) * U
    for got, want, bound in ((db, want_b, tree * mag_b), (dw, want_w, tree * mag_w + 64 * U * part)):
        assert ((got.double() - want).abs() <= bound + 2 * U * want.abs()).all()
        assert float((got.double() - want).norm()) <= 1e-5 * float(mag_b.norm())
