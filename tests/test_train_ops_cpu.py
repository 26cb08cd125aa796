"""CPU checks of the training operators' entry points: argument validation of the C ABI before
any launch, and the Python wrappers' refusals. No kernel is launched here."""

import ctypes

import pytest
import torch

import genie_tk
import genie_tk._lib as L
from genie_tk import ops

P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    return L.load()


def test_layernorm_entry_points(lib):
    p, q = P(1 << 20), P((1 << 20) + 2)
    ws = lib.gtk_layernorm_backward_workspace_bytes
    assert ws(1, 128) == 2 * 128 * 4 and ws(0, 128) == 0 and ws(4, 0) == 0 and ws(4, (1 << 20) + 1) == 0
    assert ws(10 ** 6, 128) <= 148 * 16 * 2 * 128 * 4 and ws(10 ** 6, 20000) == 64 * 2 * 20000 * 4

    def fwd(x=p, rows=None, xt=0, w=p, b=p, wt=0, y=p, m=p, r=p, n=4, d=8, eps=1e-5):
        return lib.gtk_layernorm_forward(x, rows, xt, w, b, wt, y, m, r, n, d, eps, None)

    assert fwd(n=0) == -1 and fwd(n=1 << 31) == -1 and fwd(d=0) == -1 and fwd(d=(1 << 20) + 1) == -1
    assert fwd(xt=3) == -2 and fwd(xt=0, wt=1) == -2 and fwd(xt=1, wt=2) == -2
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(m=None) == -1
    assert fwd(x=q) == L.GTK_ERR_ALIGNMENT and fwd(w=q) == L.GTK_ERR_ALIGNMENT

    def rows(size, stride):
        return ctypes.byref(L.Rows((ctypes.c_int64 * 3)(*size), (ctypes.c_int64 * 3)(*stride)))

    assert fwd(rows=rows((1, 2, 3), (0, 8, 8))) == -1 and b"make up" in lib.gtk_last_error_string()
    assert fwd(rows=rows((1, 0, 4), (0, 8, 8))) == -1
    assert fwd(rows=rows((1, 1, 4), (0, 0, -8))) == -1 and b"negative" in lib.gtk_last_error_string()

    def bwd(dy=p, x=p, xt=0, wt=0, dx=p, dw=p, db=p, w=p, wsp=p, nb=1 << 20, n=4, d=8):
        return lib.gtk_layernorm_backward(dy, None, x, None, xt, w, wt, p, p, dx, dw, db, wsp, nb, n, d, None)

    assert bwd(nb=8) == L.GTK_ERR_WORKSPACE and bwd(wsp=None) == -1
    assert bwd(dy=None) == -1 and bwd(dx=None) == -1 and bwd(dw=q) == L.GTK_ERR_ALIGNMENT
    assert bwd(xt=7) == -2 and bwd(d=-1) == -1


def test_wrappers_refuse_cpu_tensors():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layernorm_forward(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.layernorm_backward(x, x, None, x[:, 0], x[:, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        genie_tk.LayerNorm(8)(x)


def _list(kind, *values):
    return (kind * len(values))(*values)


def test_gradient_norm_entry_points(lib):
    a = 1 << 20
    assert lib.gtk_grad_norm_workspace_bytes(-1) == 0
    sizes = [lib.gtk_grad_norm_workspace_bytes(n) for n in (0, 1, 10, 1000, 1001, 5000)]
    assert sizes[0] > 0 and sizes[0] <= sizes[1] and sizes[-1] > 5000 * 24 and sorted(sizes) == sizes

    def clip(grads, numel, types, outs=None, out_types=None, kind=2, max_norm=1.0, norm=P(a), ws=P(a), nb=1 << 20):
        n = len(numel)
        return lib.gtk_clip_grad_norm(_list(P, *grads), None if outs is None else _list(P, *outs),
                                      _list(ctypes.c_int64, *numel), _list(ctypes.c_int, *types),
                                      None if out_types is None else _list(ctypes.c_int, *out_types), n, kind,
                                      max_norm, norm, ws, nb, None)

    assert clip([a], [4], [0], max_norm=-1.0) == -1 and clip([a], [4], [0], max_norm=float("nan")) == -1
    assert clip([a], [4], [0], kind=3) == -2 and clip([a], [4], [5]) == -2
    assert clip([a], [4], [0], [a + 64], [1]) == -2  # fp32 gradients into bf16
    assert clip([None], [4], [0]) == -1 and clip([a], [-4], [0]) == -1 and clip([a + 2], [4], [0]) == L.GTK_ERR_ALIGNMENT
    assert clip([a], [4], [0], nb=8) == L.GTK_ERR_WORKSPACE and clip([a], [4], [0], norm=None) == -1
    # the same tensor twice, a partial overlap, in any order; neighbours are fine as far as this check
    for grads, numel in (([a, a], [4, 4]), ([a + 8, a], [4, 4]), ([a, a + 64, a + 12], [4, 4, 4])):
        assert clip(grads, numel, [0] * len(numel)) == -1
        assert b"overlap" in lib.gtk_last_error_string()
    assert clip([a + 16, a], [4, 4], [0, 0], nb=8) == L.GTK_ERR_WORKSPACE
    # outputs on one another, on another gradient, on their own gradient at another place
    for outs in ([a + 4096, a + 4104], [a + 16, a], [a + 8, a + 4096]):
        assert clip([a, a + 16], [4, 4], [0, 0], outs) == -1, outs
        assert b"overlap" in lib.gtk_last_error_string()
    assert clip([a, a + 16], [4, 4], [0, 0], [a, a + 16], nb=8) == L.GTK_ERR_WORKSPACE  # exactly their own: fine
    assert clip([a, a], [4, 4], [0, 0], [a + 64, a + 128], nb=8) == L.GTK_ERR_WORKSPACE  # read twice: fine
    assert lib.gtk_grad_norm(None, None, None, 2, 2, P(a), P(a), 1 << 20, None) == -1


def test_embedding_entry_points(lib):
    p, q = P(1 << 20), P((1 << 20) + 2)
    size = lib.gtk_embedding_backward_workspace_bytes
    assert size(1, 10, 8, 0) > 0 and size(0, 10, 8, 0) == 0 and size(5, 0, 8, 0) == 0
    assert size(5, 5, (1 << 20) + 1, 0) == 0 and size(5, 5, 5, 3) == 0
    assert size(1000, 10, 8, 1) % 256 == 0 and size(20000, 32000, 128, 0) > size(5000, 32000, 128, 0) > 8 * 5000

    def fwd(tok=p, bits=64, w=p, dt=0, y=p, n=4, v=10, d=8):
        return lib.gtk_embedding_forward(tok, bits, w, dt, y, n, v, d, 1.0, None, None)

    assert fwd(bits=16) == -2 and fwd(dt=3) == -2 and fwd(n=0) == -1 and fwd(v=0) == -1 and fwd(v=1 << 31) == -1
    assert fwd(d=0) == -1 and fwd(tok=None) == -1 and fwd(w=None) == -1 and fwd(y=q) == L.GTK_ERR_ALIGNMENT
    assert fwd(tok=P((1 << 20) + 4)) == L.GTK_ERR_ALIGNMENT

    def bwd(dy=p, gt=0, tok=p, bits=32, dw=p, wt=0, n=4, v=10, d=8, pad=-1, ws=p, nb=1 << 24):
        return lib.gtk_embedding_backward(dy, gt, tok, bits, dw, wt, n, v, d, 1.0, pad, ws, nb, None, None)

    assert bwd(gt=0, wt=1) == -2 and bwd(gt=1, wt=2) == -2 and bwd(pad=10) == -1 and bwd(nb=16) == L.GTK_ERR_WORKSPACE
    assert bwd(dy=None) == -1 and bwd(dw=q) == L.GTK_ERR_ALIGNMENT and bwd(n=1 << 31) == -1
    assert bwd(ws=P((1 << 20) + 16)) == L.GTK_ERR_ALIGNMENT and bwd(n=(1 << 27) + 1) == -2
    assert bwd(dy=P((1 << 20) + 4)) == L.GTK_ERR_ALIGNMENT and bwd(dw=P((1 << 20) + 8)) == L.GTK_ERR_ALIGNMENT


def test_wrappers_refuse_before_the_device_is_needed():
    x = torch.randn(4)
    for call in (lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.grad_norm([x]),
                 lambda: ops.embedding_forward(torch.tensor([1]), x.view(2, 2)),
                 lambda: ops.embedding_backward(x.view(1, 4), torch.tensor([1]), 3),
                 lambda: genie_tk.Embedding(5, 4)(torch.tensor([1]))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="empty"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        ops.clip_grad_norm([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grad_norm([x], -1.0)
    with pytest.raises(TypeError, match="not a tensor"):
        ops.grad_norm([1.0])
    p = torch.nn.Parameter(x)
    assert float(genie_tk.clip_grad_norm_([p], 1.0)) == 0.0  # no gradients yet
    assert float(genie_tk.clip_grad_norm_(p, 1.0)) == 0.0


def test_missing_binding_is_an_error(monkeypatch):
    monkeypatch.setattr(L, "_native", None)
    monkeypatch.setattr(L, "BINDING_PATH", "/nonexistent/_gtk_torch.so")
    with pytest.raises(RuntimeError, match="cannot load"):
        ops.grad_norm([torch.randn(3)])
