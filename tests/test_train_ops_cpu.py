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


def test_row_views():
    """The strided leading axes that the kernels read in place, and those that are copied."""
    x = torch.arange(2 * 5 * 5 * 4.0).view(2, 5, 5, 4)
    assert ops._row_view(x) == (x, None) or ops._row_view(x)[1] is None

    def rows_of(t):
        v, m = ops._row_view(t)
        if m is None:
            return v.reshape(-1, v.shape[-1])
        base = v.storage_offset()
        flat = torch.as_strided(v, (v.untyped_storage().nbytes() // 4 - base,), (1,), base)
        s, st, D = list(m.size), list(m.stride), v.shape[-1]
        return torch.stack([flat[a * st[0] + b * st[1] + c * st[2]:][:D] for a in range(s[0]) for b in range(s[1])
                            for c in range(s[2])])

    for t in (x.transpose(1, 2), x[:, ::2], x[:, :, 1:4], x[0].transpose(0, 1), x[:1, 2:3], x.transpose(0, 2),
              x[:, :1].expand(2, 5, 5, 4), x[:, :, :, :3], x[1, 1:].transpose(0, 1)[:, :, 1:]):
        assert torch.equal(rows_of(t), t.reshape(-1, t.shape[-1])), t.shape
    y = torch.arange(3 * 4 * 5 * 6 * 2.0).view(3, 4, 5, 6, 2).permute(3, 1, 0, 2, 4)
    v, m = ops._row_view(y)
    assert m is None and v.is_contiguous() and torch.equal(v, y)
    assert ops._row_view(x.transpose(2, 3))[1] is None  # the last axis is strided: copied
