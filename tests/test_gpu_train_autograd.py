"""GPU tests of the training operators' place in autograd: forward-mode tangents, gradients that
arrive as lazily negated views, and parameters with an axis more."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

import genie_tk
from genie_tk import autograd
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu


def test_tangents_are_refused_not_dropped():
    """The operators have no forward-mode formula: an input with a tangent raises, whether or not
    anything requires a gradient, and so does an output gradient with one."""
    dev = require_gpu()
    from genie_tk import ops
    x, t = torch.randn(4, 24, device=dev), torch.randn(4, 24, device=dev)
    w, b = torch.randn(24, device=dev), torch.randn(24, device=dev)
    table, tok = torch.randn(9, 24, device=dev), torch.tensor([1, 5, 8, 1], device=dev)
    y, mean, rstd = ops.layernorm_forward(x, w, b)
    leaf = x.clone().requires_grad_(True)
    out = autograd.layer_norm(leaf, w, b)
    row = table.clone().requires_grad_(True)
    out2 = autograd.embedding(tok, row)
    with fwad.dual_level():
        xd, wd, td = fwad.make_dual(x, t), fwad.make_dual(w, t[0]), fwad.make_dual(table, torch.randn_like(table))
        calls = [lambda: autograd.layer_norm(xd, w, b), lambda: autograd.layer_norm(x, wd, b),
                 lambda: autograd.layer_norm(x, w, wd), lambda: autograd.layer_norm(xd, w.requires_grad_(True), b),
                 lambda: genie_tk.LayerNorm(24).to(dev).requires_grad_(False)(xd), lambda: autograd.embedding(tok, td),
                 lambda: ops.layernorm_forward(xd, w, b), lambda: ops.layernorm_backward(xd, x, w, mean, rstd),
                 lambda: ops.layernorm_backward(t, xd, w, mean, rstd), lambda: ops.embedding_forward(tok, td),
                 lambda: ops.embedding_backward(xd, tok, 9), lambda: ops.grad_norm([t, xd]),
                 lambda: ops.clip_grad_norm([t, xd], 1.0), lambda: ops.clip_grad_norm([t], 1.0, out=[xd]),
                 lambda: torch.autograd.grad(out, leaf, xd, retain_graph=True),
                 lambda: torch.autograd.grad(out2, row, xd, retain_graph=True)]
        for i, call in enumerate(calls):
            with pytest.raises(NotImplementedError, match="forward.mode"):
                call()
                pytest.fail(f"call {i} returned")
        # without a tangent everything runs inside a level too
        assert torch.equal(autograd.layer_norm(x, w.detach(), b), y)
        torch.autograd.grad(out, leaf, t)
    assert float(ops.grad_norm([t])) > 0


def test_lazily_negated_output_gradients():
    """A gradient that reaches the operators through a complex view may be a lazily negated one; torch's
    own layer_norm and embedding take it."""
    dev = require_gpu()
    x, w, b = torch.randn(5, 24, device=dev), torch.randn(24, device=dev), torch.randn(24, device=dev)
    table, tok = torch.randn(9, 24, device=dev), torch.tensor([1, 5, 8, 1], device=dev)
    v = torch.randn(5, 24, device=dev)
    neg = torch.complex(torch.zeros_like(v), v).conj().imag
    assert neg.is_neg() and torch.equal(neg, -v)
    for make, n in ((lambda t: autograd.layer_norm(t, w, b), x), (lambda t: autograd.embedding(tok, t), table)):
        leaf = n.clone().requires_grad_(True)
        out = make(leaf)
        got, = torch.autograd.grad(out, leaf, neg[:out.shape[0]], retain_graph=True)
        want, = torch.autograd.grad(out, leaf, -v[:out.shape[0]])
        assert torch.equal(got, want)


def test_parameters_with_an_axis_more():
    """Weights of D elements in another shape: their gradients have that shape."""
    dev = require_gpu()
    x = torch.randn(5, 24, device=dev, requires_grad=True)
    w, b = (torch.randn(24, device=dev) for _ in range(2))
    v = torch.randn(5, 24, device=dev)
    flat = [w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    want = torch.autograd.grad((autograd.layer_norm(x, *flat) * v).sum(), [x, *flat])
    for shape in ((1, 24), (24, 1), (2, 12)):
        more = [t.view(shape).clone().requires_grad_(True) for t in (w, b)]
        got = torch.autograd.grad((autograd.layer_norm(x, *more) * v).sum(), [x, *more])
        assert got[1].shape == shape and got[2].shape == shape
        assert all(torch.equal(p, q.view(p.shape)) for p, q in zip(got, want))
        only, = torch.autograd.grad((autograd.layer_norm(x, None, more[1]) * v).sum(), more[1])
        assert only.shape == shape and torch.equal(only.view(-1), want[2])
