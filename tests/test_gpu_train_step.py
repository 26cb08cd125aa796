"""The training operators together, as a training step uses them: residue types and relative positions
through embedding tables, the pair embedding, a pair block, LayerNorm, the loss's gradients, and
clipping by their global norm."""

import copy

import pytest
import torch
import torch.nn.functional as F

import genie_tk
from gpu_util import assert_status_clean, require_gpu

pytestmark = pytest.mark.gpu


class Net(torch.nn.Module):
    """Tokens [B, N] to a score per pair; ``block`` is a pair block or None."""

    def __init__(self, block=None):
        super().__init__()
        self.types = genie_tk.Embedding(21, 48, padding_idx=20, scale=48 ** 0.5)
        self.pairs = genie_tk.PairEmbedding(48, 128)
        self.positions = genie_tk.Embedding(66, 128)
        self.block = block
        self.norm = genie_tk.LayerNorm(128)
        self.head = torch.nn.Linear(128, 3)

    @staticmethod
    def offsets(N, device):
        i = torch.arange(N, device=device)
        return (i[None] - i[:, None]).clamp(-32, 32) + 32

    def forward(self, tokens, mask):
        p, pair_mask = self.pairs(self.types(tokens), mask)
        p = p + self.positions(self.offsets(tokens.shape[1], tokens.device))
        if self.block is not None:
            p, _ = self.block((p, pair_mask))
        # the ending node's order: LayerNorm reads the transposed pair tensor
        return self.head(self.norm(p.transpose(1, 2)))

    def reference(self, tokens, mask):
        """The same in stock 64-bit operations, without the block."""
        assert self.block is None
        s = F.embedding(tokens, self.types.weight, padding_idx=20) * 48 ** 0.5
        B, N, c = s.shape
        both = torch.cat([s[:, :, None].expand(B, N, N, c), s[:, None].expand(B, N, N, c)], dim=-1)
        p = F.linear(both, self.pairs.weight, self.pairs.bias)
        p = p + F.embedding(self.offsets(N, tokens.device), self.positions.weight)
        return self.head(F.layer_norm(p.transpose(1, 2), (128,), self.norm.weight, self.norm.bias, self.norm.eps))


def _batch(dev, B=2, N=45):
    gen = torch.Generator(device=dev).manual_seed(3)
    tokens = torch.randint(0, 21, (B, N), generator=gen, device=dev)
    mask = torch.ones(B, N, device=dev)
    mask[1, -9:] = 0
    target = torch.randn(B, N, N, 3, generator=gen, device=dev)
    return tokens, mask, target


def test_steps_match_a_64_bit_reference():
    """Three steps of plain gradient descent with clipping. Every operation is fp32: a gradient is off
    by a few hundred roundings (2^-24 each) of its tensor's size, 1e-4 relative to its norm leaves a
    factor of five."""
    dev = require_gpu()
    torch.manual_seed(0)
    net = Net().to(dev)
    ref = copy.deepcopy(net).double()
    tokens, mask, target = _batch(dev)
    for step in range(3):
        loss = (net(tokens, mask) - target).square().mean()
        net.zero_grad()
        loss.backward()
        want = (ref.reference(tokens, mask.double()) - target.double()).square().mean()
        ref.zero_grad()
        want.backward()
        torch.testing.assert_close(loss.double(), want, rtol=1e-5, atol=0)
        names = [n for n, _ in net.named_parameters()]
        grads = [p.grad for p in net.parameters()]
        wants = [p.grad for p in ref.parameters()]
        assert all(g is not None for g in grads) and not net.types.weight.grad[20].any()
        for n, g, w in zip(names, grads, wants):
            assert float((g - w).norm()) <= 1e-4 * float(w.norm()) + 1e-12, n
        full = torch.sqrt(sum(w.square().sum() for w in wants))
        limit = 0.3 * float(full)
        norm = genie_tk.clip_grad_norm_(net.parameters(), limit)
        torch.testing.assert_close(norm.double(), full, rtol=1e-4, atol=0)
        torch.nn.utils.clip_grad_norm_(ref.parameters(), limit)
        for n, g, w in zip(names, grads, wants):
            assert float((g - w).norm()) <= 2e-4 * float(w.norm()) + 1e-12, n
        with torch.no_grad():
            for p, q in zip(net.parameters(), ref.parameters()):
                p -= 0.5 * p.grad
                q -= 0.5 * q.grad
    assert_status_clean(dev)


def test_step_with_a_pair_layer():
    """The same around a PairTransformLayer, whose backward runs the LayerNorm kernels inside: every
    parameter gets a finite gradient, the norm is theirs, the clipped norm is the limit, and the same
    step gives the same bits."""
    dev = require_gpu()
    torch.manual_seed(1)
    layer = genie_tk.PairTransformLayer(128, tri_dropout=0.0)
    for p in layer.parameters():  # the final layers start at zero, which would hide the block
        if not p.any():
            torch.nn.init.normal_(p, std=0.05)
    net = Net(layer).to(dev)
    tokens, mask, target = (t[:1] for t in _batch(dev, 2, 33))
    runs = []
    for _ in range(2):
        net.zero_grad()
        (net(tokens, mask) - target).square().mean().backward()
        grads = [p.grad for p in net.parameters()]
        assert all(g is not None and torch.isfinite(g).all() for g in grads)
        full = torch.sqrt(sum(g.double().square().sum() for g in grads))
        norm = genie_tk.clip_grad_norm_(net.parameters(), 0.5 * float(full))
        torch.testing.assert_close(norm.double(), full, rtol=1e-6, atol=0)
        after = torch.sqrt(sum(g.double().square().sum() for g in grads))
        torch.testing.assert_close(after, 0.5 * full, rtol=1e-5, atol=0)
        runs.append([net.types.weight.grad.clone(), net.norm.weight.grad.clone(), norm])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert_status_clean(dev)


def test_functional_step_in_a_graph():
    """LayerNorm forward and backward, the embedding's gradient and clipping captured as one graph by
    their functional forms, replayed on other data."""
    dev = require_gpu()
    from genie_tk import ops
    gen = torch.Generator(device=dev).manual_seed(5)
    tokens = torch.randint(0, 50, (4, 30), generator=gen, device=dev)
    table = torch.randn(50, 96, generator=gen, device=dev)
    w, b = torch.randn(96, generator=gen, device=dev), torch.randn(96, generator=gen, device=dev)
    dy = torch.randn(4, 30, 96, generator=gen, device=dev)

    def step():
        x = ops.embedding_forward(tokens, table, 2.0)
        y, mean, rstd = ops.layernorm_forward(x, w, b)
        dx, dw, db = ops.layernorm_backward(dy, x, w, mean, rstd)
        dt = ops.embedding_backward(dx, tokens, 50, 2.0)
        return y, dt, dw, db, ops.clip_grad_norm([dt, dw, db], 1.0)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        gen.manual_seed(seed)
        tokens.copy_(torch.randint(0, 50, (4, 30), generator=gen, device=dev))
        table.copy_(torch.randn(50, 96, generator=gen, device=dev))
        dy.copy_(torch.randn(4, 30, 96, generator=gen, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(out, want))
        assert float(out[-1]) > 1.0


def test_modules_in_a_graph():
    """Forward, backward and clipping through the modules in one graph, by PyTorch's rules for it: the
    passes before the capture run on a side stream, and nothing of their autograd graph is left."""
    dev = require_gpu()
    torch.manual_seed(2)
    emb, norm = genie_tk.Embedding(30, 64, padding_idx=3).to(dev), genie_tk.LayerNorm(64).to(dev)
    params = [*emb.parameters(), *norm.parameters()]
    tokens, target = torch.randint(0, 30, (3, 17), device=dev), torch.randn(3, 17, 64, device=dev)

    def step():
        loss = (norm(emb(tokens)) - target).square().mean()
        loss.backward()
        return loss.detach(), genie_tk.clip_grad_norm_(params, 1e-2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            for p in params:
                p.grad = None
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, total = step()
    for seed in range(2):
        torch.manual_seed(seed)
        tokens.copy_(torch.randint(0, 30, (3, 17)))
        target.copy_(torch.randn(3, 17, 64))
        graph.replay()
        torch.cuda.synchronize()
        y = F.layer_norm(F.embedding(tokens, emb.weight.double(), 3), (64,), norm.weight.double(), norm.bias.double())
        want_loss = (y - target).square().mean()
        want = torch.autograd.grad(want_loss, params)
        full = torch.sqrt(sum(w.double().square().sum() for w in want))
        torch.testing.assert_close(loss.double(), want_loss, rtol=1e-5, atol=0)
        torch.testing.assert_close(total.double(), full, rtol=1e-5, atol=0)
        for p, w in zip(params, want):
            assert float((p.grad - w * (1e-2 / full)).norm()) <= 1e-4 * float((w * (1e-2 / full)).norm()) + 1e-9
    assert_status_clean(dev)


def test_block_backward_under_autocast():
    """A block's gradients when its backward is called under autocast: the recomputation's products
    are bf16 there (2^-8 a rounding at most, up to twelve in a row), its LayerNorms stay fp32."""
    dev = require_gpu()
    torch.manual_seed(4)
    block = genie_tk.TriangleMultiplicationOutgoing(128, 128).to(dev)
    for p in block.parameters():
        torch.nn.init.normal_(p, std=0.1)
    shape = (1, 20, 20, 128)
    x = torch.randn(shape, device=dev, requires_grad=True)
    mask = torch.ones(shape[:-1], device=dev)
    dy = torch.randn(shape, device=dev)
    grads = []
    for cast in (False, True):
        y = block(x, mask)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=cast):
            grads.append(torch.autograd.grad(y, [x, *block.parameters()], dy))
    for a, b in zip(*grads):
        assert a.dtype == b.dtype and float((a - b).norm()) <= 0.05 * float(a.norm())
