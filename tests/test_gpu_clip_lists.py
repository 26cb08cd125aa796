"""GPU tests of the lists that the gradient norm and clipping take: views that overlap in memory,
refused calls, sequences that make their items, copies on write, and factors below fp32's range.

Tolerances as in test_gpu_grad_clip.py."""

import math

import pytest
import torch

import genie_tk
from gpu_util import require_gpu
from test_gpu_grad_clip import U, _check_scaled, _make, _norm

pytestmark = pytest.mark.gpu


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
