"""Utility functions with the reference's names (src/genie_tk/utils.py)."""

from __future__ import annotations

import math
from typing import Any, Callable, Dict, Iterable, Union

import torch
from torch import Tensor

from . import _lib, ops


def has_cuda_kernels() -> bool:
    """True when the B200 kernel library loads and a CUDA device is present (utils.py:12-18)."""
    return _lib.available() and torch.cuda.is_available()


def get_device_info() -> Dict[str, Any]:
    """Device summary (utils.py:21-42), plus the library version."""
    info: Dict[str, Any] = {
        "cuda_available": torch.cuda.is_available(),
        "cuda_kernels_available": has_cuda_kernels(),
        "device_count": 0,
        "devices": [],
        "library": _lib.LIB_PATH,
        "library_version": _lib.load().gtk_version() if _lib.available() else None,
    }
    if torch.cuda.is_available():
        info["device_count"] = torch.cuda.device_count()
        for i in range(info["device_count"]):
            props = torch.cuda.get_device_properties(i)
            info["devices"].append({
                "name": props.name,
                "total_memory": props.total_memory,
                "major": props.major,
                "minor": props.minor,
                "multi_processor_count": props.multi_processor_count,
            })
    return info


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> Tensor:
    """torch.nn.utils.clip_grad_norm_ on the library's kernels: scale the parameters' gradients
    in place by min(1, max_norm / (norm + 1e-6)) and return their total norm (0-d, fp32).

    ``norm_type`` is 2.0 or inf. Two launches for up to 1000 gradients, nothing copied to or from
    the host; with ``error_if_nonfinite`` the norm is read back first, and a norm that is NaN or
    infinite raises with the gradients left as they were."""
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not math.isfinite(float(ops.grad_norm(grads, float(norm_type)))):
        raise RuntimeError(f"genie_tk (B200): the total norm of order {norm_type} of the gradients is not finite, so it "
                           "cannot be clipped; error_if_nonfinite=False scales by it anyway")
    return ops.clip_grad_norm(grads, float(max_norm), float(norm_type))


def permute_final_dims(tensor: Tensor, *dims: int) -> Tensor:
    """Permute the trailing ``len(dims)`` axes (utils.py:45-60)."""
    lead = tensor.dim() - len(dims)
    return tensor.permute(list(range(lead)) + [lead + d for d in dims])


def flatten_final_dims(tensor: Tensor, num_dims: int) -> Tensor:
    """Flatten the trailing ``num_dims`` axes (utils.py:63-75)."""
    return tensor.reshape(tensor.shape[:-num_dims] + (-1,))


def chunk_layer(layer: Callable, inputs: Dict[str, Tensor], chunk_size: int, no_batch_dims: int) -> Tensor:
    """Apply ``layer`` over the flattened leading batch axes in chunks (utils.py:78-123)."""
    first = next(iter(inputs.values()))
    batch_shape = first.shape[:no_batch_dims]
    flat = {k: v.reshape((-1,) + v.shape[no_batch_dims:]) for k, v in inputs.items()}
    total = next(iter(flat.values())).shape[0]
    outs = [layer(**{k: v[s:s + chunk_size] for k, v in flat.items()}) for s in range(0, total, chunk_size)]
    out = torch.cat(outs, dim=0)
    return out.reshape(batch_shape + out.shape[1:])
