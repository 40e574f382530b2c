"""The global gradient norm, clipping by it, and the state-free SGD update with the clip folded in.

The reference's launcher clips gradients at a norm of 1.0 (``configs/zero3.yaml:6``).  Here that is two launches for up to
256 tensors, whatever their sizes and types, behind the C ABI of ``include/b200train.h``: one reads every gradient once, the
other knows the norm and writes the gradients (nothing, where they are under the limit) or the updated parameters.  Nothing
synchronises with the host, and both calls can be captured into a graph:

    n = sqrt(sum of g^2),   c = min(1, max_norm / (n + 1e-6)),   g <- c g     or     p <- p - lr c g

``clip_grad_norm`` stands in for ``torch.nn.utils.clip_grad_norm_`` (2-norm; the same ``c``, the same handling of a norm that
is not finite); ``clipped_sgd_step`` for a clip followed by ``p -= lr * g``, with two thirds of the memory traffic and one
rounding instead of two; the gradients stay as they were.  Tensors are bf16, fp16 or fp32, mixed at will, a parameter and
its gradient of one type, all on one device.  Results are bit-reproducible: every sum has an order fixed by the sizes.
"""
from __future__ import annotations

from array import array
from typing import Iterable, Union

import torch

from . import _cabi

__all__ = ["global_grad_norm", "clip_grad_norm", "clipped_sgd_step"]

_Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _listed(tensors: _Tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _device(name, tensors) -> int:
    found = {t.get_device() for t in tensors}
    if len(found) != 1 or -1 in found:
        raise RuntimeError(f"{name} needs CUDA tensors on one device (the sm_100a library is the only code path)")
    return found.pop()


def _addresses(tensors) -> array:
    return array("q", [t.data_ptr() for t in tensors])


def _host(a: array) -> int:
    return a.buffer_info()[0]


def _types(name, tensors) -> array:
    dtypes = array("i", [_cabi.TRAIN_DTYPES.get(t.dtype, -1) for t in tensors])
    if min(dtypes) < 0:
        raise TypeError(f"{name} supports bfloat16, float16 and float32, got {sorted({str(t.dtype) for t in tensors})}")
    return dtypes


def _run(name, grads, params, *numbers) -> torch.Tensor:
    """One call of the library on contiguous tensors; returns the norm."""
    dev = _device(name, grads + params if params else grads)
    dtypes, counts = _types(name, grads), array("q", [g.numel() for g in grads])
    lib = _cabi.load()
    doubles = lib.b200train_clip_scratch_doubles(len(grads), dev)
    scratch = torch.empty(doubles, dtype=torch.float64, device=grads[0].device)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    addresses, others = _addresses(grads), _addresses(params) if params else None
    args = [_host(addresses)] + ([_host(others)] if params else []) + [_host(counts), _host(dtypes), len(grads), *numbers]
    rc = getattr(lib, name)(*args, scratch.data_ptr(), doubles, norm.data_ptr(), dev, torch.cuda.current_stream(dev).cuda_stream)
    _cabi.check(rc, name)
    return norm


def _limit(name, max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{name}: max_norm must not be negative, got {max_norm}")
    return max_norm


def global_grad_norm(tensors: _Tensors) -> torch.Tensor:
    """The 2-norm of all the tensors' elements together, an fp32 scalar on their device."""
    grads = _listed(tensors)
    if not grads:
        return torch.tensor(0.0)
    return _run("b200train_grad_norm", [g if g.is_contiguous() else g.contiguous() for g in grads], None)


@torch.no_grad()
def clip_grad_norm(parameters: _Tensors, max_norm: float) -> torch.Tensor:
    """Scale the parameters' gradients in place so that their global 2-norm is at most ``max_norm``; returns the norm before.

    Parameters without a gradient are passed over.  Gradients that share memory are refused (one parameter given twice).
    """
    max_norm = _limit("clip_grad_norm", max_norm)
    grads = [p.grad for p in _listed(parameters) if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    strided = [g for g in grads if not g.is_contiguous()]
    if not strided:
        norm = _run("b200train_clip_grads", grads, None, max_norm)
    else:
        for g in strided:
            if any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                raise ValueError("clip_grad_norm: a gradient with a stride of 0 cannot be scaled in place")
        packed = [g if g.is_contiguous() else g.contiguous() for g in grads]
        norm = _run("b200train_clip_grads", packed, None, max_norm)
        for g, p in zip(grads, packed):
            if p is not g:
                g.copy_(p)
    torch.autograd.graph.increment_version(grads)
    return norm


@torch.no_grad()
def clipped_sgd_step(parameters: _Tensors, lr: float, max_norm: float = float("inf")) -> torch.Tensor:
    """``p -= lr * c * p.grad`` for every parameter that has a gradient, c from the global norm of the gradients; returns the norm.

    The gradients are not changed.  Parameters and gradients that share memory are refused.
    """
    lr, max_norm = float(lr), _limit("clipped_sgd_step", max_norm)
    params = [p for p in _listed(parameters) if p.grad is not None]
    if not params:
        return torch.tensor(0.0)
    for p in params:
        if p.grad.dtype != p.dtype:
            raise TypeError(f"clipped_sgd_step: a gradient must have its parameter's type, got {p.grad.dtype} for {p.dtype}")
    grads = [g if g.is_contiguous() else g.contiguous() for g in [p.grad for p in params]]
    packed = [p if p.is_contiguous() else p.contiguous() for p in params]
    norm = _run("b200train_clipped_sgd", grads, packed, lr, max_norm)
    for p, q in zip(params, packed):
        if q is not p:
            p.copy_(q)
    torch.autograd.graph.increment_version(params)
    return norm
