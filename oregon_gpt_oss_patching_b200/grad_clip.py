"""The global gradient norm, clipping by it, and the state-free SGD update with the clip folded in.

The reference's launcher clips gradients at a norm of 1.0 (``configs/zero3.yaml:6``).  Here that is two launches for up to
256 tensors, whatever their sizes and types, behind the C ABI of ``include/b200train.h``: one reads every gradient once, the
other knows the norm and writes the gradients (nothing, where they are under the limit) or the updated parameters.  Nothing
synchronises with the host, and both calls can be captured into a graph:

    n = sqrt(sum of g^2),   c = min(1, max_norm / (n + 1e-6)),   g <- c g     or     p <- p - lr c g

``clip_grad_norm`` stands in for ``torch.nn.utils.clip_grad_norm_`` (2-norm; the same ``c``, the same handling of a norm that
is not finite, except that an infinite ``max_norm`` is no limit and never scales); ``clipped_sgd_step`` for a clip followed by ``p -= lr * g``, with two thirds of the memory traffic and one
rounding instead of two; the gradients stay as they were.  Tensors are bf16, fp16 or fp32, mixed at will, a parameter and
its gradient of one type, all on one device.  Results are bit-reproducible: every sum has an order fixed by the sizes.
"""
from __future__ import annotations

from typing import Iterable, Union

import torch

from . import _binding

__all__ = ["global_grad_norm", "clip_grad_norm", "clipped_sgd_step"]

_Tensors = Union[torch.Tensor, Iterable[torch.Tensor]]


def _listed(tensors: _Tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def global_grad_norm(tensors: _Tensors) -> torch.Tensor:
    """The 2-norm of all the tensors' elements together, an fp32 scalar on their device (0 on the CPU for no tensors), without a gradient."""
    return _binding.load().global_grad_norm(_listed(tensors))


def clip_grad_norm(parameters: _Tensors, max_norm: float) -> torch.Tensor:
    """Scale the parameters' gradients in place so that their global 2-norm is at most ``max_norm``; returns the norm before.

    Parameters without a gradient are passed over.  Gradients that share an element (one parameter given twice, overlapping views), or
    one that has an element twice, are refused before anything is written; views that only lie in between each other are fine.
    """
    return _binding.load().clip_grad_norm(_listed(parameters), max_norm)


def clipped_sgd_step(parameters: _Tensors, lr: float, max_norm: float = float("inf")) -> torch.Tensor:
    """``p -= lr * c * p.grad`` for every parameter that has a gradient, c from the global norm of the gradients; returns the norm.

    The gradients are not changed.  A parameter that shares an element with another one or with a gradient, or has one twice, is
    refused before anything is written, and so are contiguous gradients that share memory.
    """
    return _binding.load().clipped_sgd_step(_listed(parameters), lr, max_norm)
