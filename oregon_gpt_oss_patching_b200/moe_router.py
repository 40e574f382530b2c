"""The choice of experts in front of ``moe_experts``: scores, top-k and weights as one kernel per direction.

``GptOssTopKRouter.forward`` (``transformers/models/gpt_oss/modeling_gpt_oss.py:126-133``) takes the top-k of the router's logits
and their softmax.  ``router_topk`` does so in one launch (``b200moe_router_topk``, ``include/b200moe.h``), and its backward
writes the logits' gradient in another; ``patch_moe_router`` puts it into the model, exactly as the experts' patch does.  It also
takes the other ways in which mixtures of experts are routed: sigmoid scores, a bias that takes part in the choice but not in the
weights (to balance the load without a loss), experts in groups of which only the best are eligible, weights that are not
renormalised, and a factor on them.

The choice is exact: it follows the order of the real numbers, ties go to the lowest index (``torch.topk`` leaves them open on
a GPU), and results are bit-reproducible.  A logit of -inf masks an expert: it is chosen only where nothing else is left, with
weight 0.  There is no other code path: if the library is missing or rejects a call an exception is raised.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _cabi

__all__ = ["router_topk", "b200_router_forward", "patch_moe_router", "unpatch_moe_router"]

_SCORINGS = {"softmax": 0, "sigmoid": 1}


def _check(logits, top_k, scoring, bias, num_groups, top_groups):
    if not logits.is_cuda:
        raise RuntimeError("router_topk needs CUDA tensors (the sm_100a library is the only code path)")
    if logits.dtype not in _cabi.MOE_DTYPES:
        raise TypeError(f"router_topk supports bfloat16, float16 and float32 logits, got {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"router_topk: logits must be (tokens, experts), got {tuple(logits.shape)}")
    if scoring not in _SCORINGS:
        raise ValueError(f"router_topk: scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    E = logits.shape[1]
    if not 1 <= E <= _cabi.MOE_ROUTER_MAX_EXPERTS:
        raise ValueError(f"router_topk: 1 to {_cabi.MOE_ROUTER_MAX_EXPERTS} experts, got {E}")
    if not 1 <= num_groups <= _cabi.MOE_ROUTER_MAX_GROUPS or E % num_groups or not 1 <= top_groups <= num_groups:
        raise ValueError(f"router_topk: {E} experts cannot form {num_groups} equal groups of which {top_groups} are eligible")
    if not 1 <= top_k <= min(_cabi.MOE_ROUTER_MAX_TOP_K, E // num_groups * top_groups):
        raise ValueError(f"router_topk: cannot choose {top_k} of {E // num_groups * top_groups} eligible experts (at most "
                         f"{_cabi.MOE_ROUTER_MAX_TOP_K})")
    if bias is not None and (bias.shape != (E,) or bias.device != logits.device or not bias.is_floating_point()):
        raise ValueError(f"router_topk: bias must be {E} floating point values on {logits.device}")


class _router_topk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, top_k, sigmoid, num_groups, top_groups, renormalize, scale):
        if logits.stride(1) != 1 and logits.shape[1] > 1:
            logits = logits.contiguous()
        T, E = logits.shape
        if bias is not None:
            bias = bias.to(torch.float32).contiguous()
        weights = torch.empty((T, top_k), dtype=logits.dtype, device=logits.device)
        indices = torch.empty((T, top_k), dtype=torch.int64, device=logits.device)
        dev = logits.device
        rc = _cabi.load().b200moe_router_topk(
            logits.data_ptr(), logits.stride(0), None if bias is None else bias.data_ptr(), weights.data_ptr(), indices.data_ptr(), T, E,
            top_k, num_groups, top_groups, sigmoid, renormalize, scale, _cabi.MOE_DTYPES[logits.dtype], dev.index,
            torch.cuda.current_stream(dev).cuda_stream)
        _cabi.check(rc, "b200moe_router_topk")
        ctx.save_for_backward(logits, indices)
        ctx.how = sigmoid, renormalize, scale
        ctx.mark_non_differentiable(indices)
        return weights, indices

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        logits, indices = ctx.saved_tensors
        sigmoid, renormalize, scale = ctx.how
        T, E = logits.shape
        dev = logits.device
        dweights = dweights.contiguous()
        dlogits = torch.empty((T, E), dtype=logits.dtype, device=dev)
        rc = _cabi.load().b200moe_router_topk_bwd(
            logits.data_ptr(), logits.stride(0), indices.data_ptr(), dweights.data_ptr(), dlogits.data_ptr(), T, E, indices.shape[1], sigmoid,
            renormalize, scale, _cabi.MOE_DTYPES[logits.dtype], dev.index, torch.cuda.current_stream(dev).cuda_stream)
        _cabi.check(rc, "b200moe_router_topk_bwd")
        return dlogits, None, None, None, None, None, None, None


def router_topk(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
                top_groups: Optional[int] = None, renormalize: bool = True, scale: float = 1.0):
    """``(weights, indices)`` of the ``top_k`` experts of every token, both (tokens, top_k), best first.

    logits (tokens, experts): bf16, fp16 or fp32, at most 256 experts; weights have the logits' type, indices are int64, as
    ``moe_experts`` takes them.  ``scoring`` is "softmax" (over all experts) or "sigmoid"; ``bias`` (experts) is added to the scores
    for the choice alone and gets no gradient; with ``num_groups`` only the experts of the ``top_groups`` groups with the
    largest sums of their two best values are eligible; ``renormalize`` divides the weights by their sum; ``scale`` multiplies them.
    """
    top_groups = num_groups if top_groups is None else top_groups
    _check(logits, top_k, scoring, bias, num_groups, top_groups)
    return _router_topk.apply(logits, None if bias is None else bias.detach(), int(top_k), _SCORINGS[scoring], int(num_groups), int(top_groups),
                              int(bool(renormalize)), float(scale))


def b200_router_forward(self, hidden_states: torch.Tensor):
    """Same signature and result as ``GptOssTopKRouter.forward`` (modeling_gpt_oss.py:126-133)."""
    router_logits = torch.nn.functional.linear(hidden_states, self.weight, self.bias)
    router_scores, router_indices = router_topk(router_logits, self.top_k)
    return router_logits, router_scores, router_indices


_original_router_forward = None


def patch_moe_router():
    """Route every ``GptOssTopKRouter`` through ``router_topk`` (``unpatch_moe_router`` restores the original)."""
    global _original_router_forward
    from transformers.models.gpt_oss import modeling_gpt_oss
    if _original_router_forward is None:
        _original_router_forward = modeling_gpt_oss.GptOssTopKRouter.forward
    modeling_gpt_oss.GptOssTopKRouter.forward = b200_router_forward


def unpatch_moe_router():
    from transformers.models.gpt_oss import modeling_gpt_oss
    if _original_router_forward is not None:
        modeling_gpt_oss.GptOssTopKRouter.forward = _original_router_forward
