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

from . import _binding

__all__ = ["router_topk", "b200_router_forward", "patch_moe_router", "unpatch_moe_router"]

def router_topk(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
                top_groups: Optional[int] = None, renormalize: bool = True, scale: float = 1.0):
    """``(weights, indices)`` of the ``top_k`` experts of every token, both (tokens, top_k), best first.

    logits (tokens, experts): bf16, fp16 or fp32, at most 256 experts; weights have the logits' type, indices are int64, as
    ``moe_experts`` takes them.  ``scoring`` is "softmax" (over all experts) or "sigmoid"; ``bias`` (experts; bf16, fp16 or fp32)
    is added to the scores for the choice alone and gets no gradient; with ``num_groups`` only the experts of the ``top_groups`` groups with the
    largest sums of their two best values are eligible; ``renormalize`` divides the weights by their sum; ``scale`` multiplies them.
    """
    return _binding.load().router_topk(logits, top_k, scoring, bias, num_groups, num_groups if top_groups is None else top_groups, renormalize, scale)


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
