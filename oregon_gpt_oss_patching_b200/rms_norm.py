"""RMS norm with the residual sum in front of it, as one kernel per direction.

``GptOssDecoderLayer.forward`` (``transformers/models/gpt_oss/modeling_gpt_oss.py:357-386``) adds a block's output to
the residual stream and normalises the sum before the next block; ``GptOssRMSNorm.forward`` (``:57-63``) does so in eight
elementwise passes and a reduction over an fp32 copy, and autograd derives as many again.  ``add_rms_norm`` reads both
rows once, writes the sum and its norm once, and its backward makes the one gradient that both summands share from
the gradients of the norm and of the stream, behind the C ABI of ``include/b200train.h``:

    h = round(x + residual)          the residual stream, in the tensors' type
    y = round(weight * h * rsqrt(mean(h * h) + eps))

``rms_norm`` is the same without a sum.  ``patch_rms_norm`` puts both into the model, exactly as the attention patch does.
There is no other code path: if the library is missing or rejects a call an exception is raised.

Tensors are bf16, fp16 or fp32 of any leading shape; the weight has the tensors' type or fp32 (a checkpoint's norms are
kept in fp32).  Statistics, the weight's gradient and everything between are fp32; a result is rounded once.  The order of
every sum is fixed by the sizes, so results are bit-reproducible.  Rows of up to 16384 elements.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch

from . import _cabi

__all__ = ["rms_norm", "add_rms_norm", "b200_rms_norm_forward", "b200_decoder_layer_forward", "patch_rms_norm", "unpatch_rms_norm"]


def _check(name, x, residual, weight, eps):
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs CUDA tensors (the sm_100a library is the only code path)")
    if x.dtype not in _cabi.TRAIN_DTYPES:
        raise TypeError(f"{name} supports bfloat16, float16 and float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: x must have a last dimension to normalise, got shape {tuple(x.shape)}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"{name}: weight must be ({x.shape[-1]},), got {tuple(weight.shape)}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"{name}: weight must be {x.dtype} or float32, got {weight.dtype}")
    if weight.device != x.device:
        raise RuntimeError(f"{name}: weight is on {weight.device}, x on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"{name}: residual must match x ({tuple(x.shape)}, {x.dtype}, {x.device}), got "
                         f"{tuple(residual.shape)}, {residual.dtype}, {residual.device}")
    if not eps >= 0.0:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")


def _rows(t, cols):
    """``(tensor, row stride)`` that the kernels can address in place: ``t`` itself, rows of a view of it, or a contiguous copy."""
    if not t.is_contiguous():
        t = t.reshape(-1, cols)
        per_word = 16 // t.element_size()
        if t.is_contiguous() or t.stride(1) != 1 or cols % per_word or t.stride(0) % per_word:
            t = t.contiguous()
        elif t.data_ptr() % 16 == 0:
            return t, t.stride(0)
    return (t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)), cols


def _forward(x, residual, weight, eps):
    """Returns (y, h, weight, what the backward reads as h, its row stride); h is None without a residual."""
    cols = x.shape[-1]
    xr, x_stride = _rows(x, cols)
    w = weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else weight.clone(memory_format=torch.contiguous_format)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    dev = x.get_device()
    if residual is None:
        h, kept, kept_stride, r_ptr, r_stride, h_ptr = None, xr, x_stride, None, 0, None
    else:
        r, r_stride = _rows(residual, cols)
        h = torch.empty_like(y)
        kept, kept_stride, r_ptr, h_ptr = h, cols, r.data_ptr(), h.data_ptr()
    rc = _cabi.load().b200train_add_rms_norm(xr.data_ptr(), x_stride, r_ptr, r_stride, w.data_ptr(), y.data_ptr(), h_ptr, x.numel() // cols, cols,
                                             eps, _cabi.TRAIN_DTYPES[x.dtype], _cabi.TRAIN_DTYPES[w.dtype], dev, _cabi.stream_of(dev))
    _cabi.check(rc, "b200train_add_rms_norm")
    return y, h, w, kept, kept_stride


@lru_cache(maxsize=1024)
def _scratch_floats(rows, cols, dtype, dev):
    return _cabi.load().b200train_norm_scratch_floats(rows, cols, dtype, dev)


class _add_rms_norm(torch.autograd.Function):
    """forward(x, residual or None, weight, eps, passed) -> (y, h): h is the sum; without a residual x itself if `passed`, or None."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, passed):
        y, h, w, kept, ctx.h_stride = _forward(x, residual, weight, eps)
        if kept is h:       # (an output saved as it is would keep itself alive; a view shares its memory and its version)
            kept = h.detach()
        elif kept is x:
            kept = x.detach()
        ctx.save_for_backward(kept, w)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, (x if passed else None) if h is None else h

    @staticmethod
    def backward(ctx, dy, dh):
        if torch.is_grad_enabled():
            raise RuntimeError("add_rms_norm cannot be differentiated twice")
        if dy is None:      # the norm was not used: the stream's gradient passes through
            return dh, dh if ctx.needs_input_grad[1] else None, None, None, None
        h, w = ctx.saved_tensors
        cols = w.shape[0]
        rows = dy.numel() // cols
        wants = ctx.needs_input_grad
        dyr, dy_stride = _rows(dy, cols)
        dhr, dh_stride = (None, 0) if dh is None else _rows(dh, cols)
        dev = dy.get_device()
        dt = _cabi.TRAIN_DTYPES[dy.dtype]
        dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
        dw = scratch = None
        floats = 0
        if wants[2]:
            dw = torch.empty_like(w)
            floats = _scratch_floats(rows, cols, dt, dev)
            scratch = torch.empty(floats, dtype=torch.float32, device=dy.device)
        rc = _cabi.load().b200train_add_rms_norm_bwd(
            dyr.data_ptr(), dy_stride, None if dhr is None else dhr.data_ptr(), dh_stride, h.data_ptr(), ctx.h_stride, w.data_ptr(),
            dx.data_ptr(), None if dw is None else dw.data_ptr(), None if scratch is None else scratch.data_ptr(), floats, rows, cols, ctx.eps,
            dt, _cabi.TRAIN_DTYPES[w.dtype], dev, _cabi.stream_of(dev))
        _cabi.check(rc, "b200train_add_rms_norm_bwd")
        return dx, dx if wants[1] else None, dw, None, None


def _differentiates(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5):
    """``(y, h)``: h = x + residual in the tensors' type, y = the RMS norm of h times ``weight``.

    With ``residual=None`` h is ``x`` itself: passing the stream through the norm this way lets the backward add the
    stream's gradient in the same kernel.
    """
    eps = float(eps)
    _check("add_rms_norm", x, residual, weight, eps)
    if _differentiates(x, residual, weight):
        return _add_rms_norm.apply(x, residual, weight, eps, True)
    y, h, _, _, _ = _forward(x, residual, weight, eps)
    return y, x if h is None else h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """The RMS norm of ``x`` over its last dimension, times ``weight``."""
    eps = float(eps)
    _check("rms_norm", x, None, weight, eps)
    if _differentiates(x, weight):
        return _add_rms_norm.apply(x, None, weight, eps, False)[0]
    return _forward(x, None, weight, eps)[0]


def b200_rms_norm_forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
    """Same signature and result as ``GptOssRMSNorm.forward`` (modeling_gpt_oss.py:57-63)."""
    return rms_norm(hidden_states, self.weight, self.variance_epsilon)


def b200_decoder_layer_forward(self, hidden_states, attention_mask=None, position_ids=None, past_key_values=None, use_cache=False,
                               position_embeddings=None, **kwargs):
    """Same signature and result as ``GptOssDecoderLayer.forward`` (modeling_gpt_oss.py:357-386), its first sum and both norms fused."""
    norm = self.input_layernorm
    hidden_states, residual = add_rms_norm(hidden_states, None, norm.weight, norm.variance_epsilon)
    hidden_states, _ = self.self_attn(hidden_states=hidden_states, attention_mask=attention_mask, position_ids=position_ids,
                                      past_key_values=past_key_values, use_cache=use_cache, position_embeddings=position_embeddings, **kwargs)
    norm = self.post_attention_layernorm
    hidden_states, residual = add_rms_norm(hidden_states, residual, norm.weight, norm.variance_epsilon)
    hidden_states, _ = self.mlp(hidden_states)
    return residual + hidden_states


_originals = None


def patch_rms_norm():
    """Route every ``GptOssRMSNorm`` and ``GptOssDecoderLayer`` through the fused kernels (``unpatch_rms_norm`` restores the originals)."""
    global _originals
    from transformers.models.gpt_oss import modeling_gpt_oss
    if _originals is None:
        _originals = (modeling_gpt_oss.GptOssRMSNorm.forward, modeling_gpt_oss.GptOssDecoderLayer.forward)
    modeling_gpt_oss.GptOssRMSNorm.forward = b200_rms_norm_forward
    modeling_gpt_oss.GptOssDecoderLayer.forward = b200_decoder_layer_forward


def unpatch_rms_norm():
    from transformers.models.gpt_oss import modeling_gpt_oss
    if _originals is not None:
        modeling_gpt_oss.GptOssRMSNorm.forward, modeling_gpt_oss.GptOssDecoderLayer.forward = _originals
