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

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

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
    """``t`` as (rows, cols) with a row stride the kernels can address in place, else a contiguous copy."""
    if t.is_contiguous():
        t = t.view(-1, cols)
    else:
        t = t.reshape(-1, cols)
        per_word = 16 // t.element_size()
        if t.stride(1) != 1 or cols % per_word or t.stride(0) % per_word:
            t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]   # (a single row may carry any stride)


def _forward(x, residual, weight, eps):
    """x, residual: (rows, cols); returns (y, h), h None without a residual."""
    rows, cols = x.shape
    y = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    h = None if residual is None else torch.empty_like(y)
    rc = _cabi.load().b200train_add_rms_norm(
        x.data_ptr(), _stride(x), None if residual is None else residual.data_ptr(), 0 if residual is None else _stride(residual),
        weight.data_ptr(), y.data_ptr(), None if h is None else h.data_ptr(), rows, cols, eps, _cabi.TRAIN_DTYPES[x.dtype],
        _cabi.TRAIN_DTYPES[weight.dtype], x.device.index, torch.cuda.current_stream(x.device).cuda_stream)
    _cabi.check(rc, "b200train_add_rms_norm")
    return y, h


def _weight(weight):
    weight = weight.contiguous()
    return weight if weight.data_ptr() % 16 == 0 else weight.clone()


class _add_rms_norm(torch.autograd.Function):
    """forward(x, residual or None, weight, eps) -> (y, h): h is the sum, or x itself where there is no residual."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        cols = x.shape[-1]
        x2, w = _rows(x, cols), _weight(weight)
        y, h = _forward(x2, None if residual is None else _rows(residual, cols), w, eps)
        ctx.save_for_backward(x2 if h is None else h, w)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y.view(x.shape), x if h is None else h.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, w = ctx.saved_tensors
        if dy is None:      # the norm was not used: the stream's gradient passes through
            return dh, dh if ctx.needs_input_grad[1] else None, None, None
        rows, cols = h.shape
        shape = dy.shape
        dy = _rows(dy, cols)
        if dh is not None:
            dh = _rows(dh, cols)
        lib = _cabi.load()
        dt, dev = _cabi.TRAIN_DTYPES[h.dtype], h.device
        dx = torch.empty((rows, cols), dtype=h.dtype, device=dev)
        dw = scratch = None
        floats = 0
        if ctx.needs_input_grad[2]:
            dw = torch.empty_like(w)
            floats = lib.b200train_norm_scratch_floats(rows, cols, dt, dev.index)
            scratch = torch.empty(floats, dtype=torch.float32, device=dev)
        rc = lib.b200train_add_rms_norm_bwd(
            dy.data_ptr(), _stride(dy), None if dh is None else dh.data_ptr(), 0 if dh is None else _stride(dh), h.data_ptr(), _stride(h),
            w.data_ptr(), dx.data_ptr(), None if dw is None else dw.data_ptr(), None if scratch is None else scratch.data_ptr(), floats, rows,
            cols, ctx.eps, dt, _cabi.TRAIN_DTYPES[w.dtype], dev.index, torch.cuda.current_stream(dev).cuda_stream)
        _cabi.check(rc, "b200train_add_rms_norm_bwd")
        dx = dx.view(shape)
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-5):
    """``(y, h)``: h = x + residual in the tensors' type, y = the RMS norm of h times ``weight``.

    With ``residual=None`` h is ``x`` itself: passing the stream through the norm this way lets the backward add the
    stream's gradient in the same kernel.
    """
    _check("add_rms_norm", x, residual, weight, eps)
    return _add_rms_norm.apply(x, residual, weight, float(eps))


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """The RMS norm of ``x`` over its last dimension, times ``weight``."""
    _check("rms_norm", x, None, weight, eps)
    return _add_rms_norm.apply(x, None, weight, float(eps))[0]


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
