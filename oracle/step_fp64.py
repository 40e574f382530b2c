"""64-bit restatements of the steps of a fine-tuning step around attention and the experts (TEST INFRASTRUCTURE ONLY).

``add_rms_norm`` restates ``GptOssRMSNorm.forward`` (``transformers/models/gpt_oss/modeling_gpt_oss.py:57-63``) behind the sum
of ``GptOssDecoderLayer.forward`` (``:357-386``).  Gradients are written out as formulas; ``tests/test_step_oracle.py`` holds
them against differences, and the forward functions against the installed modules.
"""
import torch


def add_rms_norm(x, residual, weight, eps):
    """(y, h) in 64 bits.  The sum is rounded to x's type first, as the residual stream is a tensor of that type."""
    h = x.double() if residual is None else (x.double() + residual.double()).to(x.dtype).double()
    n = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return weight.double() * n, h


def add_rms_norm_bwd(h, weight, dy, dh, eps):
    """(dx, dweight) from the stream's row h; dh None where no gradient arrives through it."""
    h, w, dy = h.double(), weight.double(), dy.double()
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n, g = h * r, dy * w
    dx = r * (g - n * (g * n).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return dx, (dy * n).reshape(-1, h.shape[-1]).sum(0)


def grad_norm(grads):
    return torch.sqrt(sum((g.double() ** 2).sum() for g in grads))


def clip_coefficient(norm, max_norm):
    """min(1, max_norm / (norm + 1e-6)), NaN for a NaN norm: ``torch.nn.utils.clip_grad_norm_``."""
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)
