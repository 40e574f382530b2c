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


def router_topk(logits, top_k, sigmoid=False, bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(weights, indices) in 64 bits; ``GptOssTopKRouter.forward`` (modeling_gpt_oss.py:126-133) with its defaults."""
    l = logits.double()
    masked = torch.isneginf(l)
    s = _scores(l, sigmoid)
    v = l if bias is None and groups == 1 else s + (0.0 if bias is None else bias.double())
    v = v.masked_fill(masked, -torch.inf)
    if groups > 1:
        parts = v.view(len(v), groups, -1)
        best = parts.sort(dim=-1, descending=True).values[..., :2]
        value = torch.where(torch.isneginf(best[..., 0]), best[..., 0], best.masked_fill(torch.isneginf(best), 0.0).sum(-1))
        kept = value.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        closed = torch.ones_like(value, dtype=torch.bool).scatter(1, kept, False).repeat_interleave(parts.shape[-1], dim=1)
        # masked experts of an eligible group still rank above every expert of a closed one
        rank = torch.where(closed, 2, masked.int())
        if bias is None:   # scores rise with logits, past the point where 64 bits tell them apart
            v = l
        order = v.sort(dim=1, descending=True, stable=True).indices
        order = order.gather(1, rank.gather(1, order).sort(dim=1, stable=True).indices)
        indices = order[:, :top_k]
    else:
        indices = v.sort(dim=1, descending=True, stable=True).indices[:, :top_k]
    w = s.gather(1, indices)
    if renormalize:
        total = w.sum(1, keepdim=True)
        if not sigmoid:   # the quotient does not depend on the experts left out
            m = l.gather(1, indices).amax(1, keepdim=True)
            w = torch.where(torch.isneginf(m), torch.zeros_like(w), torch.exp(l.gather(1, indices) - m))
            total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale, indices


def _scores(l, sigmoid):
    if sigmoid:
        return 1.0 / (1.0 + torch.exp(-l))
    m = l.amax(1, keepdim=True)
    e = torch.where(torch.isneginf(l), torch.zeros_like(l), torch.exp(l - m))
    z = e.sum(1, keepdim=True)
    return torch.where(z == 0, torch.zeros_like(e), e / z)


def router_topk_bwd(logits, indices, dweights, sigmoid=False, renormalize=True, scale=1.0):
    """dlogits from the gradient of the weights, by the formula."""
    l = logits.double()
    s = _scores(l, sigmoid)
    d = dweights.double() * scale
    if renormalize:
        chosen = s.gather(1, indices)
        if not sigmoid:
            lc = l.gather(1, indices)
            chosen = torch.where(torch.isneginf(lc), torch.zeros_like(lc), torch.exp(lc - lc.amax(1, keepdim=True)))
        total = chosen.sum(1, keepdim=True)
        r = torch.where(total == 0, torch.zeros_like(chosen), chosen / total)
        d = d - (d * r).sum(1, keepdim=True)
        dl = r * d * ((1 - chosen) if sigmoid else 1.0)
        return torch.zeros_like(l).scatter(1, indices, dl)
    ds = torch.zeros_like(l).scatter(1, indices, d)
    return ds * s * (1 - s) if sigmoid else s * (ds - (ds * s).sum(1, keepdim=True))
