"""The 64-bit restatements of ``oracle/step_fp64.py`` against differences and against the installed modules (no GPU)."""
import pytest
import torch

from oracle import step_fp64


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h = step_fp64.add_rms_norm(x, residual, weight, eps)
        ctx.save_for_backward(h, weight)
        ctx.eps = eps
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        dx, dw = step_fp64.add_rms_norm_bwd(*ctx.saved_tensors, dy, dh, ctx.eps)
        return dx, dx, dw, None


@pytest.mark.parametrize("shape", [(3, 8), (2, 2, 5), (1, 1)])
def test_norm_gradient_formula_against_differences(shape):
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(*shape, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w = torch.randn(shape[-1], generator=g, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *t: _Norm.apply(*t, 1e-5), (x, r, w))


def test_norm_restates_the_installed_module():
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssRMSNorm
    mod = GptOssRMSNorm(24, eps=1e-5)
    g = torch.Generator().manual_seed(2)
    with torch.no_grad():
        mod.weight.copy_(torch.randn(24, generator=g))
    x = torch.randn(7, 24, generator=g)
    y, h = step_fp64.add_rms_norm(x, None, mod.weight.detach(), 1e-5)
    # the module computes in fp32: a sum of 24 squares, a root, two products
    assert torch.allclose(mod(x).double(), y, rtol=32 * 2.0 ** -24, atol=0)
    assert torch.equal(h, x.double())


@pytest.mark.parametrize("max_norm", [0.0, 0.7, 100.0, float("inf")])
def test_clip_restates_torch(max_norm):
    g = torch.Generator().manual_seed(3)
    params = [torch.nn.Parameter(torch.zeros(n, dtype=torch.float64)) for n in (1, 5, 30)]
    for p in params:
        p.grad = torch.randn(p.shape, generator=g, dtype=torch.float64)
    before = [p.grad.clone() for p in params]
    norm = torch.nn.utils.clip_grad_norm_(params, max_norm)
    assert torch.allclose(norm, step_fp64.grad_norm(before), rtol=1e-14)
    c = step_fp64.clip_coefficient(norm, max_norm)
    for p, b in zip(params, before):
        assert torch.allclose(p.grad, b * c, rtol=1e-14)
