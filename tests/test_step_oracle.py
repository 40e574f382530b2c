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


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_router_gradient_formula_against_autograd_and_differences(sigmoid, renormalize):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(5, 9, generator=g, dtype=torch.float64, requires_grad=True)
    _, idx = step_fp64.router_topk(logits.detach(), 3, sigmoid=sigmoid)
    d = torch.randn(5, 3, generator=g, dtype=torch.float64)

    def weights(l):
        w = (torch.sigmoid(l) if sigmoid else torch.softmax(l, 1)).gather(1, idx)
        return 2.5 * (w / w.sum(1, keepdim=True) if renormalize else w)

    w, _ = step_fp64.router_topk(logits.detach(), 3, sigmoid=sigmoid, renormalize=renormalize, scale=2.5)
    assert torch.allclose(w, weights(logits), rtol=1e-13)
    formula = step_fp64.router_topk_bwd(logits.detach(), idx, d, sigmoid=sigmoid, renormalize=renormalize, scale=2.5)
    (auto,) = torch.autograd.grad(weights(logits), logits, d)
    assert torch.allclose(formula, auto, rtol=1e-12, atol=1e-15)
    h = 1e-6
    for t, e in ((0, 0), (1, int(idx[1, 0])), (4, int(idx[4, 2]))):
        step = torch.zeros_like(logits)
        step[t, e] = h
        with torch.no_grad():
            diff = ((weights(logits + step) - weights(logits - step)) * d).sum() / (2 * h)
        assert abs(float(diff - formula[t, e])) < 1e-8


def test_router_restates_the_installed_module():
    from transformers import GptOssConfig
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssTopKRouter
    mod = GptOssTopKRouter(GptOssConfig(num_local_experts=16, num_experts_per_tok=4, hidden_size=24)).double()
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        mod.weight.copy_(torch.randn(16, 24, generator=g))
        mod.bias.copy_(torch.randn(16, generator=g))
        logits, scores, indices = mod(torch.randn(50, 24, generator=g, dtype=torch.float64))
    w, i = step_fp64.router_topk(logits, 4)
    assert torch.equal(i, indices) and torch.allclose(w, scores, rtol=1e-12)


def test_router_groups_by_hand():
    inf = float("inf")
    # groups (0.9, 0.1), (0.6, 0.6), (0.8, masked), (masked, masked)
    l = torch.tensor([[0.9, 0.1, 0.6, 0.6, 0.8, -inf, -inf, -inf]], dtype=torch.float64)
    zero = torch.zeros(8)
    p = torch.logit(l.clamp(1e-9, 1 - 1e-9)).masked_fill(torch.isneginf(l), -inf)
    w, i = step_fp64.router_topk(p, 3, sigmoid=True, bias=zero, groups=4, top_groups=2, renormalize=False)
    assert i.tolist() == [[0, 2, 3]] and torch.allclose(w, torch.tensor([[0.9, 0.6, 0.6]], dtype=torch.float64))
    _, i = step_fp64.router_topk(p, 4, sigmoid=True, bias=torch.tensor([0, 0, 0, 0, 0.7, 9.0, 9.0, 9.0]), groups=4, top_groups=2)
    assert i.tolist() == [[4, 2, 3, 5]]      # (0.6, 0.6) and (1.5); the masked expert of the second is last
