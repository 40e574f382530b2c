"""Tensors that torch keeps negated lazily (the imaginary part of a conjugate): their values count, not what lies in memory."""
import pytest
import torch

from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step
from oregon_gpt_oss_patching_b200.moe_router import router_topk
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def negated(t):
    view = torch._neg_view(t.neg())
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_norm_and_router():
    x, r, dy, w = torch.randn(9, 64, device=DEV), torch.randn(9, 64, device=DEV), torch.randn(9, 64, device=DEV), torch.randn(64, device=DEV)
    bias = torch.randn(64, device=DEV) * 0.3

    def all_of(change):
        leaves = [change(t).detach().requires_grad_(True) for t in (x, r, w)]
        y, h = add_rms_norm(*leaves)
        z = rms_norm(change(x), change(w))
        grads = torch.autograd.grad((y, h), leaves, (change(dy), change(r)))
        logits = change(x).detach().requires_grad_(True)
        t, i = router_topk(logits, 4, scoring="sigmoid", bias=change(bias))
        return [y, h, z, *grads, t, i, torch.autograd.grad(t, logits, change(dy)[:, :4])[0]]

    for a, b in zip(all_of(lambda t: t), all_of(negated)):
        assert torch.equal(a, b)


def test_gradients_of_a_complex_product():
    """A parameter of one element takes the gradient as it comes, a negated view."""
    p = torch.nn.Parameter(torch.full((1,), 2.0, device=DEV))
    z = torch.complex(torch.ones(1, device=DEV), p)
    (z * z.conj()).real.backward()                     # 1 + p^2
    for grad in (p.grad, negated(torch.full((1,), 4.0, device=DEV))):
        p.grad = grad
        with torch.no_grad():
            p.fill_(2.0)
        assert float(clipped_sgd_step([p], 0.25)) == 4.0 and float(p) == 1.0
        clip_grad_norm([p], 1.0)
        assert float(p.grad) == pytest.approx(1.0, rel=1e-6)
    q = torch.nn.Parameter(negated(torch.ones(8, device=DEV)))
    q.grad = torch.full((8,), 0.5, device=DEV)
    clipped_sgd_step([q], 1.0)
    assert q.tolist() == [0.5] * 8


def test_a_negated_gradient_given_twice_is_refused():
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    p.grad = negated(torch.full((8,), 0.5, device=DEV))
    other = torch.nn.Parameter(torch.ones(8, device=DEV))
    other.grad = torch.ones(8, device=DEV)
    for call in (lambda: clip_grad_norm([other, p, p], 0.1), lambda: clipped_sgd_step([p, other, p], 0.1)):
        with pytest.raises(RuntimeError, match="share memory"):
            call()
    assert p.tolist() == other.tolist() == [1.0] * 8 and p.grad.tolist() == [0.5] * 8
