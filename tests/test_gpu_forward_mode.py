"""Forward-mode derivatives of the training-step operators: refused, as the attention, rotary and expert calls refuse them, not
dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step, global_grad_norm
from oregon_gpt_oss_patching_b200.moe_router import router_topk
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_dual_tensors_are_refused():
    x, r, w = torch.randn(5, 32, device=DEV), torch.randn(5, 32, device=DEV), torch.ones(32, device=DEV)
    with fwad.dual_level():
        dx, dr, dw = (fwad.make_dual(t, torch.ones_like(t)) for t in (x, r, w))
        calls = [lambda: rms_norm(dx, w), lambda: rms_norm(x, dw), lambda: add_rms_norm(x, dr, w), lambda: add_rms_norm(dx, None, w),
                 lambda: add_rms_norm(x, r, dw), lambda: router_topk(dx, 4), lambda: router_topk(x, 4, bias=dw), lambda: global_grad_norm([x, dx])]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        p = torch.nn.Parameter(x.clone())
        p.grad = dx
        for call in (lambda: clip_grad_norm([p], 0.1), lambda: clipped_sgd_step([p], 0.1)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(fwad.unpack_dual(p.grad).primal, x) and torch.equal(p.detach(), x)
        rms_norm(x, w), router_topk(x, 4), add_rms_norm(x, r, w)       # what has no tangent is computed as ever


def test_a_parameter_with_a_tangent_is_not_updated():
    with fwad.dual_level():
        p = fwad.make_dual(torch.ones(8, device=DEV), torch.ones(8, device=DEV))
        p.grad = torch.ones(8, device=DEV)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            clipped_sgd_step([p], 0.1)
        assert bool((fwad.unpack_dual(p).primal == 1).all())
