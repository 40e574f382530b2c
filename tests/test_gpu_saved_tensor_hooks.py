"""Saved-tensor hooks between the passes of the norm and the router: what a hook gives back has the saved values, but not
the memory order, the alignment or the place they had.  Gradients are those of the same call without a hook, to the bit."""
import pytest
import torch

from oregon_gpt_oss_patching_b200.moe_router import router_topk
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _columns_first(t):
    return t.clone() if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


def _off_the_grid(t):
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.view(t.shape).copy_(t)


HOOKS = {
    "clone": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t),
    "compact": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t),
    "cpu": lambda: torch.autograd.graph.save_on_cpu(),
    "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "columns_first": lambda: torch.autograd.graph.saved_tensors_hooks(_columns_first, lambda t: t),
    "off_the_grid": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, _off_the_grid),
    "wider_rows": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t, lambda t: t if t.dim() < 2 else torch.cat([t, t[..., :16]], -1)[..., :t.shape[-1]]),
}


def _rows(cols, dtype):
    g = torch.Generator().manual_seed(cols)
    big = torch.randn(40, cols + 64, generator=g).to(device=DEV, dtype=dtype)
    return {"rows": big[:, 8:cols + 8], "whole": big[:, :cols].contiguous(), "one_for_all": big[:1, :cols].expand(40, cols),
            "off": big[:, 3:cols + 3], "deep": big.view(2, 4, 5, cols + 64)[..., 16:cols + 16]}


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("cols", [2880, 33])
def test_norm(hook, cols):
    for dtype in (torch.bfloat16, torch.float32):
        for x in _rows(cols, dtype).values():
            w = torch.randn(2 * cols, generator=torch.Generator().manual_seed(1)).to(DEV)[::2]     # (kept as a copy)
            dy, dh = torch.randn_like(x), torch.randn_like(x)

            def grads(call, *outs):
                leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
                return torch.autograd.grad(call(*leaves), leaves, outs)

            calls = [(lambda a, b: rms_norm(a, b), (dy,)), (lambda a, b: add_rms_norm(a, None, b), (dy, dh)),
                     (lambda a, b: add_rms_norm(a, a.detach(), b), (dy, dh))]
            for call, outs in calls:
                plain = grads(call, *outs)
                with HOOKS[hook]():
                    hooked = grads(call, *outs)
                assert all(torch.equal(p, q) for p, q in zip(plain, hooked))


@pytest.mark.parametrize("hook", list(HOOKS))
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_router(hook, scoring):
    for dtype in (torch.bfloat16, torch.float32):
        big = torch.randn(50, 80, generator=torch.Generator().manual_seed(2)).to(device=DEV, dtype=dtype)
        for logits in (big[:, 5:37], big[:, 8:40], big.t()[:33, :32], big[:1, :32].expand(9, 32), big):
            d = torch.randn(len(logits), 4, generator=torch.Generator().manual_seed(3)).to(device=DEV, dtype=dtype)

            def grads():
                leaf = logits.detach().requires_grad_(True)
                w, _ = router_topk(leaf, 4, scoring=scoring, renormalize=False)
                return torch.autograd.grad(w, leaf, d)[0]

            plain = grads()
            with HOOKS[hook]():
                hooked = grads()
            assert torch.equal(plain, hooked)


@pytest.mark.parametrize("wrong", [lambda t: t.double(), lambda t: t[:-1], lambda t: t.cpu()])
def test_what_a_hook_gives_back_must_be_what_was_saved(wrong):
    x = torch.randn(12, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
        y = rms_norm(x, w)
        t, _ = router_topk(x, 4)
        for out in (y, t):
            with pytest.raises(RuntimeError, match="saved"):
                torch.autograd.grad(out.sum(), x)
