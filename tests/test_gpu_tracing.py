"""The training-step operators under torch's tracers: what would leave them out of a program without a word is refused."""
import pytest
import torch

from oregon_gpt_oss_patching_b200.grad_clip import global_grad_norm
from oregon_gpt_oss_patching_b200.moe_router import router_topk
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _all(x, w):
    y, h = add_rms_norm(x, x * 0.5, w)
    weights, indices = router_topk(rms_norm(y, w), 4)
    return y + h, weights, indices, global_grad_norm([x])


CALLS = {"rms_norm": lambda x, w: rms_norm(x * 2, w) + x, "add_rms_norm": lambda x, w: add_rms_norm(x * 2, x, w)[0] + x,
         "router_topk": lambda x, w: router_topk(x * 2, 4)[0] + x[:, :4], "global_grad_norm": lambda x, w: global_grad_norm([x * 2]) + x}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_trace_is_refused(name):
    """A trace would keep the results of the inputs that it was made with."""
    x, w = torch.randn(6, 64, device=DEV), torch.ones(64, device=DEV)
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        torch.jit.trace(CALLS[name], (x, w), check_trace=False)
    CALLS[name](x, w)


def test_a_compiled_function_calls_them():
    x, w = torch.randn(6, 64, device=DEV), torch.randn(64, device=DEV)
    compiled = torch.compile(_all, backend="eager")
    for t in (x, x + 1, x[:3]):
        for a, b in zip(compiled(t, w), _all(t, w)):
            assert torch.equal(a, b)
    leaf = x.clone().requires_grad_(True)
    (a,) = torch.autograd.grad(compiled(leaf, w)[0].sum(), leaf)
    (b,) = torch.autograd.grad(_all(leaf, w)[0].sum(), leaf)
    assert torch.equal(a, b)
