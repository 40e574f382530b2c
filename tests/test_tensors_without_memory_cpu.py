"""CUDA tensors that have no memory of their own are refused before an address is made of them (no GPU needed)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oregon_gpt_oss_patching_b200 import build
from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step, global_grad_norm
from oregon_gpt_oss_patching_b200.moe_router import router_topk
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm


class _Wrapper(torch.Tensor):
    """Shape, type and device of a tensor; what it stands for is elsewhere."""

    @staticmethod
    def __new__(cls, like, offset=0):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, strides=like.stride(), storage_offset=offset, dtype=like.dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(f"{func} of a wrapper")


def _calls(x, w):
    return [lambda: rms_norm(x, w), lambda: add_rms_norm(x, x, w), lambda: add_rms_norm(x, None, w), lambda: router_topk(x, 4),
            lambda: router_topk(x, 4, bias=w), lambda: global_grad_norm([x])]


def test_fake_tensors():
    build.build()
    with FakeTensorMode():
        x, w = torch.randn(9, 64, device="cuda"), torch.ones(128, device="cuda")
        for rows, weight in ((x, w[:64]), (x[2:], w[64:])):            # at the start of no memory, and an offset behind it
            p = torch.nn.Parameter(weight)
            p.grad = weight.clone()
            for call in _calls(rows, weight) + [lambda: clip_grad_norm([p], 1.0), lambda: clipped_sgd_step([p], 1.0)]:
                with pytest.raises(RuntimeError, match="memory of their own"):
                    call()


@pytest.mark.parametrize("offset", [0, 64])
def test_wrappers(offset):
    x, w = _Wrapper(torch.empty(9, 64), offset), _Wrapper(torch.empty(64), offset)
    for call in _calls(x, w):
        with pytest.raises(RuntimeError, match="memory of their own|data pointer|storage"):
            call()
