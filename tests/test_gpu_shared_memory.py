"""Clip and update over tensors that are not contiguous: memory that two of them share, or one has twice, is noticed before
anything is written; tensors that lie in between each other without sharing an element are taken."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def parameter(data, grad):
    p = torch.nn.Parameter(data)
    p.grad = grad
    return p


def like(grad):
    return parameter(torch.zeros(grad.shape, device=DEV, dtype=grad.dtype), grad)


def refused(call, params, error=RuntimeError, match="share memory"):
    kept = [(p.detach().clone(), p.grad.clone()) for p in params]
    with pytest.raises(error, match=match):
        call(params)
    for p, (data, grad) in zip(params, kept):
        assert torch.equal(p.detach(), data) and torch.equal(p.grad, grad)


def clip(params):
    return clip_grad_norm(params, 0.25)


def sgd(params):
    return clipped_sgd_step(params, 0.5, 0.25)


def test_gradients_that_overlap_are_refused():
    wide = torch.randn(40, 64, device=DEV)
    first = like(torch.randn(7, 5, device=DEV))
    refused(clip, [first, like(wide[:, :24]), like(wide[:, 8:32])])
    refused(clip, [first, like(wide[:, 8:32]), like(wide[3:4])])                       # one of them contiguous
    refused(clip, [first, like(wide[::2]), like(wide[2])])
    refused(clip, [like(wide[:, :24].t()), like(wide[:, 23:30]), first])
    turned = like(torch.randn(24, 40, device=DEV).t())
    refused(clip, [turned, first, turned])                                               # one parameter given twice
    refused(clip, [like(wide.as_strided((8, 6), (4, 1)))], ValueError, "share memory")      # rows that overlap one another


def test_parameters_that_overlap_are_refused():
    data, grad = torch.randn(12, 30, device=DEV), torch.randn(12, 30, device=DEV)
    first = parameter(torch.randn(3, 5, device=DEV), torch.randn(3, 5, device=DEV))
    refused(sgd, [first, parameter(data, grad.clone()), parameter(data.t(), grad.t().clone())])
    refused(sgd, [first, parameter(data[:, :9], grad[:, :9].clone()), parameter(data[:, 8:], grad[:, 8:].clone())])
    refused(sgd, [first, parameter(data.t(), data.t().clone()), parameter(torch.zeros(30, device=DEV), data[2])])   # a parameter as a gradient
    turned = parameter(data.t(), grad.t().clone())
    refused(sgd, [turned, first, turned])
    refused(sgd, [first, parameter(torch.ones(4, device=DEV).expand(10, 4), torch.ones(10, 4, device=DEV))], ValueError, "stride of 0")
    refused(sgd, [first, parameter(data.view(-1).as_strided((8, 6), (4, 1)), torch.ones(8, 6, device=DEV))], ValueError, "share memory")


def check_both(params):
    """Clip, then the update, against 64 bits: a result lacks at most 64 u of what it is made of and half a step of its own."""
    before = [(p.detach().clone(), p.grad.clone()) for p in params]
    ref = step_fp64.grad_norm([g for _, g in before])
    c = step_fp64.clip_coefficient(ref, 0.25)
    for norm in (sgd(params), clip(params)):
        assert abs(float(norm) - float(ref)) <= 34 * U * float(ref)
    for p, (data, grad) in zip(params, before):
        step = 0.5 * c * grad.double()
        assert bool(((p.detach().double() - (data.double() - step)).abs() <= 64 * U * (data.double().abs() + step.abs())).all())
        assert bool(((p.grad.double() - c * grad.double()).abs() <= 64 * U * (c * grad.double()).abs()).all())


def test_tensors_between_each_other_are_taken():
    def buffer(*shape):
        return torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape))).to(DEV)

    for cut in (lambda t: [t[:, :24], t[:, 24:32], t[:, 32:]], lambda t: [t[:, 24:].t(), t[:, :24].t()], lambda t: [t[::2], t[1::2]],
                lambda t: [t[:, ::3], t[:, 1::3], t[:, 2::3]], lambda t: [t[:5], t[5:].t()],
                lambda t: [t.view(10, 4, 64)[:, 0], t.view(10, 4, 64)[:, 1:3], t.view(10, 4, 64)[:, 3, ::2], t.view(10, 4, 64)[:, 3, 1::2]],
                lambda t: [t[:, 1::2], t[::2, ::2], t[1::2, ::2]]):
        data, grads = cut(buffer(40, 64)), cut(buffer(40, 64) * 2)
        check_both([parameter(d, g) for d, g in zip(data, grads)])
    t, g = buffer(4, 6, 8, 10), buffer(4, 6, 8, 10)
    check_both([parameter(a, b) for a, b in zip(t.permute(2, 0, 3, 1).split(3), g.permute(2, 0, 3, 1).split(3))])


def test_many_slices_of_one_buffer():
    data, grads = torch.randn(16, 600, device=DEV), torch.randn(16, 600, device=DEV)
    check_both([parameter(d, g) for d, g in zip(data.split(2, 1), grads.split(2, 1))])


def test_gradients_may_share_what_is_only_read():
    wide = torch.randn(40, 64, device=DEV)
    params = [parameter(torch.zeros(40, 24, device=DEV), wide[:, :24]), parameter(torch.zeros(40, 24, device=DEV), wide[:, 8:32])]
    kept = wide.clone()
    norm = sgd(params)
    ref = step_fp64.grad_norm([p.grad for p in params])
    assert abs(float(norm) - float(ref)) <= 34 * U * float(ref) and torch.equal(wide, kept)
