"""The router far out: sigmoid scores of large negative logits, infinite logits in front of groups.

Tolerances.  u = 2^-24.  A weight is a quotient of exponentials whose arguments differ by at most the row's spread D: their
rounding gives D u, the exponentials, sums and quotients 64 u more (as in the router's other tests).  Below the smallest normal
number a value is off by a few of the subnormals instead: 8 * 2^-149, and half a subnormal of the type it is rounded to."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200.moe_router import router_topk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def rounding(ref, dtype):
    subnormal = {BF16: 2.0 ** -133, FP16: 2.0 ** -24, FP32: 2.0 ** -149}[dtype]
    return torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * ref.abs() + subnormal / 2 + 8 * 2.0 ** -149


def rows(base, mixed, dtype):
    l = torch.randn(40, 64, generator=torch.Generator().manual_seed(int(-base) + mixed)) * 2 + base
    if mixed:                                         # some experts near 0, so that the chosen lie on both sides
        l[:, :: 64 // mixed] -= base
    return l.to(device=DEV, dtype=dtype)


@pytest.mark.parametrize("base", [-80.0, -87.0, -89.0, -95.0, -103.0, -200.0, -650.0])
@pytest.mark.parametrize("mixed", [0, 2])
@pytest.mark.parametrize("top_k,groups", [(4, 1), (8, 4), (12, 1), (5, 2)])
def test_sigmoid_shares_of_large_negative_logits(base, mixed, top_k, groups):
    for dtype in (BF16, FP16, FP32):
        for renormalize in (True, False):
            logits = rows(base, mixed, dtype)
            leaf = logits.clone().requires_grad_(True)
            how = dict(sigmoid=True, renormalize=renormalize, scale=2.5)
            w, i = router_topk(leaf, top_k, scoring="sigmoid", num_groups=groups, renormalize=renormalize, scale=2.5)
            ref_w, ref_i = step_fp64.router_topk(logits, top_k, groups=groups, top_groups=groups, **how)
            assert torch.equal(i, ref_i)
            chosen = logits.double().gather(1, i)
            spread = chosen.amax(1, keepdim=True) - chosen if renormalize else chosen.abs()
            k = 64 + spread
            assert bool(((w.double() - ref_w).abs() <= rounding(ref_w, dtype) + k * U * ref_w.abs()).all())
            d = torch.randn(40, top_k, generator=torch.Generator().manual_seed(4)).to(device=DEV, dtype=dtype)
            (dl,) = torch.autograd.grad(w, leaf, d)
            ref = step_fp64.router_topk_bwd(logits, ref_i, d, **how)
            s, a = ref_w.abs() / 2.5, d.double().abs() * 2.5
            size = torch.zeros_like(ref).scatter(1, ref_i, k * s * (a + (k / 64 * a * s).sum(1, keepdim=True)))
            assert bool(((dl.double() - ref).abs() <= rounding(ref, dtype) + 2 * U * size + 64 * 2.0 ** -149).all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masks_of_the_type_s_lowest_value(dtype, scoring):
    low = torch.finfo(dtype).min
    l = torch.full((3, 32), low, device=DEV, dtype=dtype)
    l[1, 7], l[1, 20] = 1.0, 1.0
    leaf = l.clone().requires_grad_(True)
    w, i = router_topk(leaf, 4, scoring=scoring)
    assert i.tolist() == [[0, 1, 2, 3], [7, 20, 0, 1], [0, 1, 2, 3]]
    assert w.tolist() == [[0.25] * 4, [0.5, 0.5, 0.0, 0.0], [0.25] * 4]          # equal logits have equal shares, however low
    d = torch.tensor([[1.0, 2.0, 3.0, 6.0]], device=DEV, dtype=dtype).expand(3, 4)
    (dl,) = torch.autograd.grad(w, leaf, d)
    assert bool(torch.isfinite(dl).all())
    assert dl[0, :5].tolist() == [-0.5, -0.25, 0.0, 0.75, 0.0]                     # (d - 3) / 4
    slope = 0.5 * (1.0 if scoring == "softmax" else 1 / (1 + 2.718281828459045))    # r (d - 1.5), times 1 - s
    assert dl[1, 7].item() == pytest.approx(-0.5 * slope, rel=2.0 ** -7) and dl[1, 20].item() == pytest.approx(0.5 * slope, rel=2.0 ** -7)


@pytest.mark.parametrize("groups,top_groups", [(8, 3), (4, 2), (2, 1), (16, 5)])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_an_infinite_logit_does_not_open_a_masked_group(groups, top_groups, with_bias, dtype):
    """A softmax over +inf has no score that is a number: every expert that is not masked ranks alike, and groups follow their
    lowest index; a group that is masked as a whole comes last, in every form of the election."""
    l = (torch.randn(20, 64, generator=torch.Generator().manual_seed(5)) * 2).to(device=DEV, dtype=dtype)
    size = 64 // groups
    l[:, :size] = -INF                                   # the first group is masked
    l[::2, 2 * size - 1] = INF
    l[1::4, 63] = INF
    bias = torch.linspace(-1, 1, 64, device=DEV) if with_bias else None
    k = min(4, size)
    _, i = router_topk(l, k, bias=bias, num_groups=groups, top_groups=top_groups)
    # (on the CPU: what torch's sort does with NaN on a GPU depends on the sort's size)
    _, ref = step_fp64.router_topk(l.cpu(), k, bias=None if bias is None else bias.cpu(), groups=groups, top_groups=top_groups)
    assert torch.equal(i.cpu(), ref)
    if top_groups < groups:
        assert bool((i >= size).all())


def test_a_bias_keeps_all_its_bits():
    l = torch.randn(5, 32, device=DEV)
    with pytest.raises(TypeError, match="bias"):
        router_topk(l, 4, scoring="sigmoid", bias=torch.zeros(32, device=DEV, dtype=torch.float64))
    for dtype in (BF16, FP16, FP32):
        b = (torch.randn(32, generator=torch.Generator().manual_seed(6)) * 0.1).to(device=DEV, dtype=dtype)
        _, i = router_topk(l, 4, scoring="sigmoid", bias=b)
        assert torch.equal(i, step_fp64.router_topk(l, 4, sigmoid=True, bias=b)[1])
