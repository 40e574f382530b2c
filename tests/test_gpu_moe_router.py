"""The choice of experts (`b200moe_router_topk`, `_bwd`) on the GPU against 64 bits.

The indices have to be the 64-bit ones.  Tolerances: u = 2^-24.  expf is right to 2 ulp (4 u) and its argument l - m, of at
most 32 here, to 32 u; a sum of up to 256 of them takes 13 roundings, the quotients and the factor 3: K u |w|, K = 64.  A
gradient is such a weight times a difference of d and a sum of d's: 2 K u times the sum of the magnitudes.  Results are rounded
once more to their type."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200.moe_router import b200_router_forward, patch_moe_router, router_topk, unpatch_moe_router

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rounding(ref, dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * ref.abs() + (2.0 ** -25 if dtype == FP16 else 0.0)


def check(logits, top_k, sigmoid=False, bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0, seed=0):
    T, E = logits.shape
    leaf = logits.detach().requires_grad_(True)
    w, i = router_topk(leaf, top_k, scoring="sigmoid" if sigmoid else "softmax", bias=bias, num_groups=groups, top_groups=top_groups,
                       renormalize=renormalize, scale=scale)
    assert w.shape == i.shape == (T, top_k) and w.dtype == logits.dtype and i.dtype == torch.int64
    how = dict(sigmoid=sigmoid, renormalize=renormalize, scale=scale)
    ref_w, ref_i = step_fp64.router_topk(logits, top_k, bias=bias, groups=groups, top_groups=top_groups, **how)
    assert torch.equal(i, ref_i), (i[(i != ref_i).any(1)][:4], ref_i[(i != ref_i).any(1)][:4])
    assert bool(((w.double() - ref_w).abs() <= rounding(ref_w, w.dtype) + 64 * U * ref_w.abs()).all())
    d = torch.randn(T, top_k, generator=torch.Generator().manual_seed(seed)).to(device=DEV, dtype=logits.dtype)
    (dl,) = torch.autograd.grad(w, leaf, d)
    ref = step_fp64.router_topk_bwd(logits, ref_i, d, **how)
    s = ref_w.abs() / scale
    a = d.double().abs() * scale
    size = s * (a + (a * s).sum(1, keepdim=True))
    full = torch.zeros_like(ref).scatter(1, ref_i, size)
    if not sigmoid and not renormalize:
        full = full + step_fp64._scores(logits.double(), False) * (a * s).sum(1, keepdim=True)
    assert bool(((dl.double() - ref).abs() <= rounding(ref, dl.dtype) + 128 * U * full).all())
    return w.detach(), i, dl


def make(T, E, dtype, seed=0, coarse=0.0):
    g = torch.Generator().manual_seed(seed + 31 * T + E)
    l = torch.randn(T, E, generator=g) * 2
    if coarse:
        l = (l / coarse).round() * coarse
    return l.to(device=DEV, dtype=dtype)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 32, 4), (3, 4, 4), (33, 31, 2), (1000, 32, 4), (257, 33, 8), (64, 64, 6), (129, 100, 32),
                                   (100, 128, 8), (77, 255, 7), (300, 256, 8), (9, 32, 32)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_sizes_types_and_scores(T, E, k, sigmoid, renormalize):
    for dtype in (BF16, FP16, FP32):
        check(make(T, E, dtype), k, sigmoid=sigmoid, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("T,E,k,groups,top_groups", [(200, 256, 8, 8, 4), (200, 160, 6, 8, 3), (50, 32, 4, 4, 2), (50, 32, 4, 32, 4), (50, 96, 3, 3, 1),
                                                     (40, 35, 5, 5, 5), (40, 35, 5, 7, 1), (20, 31, 2, 31, 2), (60, 256, 32, 2, 1), (10, 8, 2, 1, 1)])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_groups_and_bias(T, E, k, groups, top_groups, sigmoid, with_bias):
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)).mul_(0.1).to(DEV) if with_bias else None
    for dtype in (BF16, FP32):
        for renormalize in (True, False):
            check(make(T, E, dtype, seed=9), k, sigmoid=sigmoid, bias=bias, groups=groups, top_groups=top_groups, renormalize=renormalize)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_equal_values_go_to_the_lowest_index(groups, top_groups, sigmoid):
    l = make(500, 64, BF16, coarse=1.0)
    for bias in (None, torch.zeros(64, device=DEV), torch.randint(0, 2, (64,), generator=torch.Generator().manual_seed(1)).to(device=DEV, dtype=FP32)):
        check(l, 6, sigmoid=sigmoid, bias=bias, groups=groups, top_groups=top_groups)
    check(torch.zeros(7, 64, device=DEV), 5, sigmoid=sigmoid, bias=torch.zeros(64, device=DEV), groups=groups, top_groups=top_groups)
    signed = torch.zeros(7, 64, device=DEV)
    signed[:, ::2] = -0.0                                                             # no value is larger than the other
    check(signed, 5, sigmoid=sigmoid, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_values_that_fp32_cannot_tell_apart(groups, top_groups):
    # every value is 0.75 to 2^-25: the order is in the bits that fp32 sums lose
    l = make(1, 64, FP32, seed=3)
    bias = (0.75 - torch.sigmoid(l[0].double())).float()
    for shift in range(40):
        rolled = l.roll(shift, 1)
        check(torch.cat([rolled, l]), 6, sigmoid=True, bias=bias.roll(shift), groups=groups, top_groups=top_groups)
    soft = (0.5 - torch.softmax(l[0].double(), 0)).float()
    check(l, 6, bias=soft, groups=groups, top_groups=top_groups)


def test_masked_experts():
    inf = float("inf")
    for dtype in (BF16, FP32):
        l = make(400, 32, dtype)
        l[torch.rand(400, 32, generator=torch.Generator().manual_seed(2)).to(DEV) < 0.8] = -inf     # often fewer than 4 are left
        l[5] = -inf
        l[6, :31] = -inf
        bias = torch.linspace(-1, 1, 32, device=DEV)
        for sigmoid in (False, True):
            for renormalize in (False, True):
                for b in (None, bias):
                    for groups, top in ((1, 1), (4, 2)):
                        w, i, dl = check(l, 4, sigmoid=sigmoid, bias=b, groups=groups, top_groups=top, renormalize=renormalize)
                        assert bool((w[5] == 0).all()) and bool((dl[5] == 0).all()) and not bool(torch.isnan(w).any())
                        assert bool((w[torch.isneginf(l.gather(1, i))] == 0).all())


def test_values_that_are_not_numbers_give_a_valid_choice():
    l = make(64, 40, FP32)
    l[3, 7] = float("nan")
    l[4] = float("nan")
    l[5, 9] = float("inf")
    l[6] = float("inf")
    for bias in (None, torch.zeros(40, device=DEV)):
        for groups in (1, 4):
            for scoring in ("softmax", "sigmoid"):
                w, i = router_topk(l, 4, scoring=scoring, bias=bias, num_groups=groups, top_groups=max(1, groups // 2))
                assert bool(((i >= 0) & (i < 40)).all())
                assert bool((i.sort(1).values.diff(dim=1) > 0).all())
                fine = [t for t in range(64) if t not in (3, 4, 5, 6)]
                assert not bool(torch.isnan(w[fine]).any())
    for dtype, bits in ((BF16, -64), (FP32, -4194304)):      # a NaN with its sign bit set is one like any other
        m = make(64, 40, dtype).contiguous()
        m.view(torch.int16 if dtype == BF16 else torch.int32)[2, 11] = bits
        assert bool(torch.isnan(m[2, 11]))
        assert int(router_topk(m, 4)[1][2, 0]) == 11
        assert int(router_topk(m, 4, scoring="sigmoid", num_groups=4, top_groups=2)[1][2, 0]) == 11
        # groups go by scores, and a softmax over a NaN has no score that is a number: the first two groups; in them by logits
        i = router_topk(m, 4, num_groups=4, top_groups=2)[1][2]
        assert int(i[0]) == 11 and bool((i < 20).all())
    w, i = router_topk(l, 4)
    assert int(i[3, 0]) == 7 and i[4].tolist() == [0, 1, 2, 3] and int(i[5, 0]) == 9


def test_strides_no_tokens_and_refusals():
    big = make(40, 80, BF16)
    check(big[:, 5:37], 4)
    check(big[::2, 1:34], 4)
    check(big.t()[:33], 4)                                       # (experts are not the last dimension in memory)
    check(big[:1].expand(9, 80), 4)
    w, i, dl = check(big[:0], 4)
    assert w.shape == (0, 4) and dl.shape == (0, 80)
    half = torch.zeros(80, device=DEV, dtype=BF16)
    check(big, 4, sigmoid=True, bias=half)                       # a bias of another type
    for bad in (dict(top_k=0), dict(top_k=33), dict(top_k=4, num_groups=3), dict(top_k=4, num_groups=4, top_groups=5),
                dict(top_k=21, num_groups=8, top_groups=2), dict(top_k=4, scoring="tanh"), dict(top_k=4, bias=half[:3]),
                dict(top_k=4, bias=half.cpu()), dict(top_k=4, bias=half.long()), dict(top_k=4, num_groups=0), dict(top_k=4, top_groups=0)):
        with pytest.raises(ValueError):
            router_topk(big, **bad)
    for bad in (big[0], big[None]):
        with pytest.raises(ValueError):
            router_topk(bad, 2)
    with pytest.raises(ValueError):
        router_topk(torch.zeros(2, 257, device=DEV), 2)
    with pytest.raises(TypeError):
        router_topk(big.double(), 2)


def test_offsets_past_32_bits():
    T, E = 8_500_000, 256                           # 2.18e9 logits
    l = torch.empty(T, E, device=DEV, dtype=BF16).normal_(generator=torch.Generator(device=DEV).manual_seed(1)).requires_grad_(True)
    w, i = router_topk(l, 8)
    d = torch.ones_like(w)
    d[:, 0] = -1
    (dl,) = torch.autograd.grad(w, l, d)
    for part in (slice(0, 100), slice(T - 100, T), slice(8_388_600, 8_388_700)):
        rows = l.detach()[part]
        ref_w, ref_i = step_fp64.router_topk(rows, 8)
        assert torch.equal(i[part], ref_i)
        assert bool(((w.detach()[part].double() - ref_w).abs() <= rounding(ref_w, BF16) + 64 * U * ref_w.abs()).all())
        ref = step_fp64.router_topk_bwd(rows, ref_i, d[part])
        assert bool(((dl[part].double() - ref).abs() <= rounding(ref, BF16) + 256 * U).all())


def test_a_choice_of_which_only_the_indices_are_used():
    l = make(5, 32, FP32).requires_grad_(True)
    w, i = router_topk(l, 4)
    assert w.requires_grad and not i.requires_grad
    (g,) = torch.autograd.grad(l.gather(1, i).sum(), l)
    assert float(g.sum()) == 20
    w, _ = router_topk(l, 4)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(w.sum(), l, create_graph=True)


def test_results_repeat_and_survive_another_stream_and_a_captured_graph():
    l = make(3000, 256, BF16)
    bias = torch.randn(256, device=DEV) * 0.05
    d = torch.randn(3000, 8, device=DEV).to(BF16)

    def step():
        leaf = l.detach().requires_grad_(True)
        w, i = router_topk(leaf, 8, scoring="sigmoid", bias=bias, num_groups=8, top_groups=4)
        return w.detach(), i, torch.autograd.grad(w, leaf, d)[0]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    l.copy_(l.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), third)) and not torch.equal(third[1], first[1])


def test_the_patched_router_in_front_of_the_experts():
    from transformers import GptOssConfig
    from transformers.models.gpt_oss import modeling_gpt_oss
    from oregon_gpt_oss_patching_b200.moe_experts import moe_experts
    cfg = GptOssConfig(num_local_experts=16, num_experts_per_tok=4, hidden_size=64, intermediate_size=64)
    torch.manual_seed(0)
    mod = modeling_gpt_oss.GptOssTopKRouter(cfg).to(device=DEV, dtype=FP32)
    with torch.no_grad():
        mod.weight.normal_()
        mod.bias.normal_()
    original = modeling_gpt_oss.GptOssTopKRouter.forward
    x = torch.randn(333, 64, device=DEV, requires_grad=True)
    d = torch.randn(333, 4, device=DEV)

    def step():
        logits, scores, indices = mod(x)
        return logits, scores, indices, *torch.autograd.grad(scores, (x, mod.weight, mod.bias), d)

    plain = step()
    patch_moe_router()
    try:
        assert modeling_gpt_oss.GptOssTopKRouter.forward is b200_router_forward
        ours = step()
    finally:
        unpatch_moe_router()
    assert modeling_gpt_oss.GptOssTopKRouter.forward is original
    assert torch.equal(plain[0], ours[0]) and torch.equal(plain[2], ours[2])
    for a, b in zip([t.detach() for t in plain], [t.detach() for t in ours]):
        # fp32 on both sides: the same products of sums of at most 333 terms, from weights right to 64 u
        assert float((a - b).double().norm()) <= 512 * U * float(a.double().norm())
    # what the router gives is what the experts take
    hidden = torch.randn(333, 64, device=DEV).to(BF16)
    w1, b1 = torch.randn(16, 64, 128, device=DEV).to(BF16), torch.randn(16, 128, device=DEV).to(BF16)
    w2, b2 = torch.randn(16, 64, 64, device=DEV).to(BF16), torch.randn(16, 64, device=DEV).to(BF16)
    logits = ours[0].to(BF16).detach().requires_grad_(True)
    w, i = router_topk(logits, 4)
    out = moe_experts(hidden, i, w, w1, b1, w2, b2)
    out.sum().backward()
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(logits.grad).all()) and float(logits.grad.abs().max()) > 0
