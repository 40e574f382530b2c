"""The residual sum with its RMS norm (`b200train_add_rms_norm`, `_bwd`) on the GPU against the formula in 64 bits.

Tolerances.  u = 2^-24.  A row's statistic is a sum of squares over at most 32 terms a thread and 10 shuffle steps: its
relative error is below 45 u, its root's below 23 u plus 2 ulp of rsqrt; with the two products y's error before rounding is
below K u |y|, K = 64.  dx is a sum of dh, rstd g and rstd n c with the same statistic and a second sum like it: K u times
the sum of the magnitudes, K = 128.  dw adds `rows` terms: (rows + K) u times the sum of magnitudes.  Every result is
rounded once more to its type: finfo.eps / 2 relative, plus half the smallest subnormal (fp16)."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, patch_rms_norm, rms_norm, unpatch_rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rounding(ref, dtype):
    half = torch.finfo(dtype).eps / 2 if dtype != FP32 else U
    return half * ref.abs() + (2.0 ** -25 if dtype == FP16 else 0.0)


def within(got, ref, slack, dtype):
    assert got.dtype == dtype
    err = (got.double() - ref).abs()
    tol = rounding(ref, dtype) * (1 + 2.0 ** -6) + slack
    bad = err > tol
    assert not bool(bad.any()), (float((err - tol).max()), int(bad.sum()))


def check(x, r, w, dy, dh, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, r, w)]
    y, h = add_rms_norm(leaves[0], leaves[1], leaves[2], eps)
    outs, grads = ([y, h], [dy, dh]) if dh is not None else ([y], [dy])
    wanted = [t for t in leaves if t is not None]
    got = torch.autograd.grad(outs, wanted, grads)
    ref_y, ref_h = step_fp64.add_rms_norm(x, r, w, eps)
    assert torch.equal(h.double(), ref_h)
    within(y, ref_y, 64 * U * ref_y.abs(), x.dtype)
    dx, dw = step_fp64.add_rms_norm_bwd(ref_h, w, dy, dh, eps)
    rstd = 1 / torch.sqrt((ref_h * ref_h).mean(-1, keepdim=True) + eps)
    n, g = ref_h * rstd, dy.double() * w.double()
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + (0 if dh is None else dh.double().abs())
    within(got[0], dx, 128 * U * size, x.dtype)
    if r is not None:
        assert torch.equal(got[1], got[0])
    cols = x.shape[-1]
    rows = x.numel() // cols
    within(got[-1], dw, (rows + 128) * U * (dy.double() * n).abs().reshape(-1, cols).sum(0), w.dtype)
    return y, h, got


def make(rows, cols, dtype, wdtype, seed=0, residual=True, lead=None):
    g = torch.Generator().manual_seed(seed + rows * 131 + cols)
    shape = (lead or (rows,)) + (cols,)
    t = [torch.randn(*shape, generator=g).to(device=DEV, dtype=dtype) for _ in range(4)]
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(device=DEV, dtype=wdtype)
    return t[0], (3 * t[1] if residual else None), w, t[2], (t[3] if residual else None)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2880), (4, 2880), (3, 7), (17, 64), (300, 2880), (299, 2881), (1000, 96), (777, 1447),
                                       (2500, 33), (40, 8192), (33, 8191), (5, 16376), (400, 16384), (700, 1024), (1201, 520)])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, FP32), (FP16, FP32), (FP32, FP32), (FP16, FP16)])
def test_sizes_and_types(rows, cols, dtype, wdtype):
    check(*make(rows, cols, dtype, wdtype))


@pytest.mark.parametrize("rows", [2, 700])
def test_without_a_residual_and_with_the_stream_passed_through(rows):
    x, _, w, dy, _ = make(rows, 2880, BF16, FP32, residual=False)
    check(x, None, w, dy, None)
    dh = torch.randn_like(dy)
    y, h, _ = check(x, None, w, dy, dh)
    assert h.data_ptr() == x.data_ptr()
    leaf = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(rms_norm(leaf, w), leaf, dy)
    assert torch.equal(dx, check(x, None, w, dy, None)[2][0])


def test_leading_shapes_strides_and_alignment():
    x, r, w, dy, dh = make(24, 2880, BF16, BF16, lead=(2, 3, 4))
    check(x, r, w, dy, dh)
    check(x[0, 0, 0], r[0, 0, 0], w, dy[0, 0, 0], dh[0, 0, 0])                       # a single vector
    big = torch.randn(30, 2880 + 64, device=DEV).to(BF16)
    check(big[:, 8:2888], big[:, 64:2944], w, big[:, :2880], big[:, 16:2896])        # strided rows
    check(big[:, 3:2883], big[:, 5:2885], w, big[:, 1:2881], big[:, 7:2887])         # rows off the 16-byte grid
    odd = torch.randn(30, 1448, device=DEV).to(BF16)
    w_odd = torch.randn(1448, device=DEV).to(BF16)[1:]                               # a weight off the grid too
    check(odd[:, 1:], odd[:, :-1], w_odd, odd[:, 1:], odd[:, :-1])
    flat = torch.randn(30 * 2880 + 1, device=DEV).to(BF16)[1:].view(30, 2880)
    check(flat, flat, w, flat, flat)
    t = torch.randn(2880, 30, device=DEV).to(BF16).t()
    check(t, t, w, t, t)
    same = torch.randn(1, 2880, device=DEV).to(BF16).expand(9, 2880)                 # one row for all, as a broadcast has it
    check(same, same, w, same, same)
    ones = torch.ones((), device=DEV, dtype=BF16).expand(9, 2880)                    # the gradient of a sum
    check(same, same, w, ones, ones)


def test_no_rows():
    x, r, w, dy, dh = make(0, 2880, BF16, BF16)
    _, _, got = check(x, r, w, dy, dh)
    assert got[0].shape == (0, 2880) and bool((got[-1] == 0).all())


def test_rows_of_zeros_and_large_values():
    x, r, w, dy, dh = make(6, 2880, BF16, FP32)
    x[0], r[0] = 0, 0
    x[1], r[1] = 1e15, 1e15
    x[2], r[2] = 1e-15, 0
    check(x, r, w, dy, dh)
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    y, h = add_rms_norm(x, r, w)
    ref_y, _ = step_fp64.add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(torch.isnan(y), torch.isnan(ref_y)) and not bool(torch.isnan(y[[0, 1, 2, 5]]).any())
    assert bool((y[3].isnan() | (y[3] == 0)).all()) and bool(y[4].isnan().all())


def test_only_the_wanted_gradients():
    x, r, w, dy, dh = make(300, 2880, BF16, BF16)
    full = check(x, r, w, dy, dh)[2]
    for wants in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        leaves = [t.detach().requires_grad_(q) for t, q in zip((x, r, w), wants)]
        y, h = add_rms_norm(*leaves)
        got = torch.autograd.grad((y, h), [t for t in leaves if t.requires_grad], (dy, dh))
        for a, b in zip(got, [t for t, q in zip(full, wants) if q]):
            assert torch.equal(a, b)
    # only the stream is used, only the norm is used
    leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
    y, h = add_rms_norm(*leaves)
    dx, dr, dw = torch.autograd.grad(h, leaves, dh, allow_unused=True)
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and dw is None
    check(x, r, w, dy, None)


def test_results_repeat_and_survive_another_stream_and_a_captured_graph():
    x, r, w, dy, dh = make(2000, 2880, BF16, BF16)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, h = add_rms_norm(*leaves)
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh))]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.cuda.graph(graph):
        third = step()
    x.mul_(2)
    graph.replay()
    after = step()
    assert all(torch.equal(a, b) for a, b in zip(after, third)) and not torch.equal(after[0], first[0])


def test_a_module_s_weight_of_another_type():
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssRMSNorm
    from oregon_gpt_oss_patching_b200.rms_norm import b200_rms_norm_forward
    mod = GptOssRMSNorm(96, eps=1e-5).to(device=DEV, dtype=BF16)
    x = torch.randn(5, 96, device=DEV)
    ref, _ = step_fp64.add_rms_norm(x, None, mod.weight.detach(), 1e-5)
    y = b200_rms_norm_forward(mod, x)
    within(y.detach(), ref, 64 * U * ref.abs(), FP32)
    y.sum().backward()
    assert mod.weight.grad.dtype == BF16


def test_what_is_changed_between_the_passes_is_noticed():
    x, r, w, dy, dh = make(7, 2880, BF16, BF16)
    for change in (lambda y, h: h.add_(1), lambda y, h: w.add_(1)):
        leaves = [t.detach().requires_grad_(True) for t in (x, r)] + [w.requires_grad_(True)]
        y, h = add_rms_norm(*leaves)
        with torch.no_grad():
            change(y, h)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)
    w.requires_grad_(False)
    leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
    y, h = add_rms_norm(*leaves)
    once = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    again = torch.autograd.grad((y, h), leaves, (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    y, h = add_rms_norm(*leaves)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad((y, h), leaves, (dy, dh), create_graph=True)


def test_offsets_past_32_bits():
    rows, cols = 760_000, 2880                      # 2.19e9 elements
    x = torch.empty(rows, cols, device=DEV, dtype=BF16).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w = (1 + 0.1 * torch.randn(cols, device=DEV)).to(BF16)
    leaf = x.requires_grad_(True)
    y = rms_norm(leaf, w)
    (dx,) = torch.autograd.grad(y, leaf, x.detach())
    for part in (slice(0, 3), slice(rows - 3, rows), slice(745_600, 745_700)):
        rows_of = x.detach()[part]
        ref, h = step_fp64.add_rms_norm(rows_of, None, w, 1e-5)
        within(y.detach()[part], ref, 64 * U * ref.abs(), BF16)
        ref_dx, _ = step_fp64.add_rms_norm_bwd(h, w, rows_of, None, 1e-5)
        n = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
        g = h * w.double()
        size = (n / h).abs().nan_to_num() * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
        within(dx[part], ref_dx, 128 * U * size, BF16)


def test_the_patched_layer_gives_the_model_s_results():
    from transformers import GptOssConfig
    from transformers.models.gpt_oss import modeling_gpt_oss
    originals = modeling_gpt_oss.GptOssRMSNorm.forward, modeling_gpt_oss.GptOssDecoderLayer.forward
    cfg = GptOssConfig(num_hidden_layers=2, hidden_size=128, intermediate_size=64, num_local_experts=4, num_experts_per_tok=2, vocab_size=64,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=64, layer_types=["sliding_attention", "full_attention"],
                       use_cache=False)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    with torch.device(DEV):
        model = modeling_gpt_oss.GptOssForCausalLM(cfg).float()
    ids = torch.randint(0, 64, (2, 33), device=DEV)

    def step():
        model.zero_grad(set_to_none=True)
        loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}

    loss0, grads0 = step()
    patch_rms_norm()
    try:
        loss1, grads1 = step()
    finally:
        unpatch_rms_norm()
    assert (modeling_gpt_oss.GptOssRMSNorm.forward, modeling_gpt_oss.GptOssDecoderLayer.forward) == originals
    # an fp32 model of two layers: both sides round every one of some dozens of chained steps at 2^-24 (products of
    # 128 terms among them), so 2^-24 * 128 * 32 bounds the relative distance of a gradient's norm
    assert abs(float(loss1 - loss0)) <= 2.0 ** -12 * abs(float(loss0))
    assert grads0.keys() == grads1.keys()
    for name, a in grads0.items():
        assert float((grads1[name] - a).norm()) <= 2.0 ** -12 * float(a.norm()) + 1e-9, name
