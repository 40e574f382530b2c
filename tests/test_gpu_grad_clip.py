"""Gradient norm, clipping and the clipped SGD update on the GPU against 64 bits.

Tolerances.  u = 2^-24.  A thread adds at most 64 fp32 squares of a chunk (8 words of 8) before fp64 takes over: the sum of
non-negative terms is right to 65 u relative, its root to 33 u, and the fp32 result is rounded once: K u, K = 34.  The
coefficient is a sum and a quotient of it (2 u more).  A clipped gradient is one product of it: (K + 3) u and its rounding;
an updated parameter lacks (K + 5) u of lr c |g| and one fp32 rounding of the sum before its own."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step, global_grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rounding(ref, dtype):
    return torch.finfo(dtype).eps / 2 * ref.abs() + (2.0 ** -25 if dtype == FP16 else 0.0)


def make(sizes, seed=0, scale=1.0):
    """Parameters with gradients from (shape, dtype) pairs."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape, dtype in sizes:
        p = torch.nn.Parameter(torch.randn(shape, generator=g).to(device=DEV, dtype=dtype))
        p.grad = (torch.randn(shape, generator=g) * scale).to(device=DEV, dtype=dtype)
        out.append(p)
    return out


def check_clip(params, max_norm):
    before = [p.grad.clone() for p in params if p.grad is not None]
    values = [p.detach().clone() for p in params]
    norm = clip_grad_norm(params, max_norm)
    assert norm.dtype == FP32 and norm.shape == () and norm.is_cuda
    ref = step_fp64.grad_norm(before)
    assert abs(float(norm) - float(ref)) <= 34 * U * float(ref)
    c = step_fp64.clip_coefficient(ref, max_norm)
    for p, b in zip([p for p in params if p.grad is not None], before):
        want = b.double() * c
        tol = rounding(want, b.dtype) * (1 + 2.0 ** -6) + 37 * U * want.abs()
        assert bool(((p.grad.double() - want).abs() <= tol).all())
        if float(ref) * (1 + 64 * U) + 1e-6 < max_norm:
            assert torch.equal(p.grad, b)
    for p, v in zip(params, values):
        assert torch.equal(p.detach(), v)
    return norm


def check_sgd(params, lr, max_norm):
    before = [p.detach().clone() for p in params]
    grads = [p.grad.clone() if p.grad is not None else None for p in params]
    norm = clipped_sgd_step(params, lr, max_norm)
    ref = step_fp64.grad_norm([g for g in grads if g is not None])
    assert abs(float(norm) - float(ref)) <= 34 * U * float(ref)
    c = step_fp64.clip_coefficient(ref, max_norm)
    for p, b, g in zip(params, before, grads):
        if g is None:
            assert torch.equal(p.detach(), b)
            continue
        step = lr * c * g.double()
        want = b.double() - step
        tol = rounding(want, b.dtype) * (1 + 2.0 ** -6) + 39 * U * step.abs() + U * want.abs()
        assert bool(((p.detach().double() - want).abs() <= tol).all())
        assert torch.equal(p.grad, g)
    return norm


SIZES = {
    "one": [((1,), FP32)],
    "one_bf16": [((1,), BF16)],
    "small": [((3,), BF16), ((17, 5), FP32), ((1,), FP16), ((8,), BF16), ((0,), BF16), ((2, 0, 3), FP32), ((255,), FP16)],
    "layer": [((64, 288), BF16), ((64,), FP32), ((4, 288, 576), BF16), ((4, 576), BF16), ((1447, 33), BF16)],
    "chunk_edges": [((16384,), BF16), ((16385,), BF16), ((16383,), BF16), ((8192,), FP32), ((8193,), FP32), ((8191,), FP32)],
    "many": [((n % 97 + 1,), (BF16, FP32, FP16)[n % 3]) for n in range(700)],
    "exactly_a_table": [((5,), FP32)] * 256,
    "long": [((3 * 10 ** 7 + 5,), BF16), ((10 ** 7 + 1,), FP32)],
}


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("max_norm", [0.0, 0.37, 1e6, float("inf")])
def test_clip_and_update_over_sizes_and_types(name, max_norm):
    check_clip(make(SIZES[name]), max_norm)
    check_sgd(make(SIZES[name], seed=1), 0.05, max_norm)


@pytest.mark.parametrize("name", ["one", "small", "many"])
def test_norm_alone(name):
    grads = [p.grad for p in make(SIZES[name])]
    kept = [g.clone() for g in grads]
    ref = float(step_fp64.grad_norm(grads))
    assert abs(float(global_grad_norm(grads)) - ref) <= 34 * U * ref
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    assert float(global_grad_norm(grads[0])) == pytest.approx(float(grads[0].double().norm()), rel=1e-5)
    assert float(global_grad_norm([])) == 0.0 and float(global_grad_norm([torch.zeros(0, device=DEV)])) == 0.0
    twice = global_grad_norm([grads[0], grads[0]])                       # reading the same tensor twice is no error
    assert float(twice) == pytest.approx(2 ** 0.5 * float(grads[0].double().norm()), rel=1e-5)


def test_parameters_without_gradients_and_the_empty_call():
    params = make(SIZES["small"])
    params[1].grad = None
    check_clip(params, 0.5)
    check_sgd(params, 0.1, 0.5)
    for p in params:
        p.grad = None
    assert float(clip_grad_norm(params, 1.0)) == 0.0 and float(clipped_sgd_step(params, 1.0, 1.0)) == 0.0
    assert float(clip_grad_norm([], 1.0)) == 0.0
    p = make(SIZES["one"])[0]
    g = float(p.grad)
    assert float(clip_grad_norm(p, 1e-3)) == pytest.approx(abs(g), rel=1e-6)
    assert float(clip_grad_norm(iter([p]), 1.0)) == pytest.approx(1e-3, rel=1e-2)


def test_offsets_and_orders_in_memory():
    base = torch.randn(4, 3000, device=DEV)
    params = []
    for i, off in enumerate((1, 3, 4, 7)):          # gradients and parameters at every place of the 16-byte grid
        p = torch.nn.Parameter(torch.randn(3000, device=DEV).to(BF16)[8 - off:2000])
        p.grad = base[i].to(BF16)[off:off + p.numel()]
        params.append(p)
    check_clip(params, 0.5)
    check_sgd(params, 0.05, 0.5)
    # transposed, sliced and mixed orders; what lies between the rows of a slice stays as it is
    wide = torch.randn(40, 64, device=DEV)
    kept = wide.clone()
    a = torch.nn.Parameter(torch.randn(40, 24, device=DEV))
    a.grad = wide[:, 8:32]
    b = torch.nn.Parameter(torch.randn(24, 40, device=DEV).t())
    b.grad = torch.randn(40, 24, device=DEV)
    c = torch.nn.Parameter(torch.randn(40, 24, device=DEV))
    c.grad = torch.randn(24, 40, device=DEV).t()
    check_clip([a, b, c], 0.5)
    check_sgd([a, b, c], 0.05, 0.5)
    assert torch.equal(wide[:, :8], kept[:, :8]) and torch.equal(wide[:, 32:], kept[:, 32:])
    # neighbours of a tensor that ends inside a 16-byte word are left alone
    store = torch.ones(64, device=DEV, dtype=BF16)
    d = torch.nn.Parameter(torch.zeros(11, device=DEV, dtype=BF16))
    d.grad = store[5:16]
    clip_grad_norm([d], 0.01)
    assert bool((store[:5] == 1).all()) and bool((store[16:] == 1).all()) and bool((store[5:16] != 1).all())


def test_norms_that_are_not_finite():
    for value, c in ((float("nan"), float("nan")), (float("inf"), 0.0)):
        params = make(SIZES["layer"])
        params[0].grad[3, 5] = value
        kept = [p.grad.clone() for p in params]
        norm = clip_grad_norm(params, 1.0)
        assert str(float(norm)) == str(float(torch.tensor(value)))
        for p, k in zip(params, kept):
            assert torch.equal(torch.isnan(p.grad), torch.isnan(k * c))
            assert bool((p.grad[~torch.isnan(p.grad)] == 0).all())


def test_no_limit_never_scales():
    params = make(SIZES["layer"])
    params[0].grad[3, 5] = float("inf")
    kept = [p.grad.clone() for p in params]
    assert float(clip_grad_norm(params, float("inf"))) == float("inf")
    assert all(torch.equal(p.grad, k) for p, k in zip(params, kept))
    before = [p.detach().clone() for p in params]
    clipped_sgd_step(params, 0.5)
    for p, b, k in list(zip(params, before, kept))[1:]:
        assert bool(torch.isfinite(p).all()) and not torch.equal(p.detach(), b)


def test_offsets_past_32_bits():
    n = 2 ** 31 + 2 ** 20 + 3
    p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=BF16))
    p.grad = torch.ones(n, device=DEV, dtype=BF16)
    p.grad[-1], p.grad[5] = 3.0, -2.0
    norm = clipped_sgd_step([p], 1.0, float("inf"))
    assert float(norm) == pytest.approx((n - 2 + 13) ** 0.5, rel=34 * U)
    assert p[-1] == -3 and p[5] == 2 and p[-2] == -1 and p[2 ** 31] == -1 and float(p.detach().sum(dtype=torch.float64)) == -(n - 2) - 3 + 2
    clip_grad_norm([p], 0.5 * float(norm))
    assert p.grad[-1] == 1.5 and p.grad[5] == -1 and float(p.grad.sum(dtype=torch.float64)) == (n - 2) * 0.5 + 1.5 - 1


def test_zero_and_tiny_gradients():
    params = make(SIZES["layer"], scale=0.0)
    assert float(check_clip(params, 1.0)) == 0.0
    params = make(SIZES["layer"], scale=1e-12)
    check_clip(params, 1.0)
    assert float(clip_grad_norm(make(SIZES["layer"]), 0.0)) > 0


def test_results_repeat_and_survive_another_stream_and_a_captured_graph():
    params = make(SIZES["long"])
    fresh = [p.grad.clone() for p in params]

    def clip():
        for p, f in zip(params, fresh):
            p.grad.copy_(f)
        return clip_grad_norm(params, 0.9), [p.grad.clone() for p in params]

    n0, g0 = clip()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n1, g1 = clip()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(g0, g1))
    graphs = []
    for _ in range(2):      # two graphs of the same gradients, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, *clip()))
    for graph, n, g in graphs + graphs:
        n.zero_()
        graph.replay()
        assert torch.equal(n, n0) and all(torch.equal(a, b) for a, b in zip(g, g0))


def test_updates_are_seen_by_autograd():
    p, = make([((8,), FP32)])
    y = (p * p).sum()
    clipped_sgd_step([p], 0.1, 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_shared_memory_is_refused_before_anything_is_written():
    params = make(SIZES["layer"])
    kept = [p.grad.clone() for p in params]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm(params + [params[0]], 0.1)
    shared = torch.nn.Parameter(torch.zeros(10, device=DEV, dtype=BF16))
    shared.grad = params[0].grad.view(-1)[100:110]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm(params + [shared], 0.1)
    own = torch.nn.Parameter(torch.zeros(10, device=DEV))
    own.grad = own.detach()
    with pytest.raises(RuntimeError, match="share memory"):
        clipped_sgd_step([own], 0.1, 1.0)
    flat = torch.nn.Parameter(torch.zeros(10, 4, device=DEV))
    flat.grad = torch.ones(4, device=DEV).expand(10, 4)
    with pytest.raises(ValueError, match="stride of 0"):
        clip_grad_norm(params + [flat], 0.1)
    assert all(torch.equal(p.grad, k) for p, k in zip(params, kept))
    check_sgd([flat], 0.1, 1.0)       # read only: a broadcast gradient is fine
