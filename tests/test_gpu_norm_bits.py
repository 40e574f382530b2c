"""The global norm's sum does not depend on the sizes of its terms: fp32 within 16 bytes of a tensor, fp64 above.

Tolerance.  u = 2^-24.  The squares of 16 bytes are added in three roundings: two additions of four fp32 squares that are rounded
themselves, or three of eight 16-bit elements' squares, which fp32 holds.  So the sum is right to 3 u, its root to 1.5 u, and the
result is rounded once (u): 2.5 u.  What fp64 loses in 10^7 additions stays below u / 100."""
import pytest
import torch

from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, global_grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [8, 63, 1000, 16384, 100_003, 2_000_000])
@pytest.mark.parametrize("large", [1, 2, 8])
def test_small_squares_next_to_large_ones_count(dtype, n, large):
    # the squares of the small ones are a little below half a step of the large ones'
    t = torch.full((n,), 0.9 * 2.0 ** -12, device=DEV, dtype=dtype)
    for first in range(0, n, 4096):
        t[first:first + large] = 1.0
    ref = float((t.double() ** 2).sum().sqrt())
    for shift in (0, 1):                                        # on the 16-byte grid, and beside it
        at = torch.empty(n + shift, device=DEV, dtype=dtype)[shift:].copy_(t)
        assert abs(float(global_grad_norm([at])) - ref) <= 2.51 * U * ref
        p = torch.nn.Parameter(torch.zeros_like(at))
        p.grad = at
        assert abs(float(clip_grad_norm([p], 1e9)) - ref) <= 2.51 * U * ref


def test_zeros_subnormals_and_what_is_not_finite():
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        z = torch.zeros(20_000, device=DEV, dtype=dtype)
        assert float(global_grad_norm([z])) == 0.0
        z[7] = float("inf")
        assert float(global_grad_norm([z])) == float("inf")
        z[9] = float("nan")
        assert float(global_grad_norm([z])) != float(global_grad_norm([z]))
    tiny = torch.full((20_000,), 2.0 ** -70, device=DEV)          # squares of 2^-140 are subnormal in fp32, and exact
    assert float(global_grad_norm([tiny])) == pytest.approx(2.0 ** -70 * 20_000 ** 0.5, rel=2.51 * U)
    over = torch.full((4,), 2e19, device=DEV)                      # a square past fp32
    assert float(global_grad_norm([over])) == float("inf")
