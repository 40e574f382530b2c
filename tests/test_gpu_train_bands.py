"""Nothing is written outside a tensor, and nothing outside it counts: every buffer of the training-step entry points lies inside a
larger one filled with NaN, through the C ABI; results are those of the same call on buffers of their own, and the bands stay
as they were."""
from array import array

import pytest
import torch

from oregon_gpt_oss_patching_b200 import _cabi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BAND = 64   # elements before and behind, a multiple of 16 bytes' worth
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class Banded:
    """A tensor inside a band of NaN (or of a pattern, for integers)."""

    def __init__(self, shape, dtype, fill=None, band=BAND):
        n = 1
        for s in shape:
            n *= s
        self.band = band
        self.pattern = float("nan") if dtype.is_floating_point else -7
        self.buffer = torch.full((n + 2 * band,), self.pattern, dtype=dtype, device=DEV)
        self.t = self.buffer[band:band + n].view(shape)
        if fill is not None:
            self.t.copy_(fill)

    def untouched(self):
        bands = torch.cat([self.buffer[:self.band], self.buffer[-self.band:]])
        return bool(torch.isnan(bands).all()) if self.buffer.dtype.is_floating_point else bool((bands == self.pattern).all())

    @property
    def p(self):
        return self.t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 2880), (37, 33), (200, 2881), (1500, 71), (700, 96), (3, 16376), (160, 16384)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_norm(rows, cols, dtype):
    lib = _cabi.load()
    g = torch.Generator().manual_seed(rows + cols)
    vals = [torch.randn(rows, cols, generator=g).to(DEV) for _ in range(4)]
    weight = torch.randn(cols, generator=g).to(DEV)
    code = TYPES[dtype]
    results = []
    for residual in (True, False):
        for banded in (True, False):
            make = (lambda v: Banded(v.shape, dtype, v)) if banded else (lambda v: Banded(v.shape, dtype, v, band=0))
            x, r, dy, dh = (make(v) for v in vals)
            w = Banded(weight.shape, torch.float32, weight) if banded else Banded(weight.shape, torch.float32, weight, band=0)
            y, h, dx = (Banded((rows, cols), dtype) for _ in range(3))
            dw = Banded((cols,), torch.float32)
            floats = lib.b200train_norm_scratch_floats(rows, cols, code, 0)
            scratch = Banded((floats,), torch.float32)
            _cabi.check(lib.b200train_add_rms_norm(x.p, cols, r.p if residual else None, cols, w.p, y.p, h.p if residual else None, rows, cols, 1e-5,
                                                   code, 2, 0, stream()), "fwd")
            kept = h if residual else x
            _cabi.check(lib.b200train_add_rms_norm_bwd(dy.p, cols, dh.p if residual else None, cols, kept.p, cols, w.p, dx.p, dw.p, scratch.p,
                                                       floats, rows, cols, 1e-5, code, 2, 0, stream()), "bwd")
            torch.cuda.synchronize()
            for name, b in (("y", y), ("h", h), ("dx", dx), ("dw", dw), ("scratch", scratch)):
                assert b.untouched(), name
            if banded:
                for b in (x, r, dy, dh, w):
                    assert b.untouched()
            assert not bool(torch.isnan(y.t).any() | torch.isnan(dx.t).any() | torch.isnan(dw.t).any())
            results.append((y.t.clone(), dx.t.clone(), dw.t.clone()))
        assert all(torch.equal(a, b) for a, b in zip(results[-2], results[-1]))
    # a scratch that is too small is refused
    if rows * cols:
        assert lib.b200train_add_rms_norm_bwd(vals[0].data_ptr(), cols, None, 0, vals[0].data_ptr(), cols, weight.data_ptr(), dx.p, dw.p, scratch.p, 0,
                                              rows, cols, 1e-5, code, 2, 0, stream()) == (-4 if vals[0].data_ptr() % 16 else -8)


@pytest.mark.parametrize("T,E,k,groups", [(1, 1, 1, 1), (5, 31, 4, 1), (33, 32, 4, 4), (31, 100, 8, 4), (9, 255, 8, 5), (13, 256, 32, 8), (70, 256, 8, 8)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_router(T, E, k, groups, dtype):
    lib = _cabi.load()
    l = Banded((T, E), dtype, (torch.randn(T, E, generator=torch.Generator().manual_seed(T + E)) * 2).round().to(DEV))    # with ties: the slow election as well
    b = Banded((E,), torch.float32, torch.randn(E, generator=torch.Generator().manual_seed(E)).mul(0.1).to(DEV))
    d = Banded((T, k), dtype, torch.randn(T, k, generator=torch.Generator().manual_seed(k)).to(DEV))
    for bias in (None, b):
        for sigmoid in (0, 1):
            for renormalize in (0, 1):
                w, i, dl = Banded((T, k), dtype), Banded((T, k), torch.int64), Banded((T, E), dtype)
                _cabi.check(lib.b200moe_router_topk(l.p, E, None if bias is None else bias.p, w.p, i.p, T, E, k, groups, groups, sigmoid, renormalize,
                                                    1.0, TYPES[dtype], 0, stream()), "fwd")
                _cabi.check(lib.b200moe_router_topk_bwd(l.p, E, i.p, d.p, dl.p, T, E, k, sigmoid, renormalize, 1.0, TYPES[dtype], 0, stream()), "bwd")
                torch.cuda.synchronize()
                assert w.untouched() and i.untouched() and dl.untouched() and l.untouched() and b.untouched() and d.untouched()
                assert not bool(torch.isnan(w.t).any() | torch.isnan(dl.t).any())
                assert bool(((i.t >= 0) & (i.t < E)).all()) and bool((i.t.sort(1).values.diff(dim=1) > 0).all())


@pytest.mark.parametrize("n", [1, 7, 8, 9, 4095, 16384, 16385, 200_003])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_clip(n, dtype):
    lib = _cabi.load()
    for shift in (0, 1, 3):
        g = Banded((n,), dtype, torch.ones(n, device=DEV), band=BAND + shift)
        p = Banded((n,), dtype, torch.ones(n, device=DEV), band=BAND + 2 * shift)
        doubles = lib.b200train_clip_scratch_doubles(1, 0)
        scratch, norm = Banded((doubles,), torch.float64), Banded((1,), torch.float32)
        arrays = [array("q", [v]) for v in (g.p, p.p, n)] + [array("i", [TYPES[dtype]])]
        ga, pa, ca, da = (a.buffer_info()[0] for a in arrays)
        tail = (scratch.p, doubles, norm.p, 0, stream())
        _cabi.check(lib.b200train_clipped_sgd(ga, pa, ca, da, 1, 0.5, 1e9, *tail), "sgd")
        torch.cuda.synchronize()
        assert g.untouched() and p.untouched() and scratch.untouched() and norm.untouched()
        assert bool((p.t == 0.5).all()) and bool((g.t == 1).all()) and float(norm.t) == pytest.approx(n ** 0.5, rel=1e-5)
        _cabi.check(lib.b200train_clip_grads(ga, ca, da, 1, 0.5 * float(norm.t), *tail), "clip")
        _cabi.check(lib.b200train_grad_norm(ga, ca, da, 1, *tail), "norm")
        torch.cuda.synchronize()
        assert g.untouched() and norm.untouched() and float(norm.t) == pytest.approx(0.5 * n ** 0.5, rel=1e-2)
        assert lib.b200train_grad_norm(ga, ca, da, 1, scratch.p, 0, norm.p, 0, stream()) == -8
