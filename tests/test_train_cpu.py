"""The training-step entry points without a GPU: the ABI is exported and refuses bad arguments, the Python side refuses bad tensors."""
import os
import re

import pytest
import torch

from oregon_gpt_oss_patching_b200 import _cabi, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _cabi.load()


def test_every_declared_symbol_is_exported(lib):
    header = open(os.path.join(ROOT, "include", "b200train.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    declared = set(re.findall(r"\b(b200train_[a-z_0-9]+)\s*\(", header))
    assert declared == set(_cabi.TRAIN_EXPORTS)
    for name in declared:
        assert hasattr(lib, name), name
    enum = dict(re.findall(r"(B200TRAIN_(?:BF16|FP16|FP32)) = (\d)", header))
    assert {int(enum["B200TRAIN_BF16"]), int(enum["B200TRAIN_FP16"]), int(enum["B200TRAIN_FP32"])} == {0, 1, 2}
    assert _cabi.TRAIN_DTYPES[torch.bfloat16] == int(enum["B200TRAIN_BF16"])
    assert _cabi.TRAIN_DTYPES[torch.float16] == int(enum["B200TRAIN_FP16"])
    assert _cabi.TRAIN_DTYPES[torch.float32] == int(enum["B200TRAIN_FP32"])


def test_norm_arguments_are_validated(lib):
    buf = torch.zeros(1 << 12, dtype=torch.float32)
    p = buf.data_ptr()

    def fwd(x=p, xs=64, r=None, rs=0, w=p, y=p, h=None, rows=2, cols=64, dtype=0, wdtype=0, eps=1e-5):
        return lib.b200train_add_rms_norm(x, xs, r, rs, w, y, h, rows, cols, eps, dtype, wdtype, 0, None)

    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1
    assert fwd(rows=-1) == -1 and fwd(cols=0) == -1 and fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1
    assert fwd(dtype=3) == -1 and fwd(dtype=-1) == -1 and fwd(dtype=0, wdtype=1) == -1 and fwd(dtype=2, wdtype=0) == -1
    assert fwd(r=p, rs=64) == -1 and fwd(h=p) == -1                       # a residual and its sum come together
    assert fwd(cols=16385, xs=16385) == -2
    assert fwd(rows=1 << 40) == -2
    assert fwd(x=p + 2) == -4 and fwd(w=p + 4) == -4 and fwd(xs=60) == -4 and fwd(xs=-64) == -4
    assert fwd(cols=63, xs=64) == -4                                      # rows off the 16-byte grid must be contiguous
    assert fwd(r=p, rs=65, h=p) == -4

    def bwd(dy=p, dys=64, dh=None, h=p, w=p, dx=p, dw=None, rows=2, cols=64, dtype=0, wdtype=0):
        return lib.b200train_add_rms_norm_bwd(dy, dys, dh, 64, h, 64, w, dx, dw, None, 0, rows, cols, 1e-5, dtype, wdtype, 0, None)

    assert bwd(dy=None) == -1 and bwd(h=None) == -1 and bwd(dx=None) == -1 and bwd(w=None) == -1 and bwd(wdtype=1) == -1
    assert bwd(dys=12) == -4 and bwd(dh=p + 2) == -4 and bwd(cols=20000) == -2
    assert lib.b200train_norm_scratch_floats(0, 64, 0, 0) == 0
    assert lib.b200train_norm_scratch_floats(4, 64, 7, 0) == 0
    assert lib.b200train_norm_scratch_floats(10, 64, 0, 0) >= 64
    if not torch.cuda.is_available():
        assert fwd() in (-5, -6) and bwd() in (-5, -6)                    # no sm_100 device


def test_norm_refuses_bad_tensors():
    from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        rms_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        add_rms_norm(x, x, torch.ones(8))
    if not torch.cuda.is_available():
        return
    x = x.cuda()
    w = torch.ones(8, device="cuda")
    for bad in (lambda: rms_norm(x.double(), w), lambda: rms_norm(x, w.half()), lambda: rms_norm(x.int(), w)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: rms_norm(x, w[:7]), lambda: add_rms_norm(x, x[:2], w), lambda: add_rms_norm(x, x.half(), w),
                lambda: rms_norm(x, w, -1.0), lambda: rms_norm(x, w, float("nan")), lambda: rms_norm(x.sum(), w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="code -2"):
        rms_norm(torch.zeros(2, 16392, device="cuda"), torch.ones(16392, device="cuda"))


def test_clip_arguments_are_validated(lib):
    import array
    import ctypes
    buf = torch.zeros(1 << 8, dtype=torch.float32)
    p = buf.data_ptr()
    norm = ctypes.c_float(7.0)

    def call(kind="clip", grads=(p,), params=(p + 512,), counts=(16,), dtypes=(2,), max_norm=1.0, scratch=p, doubles=1 << 30, out=None, n=None):
        keep = [array.array(c, v) for c, v in (("q", grads), ("q", params), ("q", counts), ("i", dtypes))]
        host = [a.buffer_info()[0] for a in keep]
        n = len(grads) if n is None else n
        out = ctypes.addressof(norm) if out is None else out
        tail = (scratch, doubles, out, 0, None)
        if kind == "norm":
            return lib.b200train_grad_norm(host[0], host[2], host[3], n, *tail)
        if kind == "clip":
            return lib.b200train_clip_grads(host[0], host[2], host[3], n, max_norm, *tail)
        return lib.b200train_clipped_sgd(host[0], host[1], host[2], host[3], n, 0.1, max_norm, *tail)

    for kind in ("norm", "clip", "sgd"):
        assert call(kind, out=0) == -1 and call(kind, n=-1) == -1
        assert call(kind, dtypes=(3,)) == -1 and call(kind, dtypes=(-1,)) == -1 and call(kind, counts=(-1,)) == -1
        assert call(kind, grads=(0,)) == -1 and call(kind, grads=(p + 2,)) == -4
        assert call(kind, counts=(1 << 44,)) == -2
        assert call(kind, grads=(p, p + 1024), params=(p + 2048, p + 4096), counts=(1 << 42, (1 << 42) + 1), dtypes=(2, 2)) == -2
        if not torch.cuda.is_available():
            assert call(kind) in (-5, -6)
    for kind in ("clip", "sgd"):
        assert call(kind, max_norm=-1.0) == -1 and call(kind, max_norm=float("nan")) == -1
        assert call(kind, grads=(p, p + 60), params=(p + 512, p + 640), counts=(16, 16), dtypes=(2, 2)) == -10
    assert call("sgd", params=(0,)) == -1 and call("sgd", params=(p + 513,)) == -4
    assert call("sgd", params=(p + 32,)) == -10                            # a parameter on its own gradient
    assert lib.b200train_clip_scratch_doubles(-1, 0) == 0
    assert lib.b200train_clip_scratch_doubles(257, 0) == 2 * lib.b200train_clip_scratch_doubles(0, 0)
    assert "share memory" in _cabi.strerror(-10)


def test_clip_refuses_bad_tensors():
    from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step, global_grad_norm
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    for call in (lambda: clip_grad_norm([p], 1.0), lambda: clipped_sgd_step([p], 0.1, 1.0), lambda: global_grad_norm([p])):
        with pytest.raises(RuntimeError, match="needs CUDA tensors"):
            call()
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm([p], bad)
        with pytest.raises(ValueError, match="max_norm"):
            clipped_sgd_step([p], 0.1, bad)
    if not torch.cuda.is_available():
        return
    q = torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))
    q.grad = torch.zeros_like(q)
    with pytest.raises(TypeError):
        clip_grad_norm([q], 1.0)
    with pytest.raises(RuntimeError):
        global_grad_norm([p, q])


def test_router_arguments_are_validated(lib):
    buf = torch.zeros(1 << 10, dtype=torch.float32)
    p = buf.data_ptr()

    def fwd(l=p, stride=32, bias=None, w=p, i=p, T=2, E=32, k=4, groups=1, top=1, dtype=0):
        return lib.b200moe_router_topk(l, stride, bias, w, i, T, E, k, groups, top, 0, 1, 1.0, dtype, 0, None)

    def bwd(l=p, i=p, dw=p, dl=p, T=2, E=32, k=4, dtype=0):
        return lib.b200moe_router_topk_bwd(l, 32, i, dw, dl, T, E, k, 0, 1, 1.0, dtype, 0, None)

    assert fwd(l=None) == -1 and fwd(w=None) == -1 and fwd(i=None) == -1 and fwd(T=-1) == -1 and fwd(E=0) == -1 and fwd(k=0) == -1
    assert fwd(dtype=3) == -1 and fwd(groups=0) == -1 and fwd(top=0) == -1
    assert fwd(E=257) == -2 and fwd(k=33) == -2 and fwd(E=8, k=9) == -2 and fwd(stride=-1) == -2
    assert fwd(groups=5) == -2 and fwd(groups=4, top=5) == -2 and fwd(E=256, groups=64) == -2 and fwd(groups=8, k=5, top=1) == -2
    assert fwd(l=p + 1) == -4 and fwd(l=p + 2, dtype=2) == -4
    assert bwd(l=None) == -1 and bwd(i=None) == -1 and bwd(dw=None) == -1 and bwd(dl=None) == -1 and bwd(dtype=-1) == -1
    assert bwd(E=300) == -2 and bwd(E=3) == -2
    if not torch.cuda.is_available():
        assert fwd() in (-5, -6) and bwd() in (-5, -6)


def test_router_refuses_cpu_tensors():
    from oregon_gpt_oss_patching_b200.moe_router import router_topk
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):
        router_topk(torch.zeros(3, 8), 2)
