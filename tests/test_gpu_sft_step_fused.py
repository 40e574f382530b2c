"""The fine-tuning step with every part of it on this library's kernels: attention, rotary embedding, experts, norms, router, clip
and update in one run, as a user would start it, next to the same step with transformers' norms and router and torch's clip."""
import json
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TINY = ["--layers", "2", "--experts", "4", "--vocab", "512", "--seq", "512", "--steps", "2", "--warmup", "0"]


def _run(extra):
    env = dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    proc = subprocess.run([sys.executable, "-m", "oregon_gpt_oss_patching_b200.sft_step", *TINY, *extra],
                          cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    assert proc.returncode == 0, proc.stderr[-3000:]
    lines = [ln for ln in proc.stdout.splitlines() if ln.startswith("{")]
    assert len(lines) == 1, proc.stdout[-2000:]
    return json.loads(lines[0])


def test_the_step_with_norms_router_and_clip_runs():
    fused = _run(["--norm", "b200", "--router", "b200", "--max-grad-norm", "1.0"])
    assert (fused["norm"], fused["router"], fused["max_grad_norm"], fused["kernel_status"]) == ("b200", "b200", 1.0, 0)
    assert fused["loss"] == fused["loss"] and fused["grad_norm"] > 0
    plain = _run(["--max-grad-norm", "1.0"])
    assert (plain["norm"], plain["router"]) == ("hf", "hf") and plain["grad_norm"] > 0
    assert _run([])["grad_norm"] is None


def _model(layers=2):
    from oregon_gpt_oss_patching_b200.sft_step import build_model
    return build_model(layers, 4, 512, "cuda:0")[0]


def _gradients(model, ids):
    model.zero_grad(set_to_none=True)
    model(input_ids=ids, labels=ids, use_cache=False).loss.backward()
    return {n: p.grad.float().clone() for n, p in model.named_parameters() if p.grad is not None}


def test_gradients_of_the_fused_step_are_the_model_s():
    """Norms and router patched on top of attention and experts, against transformers' own: both bf16 models, compared with the
    same step in fp32, where a patched model may be off by as much as the unpatched one and half as much again (each rounds
    activations at the same places or fewer)."""
    from oregon_gpt_oss_patching_b200 import moe_router, rms_norm
    model = _model()
    ids = torch.randint(0, 512, (1, 300), generator=torch.Generator().manual_seed(1)).cuda()
    plain = _gradients(model, ids)
    rms_norm.patch_rms_norm()
    moe_router.patch_moe_router()
    try:
        fused = _gradients(model, ids)
    finally:
        rms_norm.unpatch_rms_norm()
        moe_router.unpatch_moe_router()
    exact = _gradients(model.float(), ids)
    assert fused.keys() == plain.keys() == exact.keys()
    for name, ref in exact.items():
        if not float(ref.norm()):
            continue
        off = float((plain[name] - ref).norm() / ref.norm())
        assert float((fused[name] - ref).norm() / ref.norm()) <= 1.5 * off + 2.0 ** -7, (name, off)


def test_nothing_is_kept_after_a_step():
    """Forward alone, forward and backward, clip and update: when their tensors are dropped, the device's memory is as it was."""
    import gc
    from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step
    from oregon_gpt_oss_patching_b200.moe_router import router_topk
    from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm
    x, r = (torch.randn(2000, 2880, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    w = torch.nn.Parameter(torch.ones(2880, device="cuda", dtype=torch.bfloat16))
    logits = torch.randn(2000, 32, device="cuda", requires_grad=True)

    def step(backward):
        y, h = add_rms_norm(x, r, w)
        z, same = add_rms_norm(y, None, w)
        t, _ = router_topk(logits, 4)
        if backward:
            (rms_norm(z, w).sum() + (h + same).sum() + t.sum()).backward()
            clip_grad_norm([w, x, r, logits], 1.0)
            clipped_sgd_step([w], 0.0, 1.0)
            for p in (w, x, r, logits):
                p.grad = None

    step(True)
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    gc.disable()           # (cycles would have to wait for the collector)
    try:
        for backward in (False, True, False, True):
            step(backward)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


def test_threads_and_streams_at_once():
    """Four threads, each on a stream of its own, run all operators on their own tensors: the same results as one after the other."""
    import threading
    from oregon_gpt_oss_patching_b200.grad_clip import clipped_sgd_step
    from oregon_gpt_oss_patching_b200.moe_router import router_topk
    from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm

    def work(seed, out):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            g = torch.Generator(device="cuda").manual_seed(seed)
            x, r, dy, dh = (torch.randn(500, 2880, device="cuda", generator=g).bfloat16() for _ in range(4))
            w = torch.nn.Parameter(torch.ones(2880, device="cuda", dtype=torch.bfloat16))
            logits = torch.randn(500, 64, device="cuda", generator=g)
            for _ in range(10):
                x.requires_grad_(True)
                y, h = add_rms_norm(x, r, w)
                gx, w.grad = torch.autograd.grad((y, h), (x, w), (dy, dh))
                norm = clipped_sgd_step([w], 0.1, 1.0)
                t, i = router_topk(logits, 6, scoring="sigmoid", bias=logits[0], num_groups=4, top_groups=2)
                x = (x + gx).detach()
            out[seed] = [v.detach().cpu() for v in (x, w, norm, t, i)]
            stream.synchronize()

    one, many = {}, {}
    for seed in range(4):
        work(seed, one)
    threads = [threading.Thread(target=work, args=(seed, many)) for seed in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert one.keys() == many.keys()
    for seed in one:
        assert all(torch.equal(a, b) for a, b in zip(one[seed], many[seed]))


def test_a_clipped_update_is_a_clip_and_an_update():
    from oregon_gpt_oss_patching_b200.grad_clip import clipped_sgd_step
    model = _model(layers=1)
    ids = torch.randint(0, 512, (1, 100), generator=torch.Generator().manual_seed(2)).cuda()
    _gradients(model, ids)
    params = [p for p in model.parameters() if p.grad is not None]
    before = [p.detach().clone() for p in params]
    grads = [p.grad.clone() for p in params]
    limit = 0.25 * float(torch.sqrt(sum((g.double() ** 2).sum() for g in grads)))
    norm = clipped_sgd_step(params, 0.5, limit)
    c = min(1.0, limit / (float(norm) + 1e-6))
    assert abs(c - 0.25) < 1e-5
    for p, b, g in zip(params, before, grads):
        want = b.double() - 0.5 * c * g.double()
        # one rounding to bf16 of a value that fp32 has to 2^-23 of its summands
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * (b.double().abs() + g.double().abs())
        assert bool(((p.detach().double() - want).abs() <= tol).all())
