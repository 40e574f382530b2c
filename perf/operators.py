"""The operators of the fine-tuning step around attention and the experts: what is timed, on which sizes, and in which plain form.

Four operators: the residual sum with its RMS norm, the routing of tokens to experts, the global gradient norm with clipping, and the
clipped SGD update.  ``run`` computes one pass: in elementary torch operations where ``own`` is false, by the framework's
public calls where it is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # a decoding step: the norm behind attention for a handful of sequences (latency)
        {"name": "norm_decode", "op": "norm", "tokens": 4, "hidden": 2880, "dtype": "bf16", "weight": "bf16", "residual": True, "train": False},
        # the norm behind attention in a fine-tuning step of 8192 tokens, forward and backward
        {"name": "norm_train", "op": "norm", "tokens": 8192, "hidden": 2880, "dtype": "bf16", "weight": "bf16", "residual": True, "train": True},
        # a short ragged batch whose norm weights are kept in 32 bits, as a loaded checkpoint has them; the norm before attention (no sum)
        {"name": "norm_fp32_weight", "op": "norm", "tokens": 1357, "hidden": 2880, "dtype": "bf16", "weight": "fp32", "residual": False, "train": True},
        # an odd width, in fp16
        {"name": "norm_odd", "op": "norm", "tokens": 2051, "hidden": 1447, "dtype": "fp16", "weight": "fp32", "residual": True, "train": True},
        # a decoding step's routing: top 4 of 32
        {"name": "router_decode", "op": "router", "tokens": 8, "experts": 32, "top_k": 4, "scoring": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "renormalize": True, "scale": 1.0, "dtype": "bf16", "train": False},
        # a fine-tuning step's routing of 8192 tokens, top 4 of 32, with its gradient
        {"name": "router_train", "op": "router", "tokens": 8192, "experts": 32, "top_k": 4, "scoring": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "renormalize": True, "scale": 1.0, "dtype": "bf16", "train": True},
        # many experts in groups, sigmoid scores and a bias that balances the load, over a long packed batch
        {"name": "router_groups", "op": "router", "tokens": 32771, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "renormalize": True, "scale": 2.5, "dtype": "bf16", "train": True},
        # the gradients of low-rank adapters: many small tensors (latency)
        {"name": "clip_adapters", "op": "clip", "layout": "adapters", "layers": 6, "rank": 8, "hidden": 2880, "experts": 0, "dtype": "bf16", "share": 0.3},
        # the gradients of one decoder layer with 32 experts
        {"name": "clip_layer", "op": "clip", "layout": "layer", "layers": 1, "rank": 0, "hidden": 2880, "experts": 32, "dtype": "bf16", "share": 0.3},
        # the same where the norm stays under the limit, as on most steps of a settled run: 8 experts, in 32 bits
        {"name": "clip_idle", "op": "clip", "layout": "layer", "layers": 1, "rank": 0, "hidden": 2880, "experts": 8, "dtype": "fp32", "share": 4.0},
        # the update of the adapters and of one decoder layer
        {"name": "sgd_adapters", "op": "sgd", "layout": "adapters", "layers": 4, "rank": 16, "hidden": 2880, "experts": 0, "dtype": "fp32", "share": 0.6},
        {"name": "sgd_layer", "op": "sgd", "layout": "layer", "layers": 1, "rank": 0, "hidden": 2880, "experts": 32, "dtype": "bf16", "share": 0.3},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "router", "router", "clip", "sgd"])
    if op == "norm":
        hidden = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            hidden = max(8, hidden // 8 * 8)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        return {"op": op, "tokens": _log(rng, 1, max(1, 8192 * 2880 // hidden)), "hidden": hidden, "dtype": dtype,
                "weight": rng.choice([dtype, "fp32"]), "residual": rng.random() < 0.7, "train": rng.random() < 0.7}
    if op == "router":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 4, 256 // groups)
        top_groups = rng.randint((groups + 1) // 2, groups)
        top_k = rng.randint(1, min(8, top_groups * (experts // groups)))
        return {"op": op, "tokens": _log(rng, 1, 32768), "experts": experts, "top_k": top_k,
                "scoring": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.4, "groups": groups, "top_groups": top_groups,
                "renormalize": top_k > 1 and rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "train": rng.random() < 0.7}
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    share = rng.choice([0.3, 0.6, 4.0])
    hidden = _log(rng, 200, 2880)
    if rng.random() < 0.5:
        return {"op": op, "layout": "adapters", "layers": rng.randint(1, 6), "rank": _log(rng, 1, 64), "hidden": hidden, "experts": 0, "dtype": dtype, "share": share}
    return {"op": op, "layout": "layer", "layers": 1, "rank": 0, "hidden": hidden, "experts": _log(rng, 1, 16), "dtype": dtype, "share": share}


def _shapes(case):
    """The tensors of low-rank adapters on the four projections of `layers` layers, or of one whole decoder layer."""
    h, r, e = case["hidden"], case["rank"], case["experts"]
    if case["layout"] == "adapters":
        return [(r, h), (4096, r), (r, h), (512, r), (r, h), (512, r), (r, 4096), (h, r)] * case["layers"]
    return [(4096, h), (4096,), (512, h), (512,), (512, h), (512,), (h, 4096), (h,), (64,), (h,), (h,), (e, h), (e,),
            (e, h, 2 * h), (e, 2 * h), (e, h, h), (e, h)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, of=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=of).mul_(scale)

    state = dict(case)
    if case["op"] == "norm":
        t, h = case["tokens"], case["hidden"]
        # activations of a residual stream: a few wide channels, and sums that outgrow the block's output
        state["x"] = normal(t, h).mul_(1 + 4 * torch.rand(h, generator=g, device="cuda").to(dtype).pow(8))
        state["r"] = normal(t, h, scale=3.0) if case["residual"] else None
        state["w"] = (1 + normal(h, scale=0.1, of=torch.float32)).to(DTYPES[case["weight"]])
        if case["train"]:
            state["dy"] = normal(t, h, scale=0.01)
            state["dh"] = normal(t, h, scale=0.01) if case["residual"] else None
            state["x"].requires_grad_(True)
            state["w"].requires_grad_(True)
            if case["residual"]:
                state["r"].requires_grad_(True)
    elif case["op"] == "router":
        t, e = case["tokens"], case["experts"]
        state["logits"] = normal(t, e, scale=2.0)
        state["b"] = normal(e, scale=0.05, of=torch.float32) if case["bias"] else None
        if case["train"]:
            state["dw"] = normal(t, case["top_k"])
            state["logits"].requires_grad_(True)
    else:
        grads = [normal(*s, scale=0.02) for s in _shapes(case)]
        count = sum(x.numel() for x in grads)
        state["max_norm"] = case["share"] * 0.02 * math.sqrt(count)
        if case["op"] == "sgd":
            state["lr"] = 1e-3
            params = [torch.nn.Parameter(normal(*s, scale=0.5)) for s in _shapes(case)]
        else:
            params = [torch.nn.Parameter(torch.empty_like(x)) for x in grads]
        for p, x in zip(params, grads):
            p.grad = x
        state["params"] = params
    return state


def run(state):
    if own:
        out = _own(state)
    else:
        with torch.no_grad():
            out = {"norm": _plain_norm, "router": _plain_router, "clip": _plain_clip, "sgd": _plain_sgd}[state["op"]](state)
    if state.get("share", 1.0) < 1.0:
        state["max_norm"] *= 0.9999   # the limit sinks a little from pass to pass: gradients that were clipped already are clipped again
    return out


def _own(s):
    if s["op"] == "norm":
        from oregon_gpt_oss_patching_b200.rms_norm import add_rms_norm, rms_norm
        if not s["train"]:
            with torch.no_grad():
                if s["residual"]:
                    y, h = add_rms_norm(s["x"], s["r"], s["w"], EPS)
                    return {"y": y, "h": h}
                return {"y": rms_norm(s["x"], s["w"], EPS)}
        if s["residual"]:
            y, h = add_rms_norm(s["x"], s["r"], s["w"], EPS)
            dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
            return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}
        y = rms_norm(s["x"], s["w"], EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if s["op"] == "router":
        from oregon_gpt_oss_patching_b200.moe_router import router_topk
        w, i = router_topk(s["logits"], s["top_k"], scoring=s["scoring"], bias=s["b"], num_groups=s["groups"], top_groups=s["top_groups"],
                           renormalize=s["renormalize"], scale=s["scale"])
        if not s["train"]:
            return {"weights": w, "indices": i}
        (dl,) = torch.autograd.grad(w, s["logits"], s["dw"])
        return {"weights": w, "indices": i, "dlogits": dl}
    from oregon_gpt_oss_patching_b200.grad_clip import clip_grad_norm, clipped_sgd_step
    if s["op"] == "clip":
        norm = clip_grad_norm(s["params"], s["max_norm"])
        return {"norm": norm, "grads": [p.grad for p in s["params"]]}
    norm = clipped_sgd_step(s["params"], s["lr"], s["max_norm"])
    return {"norm": norm, "params": s["params"]}


def _plain_norm(s):
    x, w = s["x"], s["w"].float()
    # the sum is a tensor of the residual stream: it is rounded to its type, and the norm is taken of what the stream holds
    h = (x.float() + s["r"].float()).to(x.dtype) if s["residual"] else x
    v = h.float()
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    n = v * rstd
    out = {"y": (n * w).to(x.dtype)}
    if s["residual"]:
        out["h"] = h
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
        if s["residual"]:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(x.dtype)
        if s["residual"]:
            out["dr"] = out["dx"]
        out["dw"] = (dy * n).sum(0).to(s["w"].dtype)
    return out


def _plain_router(s):
    logits, k, groups = s["logits"].float(), s["top_k"], s["groups"]
    t, e = logits.shape
    score = torch.exp(logits - logits.amax(1, keepdim=True)) if s["scoring"] == "softmax" else 1 / (1 + torch.exp(-logits))
    if s["scoring"] == "softmax":
        score = score / score.sum(1, keepdim=True)
    # without a bias and groups the scores rise with the logits; otherwise values next to a border are told apart in 64 bits
    value = logits
    if s["bias"] or groups > 1:
        value = logits.double()
        value = torch.exp(value - value.amax(1, keepdim=True)) if s["scoring"] == "softmax" else 1 / (1 + torch.exp(-value))
        if s["scoring"] == "softmax":
            value = value / value.sum(1, keepdim=True)
        if s["bias"]:
            value = value + s["b"].double()
    if groups > 1:
        best = value.view(t, groups, e // groups).sort(dim=-1, descending=True).values[..., :2].sum(-1)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        open_ = torch.zeros(t, groups, dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        value = torch.where(open_.repeat_interleave(e // groups, dim=1), value, -math.inf)
    index = value.sort(dim=1, descending=True, stable=True).indices[:, :k].contiguous()
    chosen = score.gather(1, index)
    total = chosen.sum(1, keepdim=True) if s["renormalize"] else torch.ones_like(chosen[:, :1])
    weight = chosen / total * s["scale"]
    out = {"weights": weight.to(s["logits"].dtype), "indices": index}
    if s["train"]:
        d = s["dw"].float() * s["scale"] / total
        if s["renormalize"]:
            d = d - (d * chosen / total).sum(1, keepdim=True)
        dscore = torch.zeros_like(score).scatter_(1, index, d)
        if s["scoring"] == "softmax":
            dl = score * (dscore - (dscore * score).sum(1, keepdim=True))
        else:
            dl = dscore * score * (1 - score)
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _coefficient(grads, max_norm):
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    norm, c = _coefficient(grads, s["max_norm"])
    return {"norm": norm, "grads": [g.copy_(g.float() * c) for g in grads]}


def _plain_sgd(s):
    norm, c = _coefficient([p.grad for p in s["params"]], s["max_norm"])
    return {"norm": norm, "params": [p.copy_(p.float() - s["lr"] * (c * p.grad.float())) for p in s["params"]]}


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "norm":
        # in: x (and r), dy (and dh), the weight; out: y (and h), dx (which is dr too), the weight's gradient
        n = case["tokens"] * case["hidden"]
        weight = case["hidden"] * torch.finfo(DTYPES[case["weight"]]).bits // 8
        passes = (4 if case["residual"] else 2) + ((3 if case["residual"] else 2) if case["train"] else 0)
        return {"bytes": passes * n * size + weight * (2 if case["train"] else 1), "flops": n * (14 if case["train"] else 5)}
    if case["op"] == "router":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        moved = t * e * size + t * k * (size + 8)
        if case["train"]:
            # the gradient of the weights in, the gradient of the logits out
            moved += t * k * size + t * e * size
        return {"bytes": moved + (4 * e if case["bias"] else 0), "flops": t * e * (8 if case["train"] else 4)}
    n = sum(math.prod(s) for s in _shapes(case))
    clips = case["share"] < 1.0
    if case["op"] == "clip":
        # the gradients in, and out again where they are scaled (a second read lies between, once their norm is known)
        return {"bytes": n * size * (2 if clips else 1), "flops": n * (3 if clips else 2)}
    # gradients and parameters in, the parameters out
    return {"bytes": n * size * 3, "flops": n * 4}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "router": _exact_router}.get(case["op"], _exact_clip)(s)


def _exact_norm(s):
    x, w = s["x"].double(), s["w"].double()
    h = x
    if s["residual"]:
        h = (x + s["r"].double()).to(s["x"].dtype).double()
    width = h.shape[1]
    length = (torch.linalg.vector_norm(h, dim=1) ** 2 / width + EPS).sqrt()[:, None]
    out = {"y": h / length * w}
    if s["residual"]:
        out["h"] = h
    if s["train"]:
        dy = s["dy"].double()
        u = dy * w
        dx = u / length - h * torch.einsum("th,th->t", u, h)[:, None] / (width * length ** 3)
        if s["residual"]:
            dx = dx + s["dh"].double()
        out["dx"] = dx
        if s["residual"]:
            out["dr"] = dx
        out["dw"] = torch.einsum("th,th->h", dy, h / length)
    return out


def _exact_router(s):
    logits = s["logits"].detach().double()
    t, e = logits.shape
    leaf = logits.clone().requires_grad_(True)
    with torch.enable_grad():
        score = torch.softmax(leaf, 1) if s["scoring"] == "softmax" else torch.sigmoid(leaf)
        value = score.detach()
        if s["b"] is not None:
            value = value + s["b"].double()[None]
        elif s["groups"] == 1:
            value = logits
        if s["groups"] > 1:
            parts = value.reshape(t, s["groups"], -1)
            first = parts.amax(-1)
            rest = parts.scatter(2, parts.argmax(-1, keepdim=True), -math.inf).amax(-1)
            rank = torch.argsort(first + rest, dim=1, descending=True, stable=True).argsort(dim=1)
            value = parts.masked_fill((rank >= s["top_groups"])[..., None], -math.inf).reshape(t, e)
        index = torch.argsort(value, dim=1, descending=True, stable=True)[:, :s["top_k"]].contiguous()
        weight = torch.take_along_dim(score, index, 1) * s["scale"]
        if s["renormalize"]:
            weight = weight * (s["scale"] / weight.sum(1, keepdim=True))
    out = {"weights": weight.detach(), "indices": index}
    if s["train"]:
        (out["dlogits"],) = torch.autograd.grad(weight, leaf, s["dw"].double())
    return out


def _exact_clip(s):
    params = s["params"]
    norm = math.hypot(*[float(torch.linalg.vector_norm(p.grad, dtype=torch.float64)) for p in params])
    c = min(1.0, s["max_norm"] / (norm + 1e-6))
    told = torch.tensor(norm, dtype=torch.float64, device="cuda")
    if s["op"] == "clip":
        return {"norm": told, "grads": [p.grad.double() * c for p in params]}
    return {"norm": told, "params": [p.detach().double() - s["lr"] * c * p.grad.double() for p in params]}
