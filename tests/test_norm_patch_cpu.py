"""The patched norm and decoder layer as modules, without a GPU: the fused calls are replaced by their 64-bit formula, and the layer
must give what transformers' own gives, hooks and mixed types included."""
import pytest
import torch

from oracle import step_fp64
from oregon_gpt_oss_patching_b200 import rms_norm as mod


class _Attention(torch.nn.Module):
    """Stands in for the attention: its output's type is that of an autocast matrix product."""

    def __init__(self, dtype):
        super().__init__()
        self.dtype = dtype

    def forward(self, hidden_states, **kwargs):
        return (hidden_states * 0.5 + 1.0).to(self.dtype), None


class _Mlp(torch.nn.Module):
    def forward(self, hidden_states):
        return hidden_states * 2.0, None


def _layer(dtype=torch.float32, attention=torch.float32):
    from transformers import GptOssConfig
    from transformers.models.gpt_oss import modeling_gpt_oss
    cfg = GptOssConfig(num_hidden_layers=1, hidden_size=24, intermediate_size=16, num_local_experts=2, num_experts_per_tok=1, vocab_size=8,
                       num_attention_heads=2, num_key_value_heads=1, head_dim=8)
    cfg._attn_implementation = "eager"
    layer = modeling_gpt_oss.GptOssDecoderLayer(cfg, 0)
    g = torch.Generator().manual_seed(0)
    for norm in (layer.input_layernorm, layer.post_attention_layernorm):
        norm.weight.data = (1 + 0.3 * torch.randn(24, generator=g)).to(dtype)
    layer.self_attn, layer.mlp = _Attention(attention), _Mlp()
    return layer, torch.randn(2, 5, 24, generator=g).to(dtype)


@pytest.fixture
def patched(monkeypatch):
    """Patches the model, with the kernels' formula behind the two calls; lists the fused ones."""
    fused = []

    def add_rms_norm(x, residual, weight, eps):
        if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
            raise ValueError("residual must match x")
        fused.append(residual is not None)
        y, h = step_fp64.add_rms_norm(x, residual, weight, eps)
        return y.to(x.dtype), h.to(x.dtype)

    monkeypatch.setattr(mod, "add_rms_norm", add_rms_norm)
    monkeypatch.setattr(mod, "rms_norm", lambda x, weight, eps: step_fp64.add_rms_norm(x, None, weight, eps)[0].to(x.dtype))
    mod.patch_rms_norm()
    yield fused
    mod.unpatch_rms_norm()


def _both(layer, x, fused):
    """(patched, original) results of a layer."""
    ours = layer(x)
    mod.unpatch_rms_norm()
    try:
        plain = layer(x)
    finally:
        mod.patch_rms_norm()
    assert ours.dtype == plain.dtype
    # fp32 on one side, 64 bits on the other: a sum of 24 squares, a root, a few products and sums
    assert torch.allclose(ours.double(), plain.double(), rtol=64 * 2.0 ** -24, atol=64 * 2.0 ** -24)
    return ours


def test_the_plain_layer_is_fused(patched):
    layer, x = _layer()
    _both(layer, x, patched)
    assert patched == [False, True]


@pytest.mark.parametrize("name", ["input_layernorm", "post_attention_layernorm"])
def test_hooks_of_the_norms_run(patched, name):
    layer, x = _layer()
    norm = getattr(layer, name)
    seen = []
    handles = [norm.register_forward_pre_hook(lambda m, args: seen.append(("in", args[0].clone())) or (args[0] * 1.5,)),
               norm.register_forward_hook(lambda m, args, out: seen.append(("out", out.clone())) or out + 1.0)]
    _both(layer, x, patched)
    assert [s[0] for s in seen] == ["in", "out"] * 2
    for a, b in zip(seen[:2], seen[2:]):
        assert torch.allclose(a[1], b[1], rtol=64 * 2.0 ** -24, atol=64 * 2.0 ** -24)
    for h in handles:
        h.remove()
    del patched[:]
    _both(layer, x, patched)
    assert patched == [False, True]                       # fused again


def test_a_hook_may_bring_the_weight(patched):
    """A sharded parameter is empty until a hook in front of its module gathers it."""
    layer, x = _layer()
    norm = layer.post_attention_layernorm
    whole = norm.weight.data.clone()
    norm.weight.data = torch.empty(0)
    norm.register_forward_pre_hook(lambda m, args: setattr(m.weight, "data", whole))
    norm.register_forward_hook(lambda m, args, out: setattr(m.weight, "data", torch.empty(0)))
    _both(layer, x, patched)
    assert norm.weight.numel() == 0


def test_global_hooks_backward_hooks_and_replaced_forwards_run(patched):
    layer, x = _layer()
    calls = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, args, out: calls.append(type(m).__name__))
    try:
        layer(x)
    finally:
        handle.remove()
    assert calls.count("GptOssRMSNorm") == 2
    backward = []
    handle = layer.post_attention_layernorm.register_full_backward_hook(lambda m, gi, go: backward.append(1))
    layer(x.clone().requires_grad_(True)).sum().backward()
    handle.remove()
    assert backward == [1]
    own = layer.input_layernorm.forward
    layer.input_layernorm.forward = lambda h: own(h) * 3.0            # as a wrapper of one module does
    _both_own = layer(x)
    del layer.input_layernorm.forward
    assert not torch.allclose(_both_own, layer(x))
    layer.input_layernorm = torch.nn.Identity()                        # another module in its place
    _both(layer, x, patched)


@pytest.mark.parametrize("dtype,attention", [(torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
def test_a_stream_wider_than_the_attention_s_output(patched, dtype, attention):
    layer, x = _layer(dtype, attention)
    assert _both(layer, x, patched).dtype == torch.float32
