"""The patched norms in a model whose weights are fp32 and whose matrix products run in bf16 (autocast)."""
import pytest
import torch

from oregon_gpt_oss_patching_b200.rms_norm import patch_rms_norm, unpatch_rms_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_gradients_under_autocast_are_the_model_s():
    """Both against the model in fp32: the patched one may be as far from it as the unpatched one and half as much again, since
    both round the same matrix products to bf16."""
    from transformers import GptOssConfig
    from transformers.models.gpt_oss import modeling_gpt_oss
    cfg = GptOssConfig(num_hidden_layers=2, hidden_size=128, intermediate_size=64, num_local_experts=4, num_experts_per_tok=4, vocab_size=64,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=64, layer_types=["sliding_attention", "full_attention"],
                       use_cache=False)
    cfg._attn_implementation, cfg._experts_implementation = "eager", "eager"
    torch.manual_seed(0)
    with torch.device(DEV):
        model = modeling_gpt_oss.GptOssForCausalLM(cfg).float()
    ids = torch.randint(0, 64, (2, 33), generator=torch.Generator().manual_seed(1)).to(DEV)

    def step(enabled):
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=enabled):
            loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        return {n: p.grad.double() for n, p in model.named_parameters() if p.grad is not None}

    exact, plain = step(False), step(True)
    patch_rms_norm()
    try:
        ours = step(True)
    finally:
        unpatch_rms_norm()
    assert ours.keys() == plain.keys() == exact.keys()
    for name, ref in exact.items():
        if float(ref.norm()):
            off = float((plain[name] - ref).norm() / ref.norm())
            assert float((ours[name] - ref).norm() / ref.norm()) <= 1.5 * off + 2.0 ** -7, (name, off)
