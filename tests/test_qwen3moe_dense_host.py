"""qwen3moe.use_dense_kernels and what a user does to the model beside it, on the
CPU with the kernels replaced by their formulas: hooks on the norms, modules put
in their place, mixed types."""
import copy

import pytest
import torch


@pytest.fixture
def model(monkeypatch):
    from transformers.models.qwen3_moe.configuration_qwen3_moe import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeForCausalLM
    from usaf_b200 import embedding, norms, qwen3moe

    def rms_norm(x, w, eps=1e-6, residual=None):
        if residual is not None and residual.dtype is not x.dtype:       # as the kernels' checks
            raise TypeError(f"residual: expected dtype {x.dtype}, got {residual.dtype}")
        total = x if residual is None else x + residual
        t = total.float()
        y = (t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w).to(x.dtype)
        return y if residual is None else (y, total)

    monkeypatch.setattr(norms, "rms_norm", rms_norm)
    monkeypatch.setattr(embedding, "embedding", lambda ids, table, scale=1.0, padding_idx=None, err=None, into_grad=False:
                        torch.nn.functional.embedding(ids, table, padding_idx) * scale)
    torch.manual_seed(3)
    cfg = Qwen3MoeConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=2,
                         num_attention_heads=2, num_key_value_heads=1, head_dim=16, moe_intermediate_size=16,
                         num_experts=4, num_experts_per_tok=2, max_position_embeddings=64, mlp_only_layers=[0, 1])
    return qwen3moe.use_dense_kernels(Qwen3MoeForCausalLM(cfg))


IDS = torch.arange(24).view(2, 12)


def test_hooks_of_the_norm_behind_the_attention_run(model):
    post = model.model.layers[0].post_attention_layernorm
    want = model(input_ids=IDS).logits
    seen = []
    hooks = [post.register_forward_pre_hook(lambda m, args: seen.append(("before", args[0].detach()))),
             post.register_forward_hook(lambda m, args, out: seen.append(("after", out.detach()))),
             post.register_full_backward_hook(lambda m, gin, gout: seen.append(("backward", gout[0])))]
    got = model(input_ids=IDS).logits
    got.square().mean().backward()
    assert [k for k, _ in seen] == ["before", "after", "backward"]
    x = seen[0][1]           # the sum of the residual and the attention, as the module's input is
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + post.variance_epsilon)
    assert torch.allclose(seen[1][1], x * r * post.weight, rtol=1e-5, atol=1e-6)
    assert torch.equal(got, want)
    for h in hooks:
        h.remove()
    seen.clear()
    model(input_ids=IDS)
    assert not seen
    # a hook that changes the norm's output is followed
    h = post.register_forward_hook(lambda m, args, out: out * 0)
    assert not torch.equal(model(input_ids=IDS).logits, want)
    h.remove()
    # one for all modules
    with torch.nn.modules.module.register_module_forward_hook(lambda m, a, o: seen.append(m) if m is post else None):
        model(input_ids=IDS)
    assert seen == [post]


def test_a_module_in_the_norms_place_is_called(model):
    class Twice(torch.nn.Module):
        def __init__(self, norm):
            super().__init__()
            self.norm, self.calls = norm, 0
            self.weight, self.variance_epsilon = norm.weight, norm.variance_epsilon

        def forward(self, x):
            self.calls += 1
            return 2 * self.norm(x)

    layer = model.model.layers[1]
    want = model(input_ids=IDS).logits
    layer.post_attention_layernorm = Twice(layer.post_attention_layernorm)
    got = model(input_ids=IDS).logits
    assert layer.post_attention_layernorm.calls == 1 and not torch.equal(got, want)


def test_the_fused_addition_is_what_runs_otherwise(model, monkeypatch):
    from usaf_b200 import norms
    fused, kept = [], norms.rms_norm
    monkeypatch.setattr(norms, "rms_norm", lambda x, w, eps=1e-6, residual=None:
                        (fused.append(residual is not None), kept(x, w, eps, residual))[1])
    copy.deepcopy(model)(input_ids=IDS)
    assert fused.count(True) == 2


def test_mixed_types_under_autocast(model):
    """fp32 weights with 16-bit products: the attention's rows are 16-bit, the
    residual's are not; torch's addition takes them, so the layer does."""
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = model(input_ids=IDS).logits
    want = model(input_ids=IDS).logits
    # ~20 bf16 operations in a row, 2^-8 of their sizes each
    assert got.dtype == torch.bfloat16
    assert float((got.float() - want).norm()) <= 20 * 2.0 ** -8 * float(want.norm())
    got.float().square().mean().backward()
    assert model.model.layers[0].post_attention_layernorm.weight.grad.dtype == torch.float32
