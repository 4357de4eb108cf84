"""The dense operators' host side on the CPU: layouts, refusals of CPU tensors
(no fallback), and the glue of the patched model -- decoder layer, norms and
embedding -- with torch's formulas in the kernels' place."""
import pytest
import torch


def test_state_layout():
    from usaf_b200.dense_optim import state_layout
    assert state_layout([]) == ([], 0)
    assert state_layout([1, 256, 257, 0, 5]) == ([0, 256, 512, 1024, 1024], 1280)


def test_cpu_tensors_are_refused():
    from usaf_b200 import dense_optim, embedding, norms
    x, w = torch.ones(2, 8), torch.ones(8)
    with pytest.raises(TypeError, match="CUDA"):
        norms.rms_norm(x, w)
    with pytest.raises(TypeError, match="CUDA"):
        norms.rms_norm_backward(x, x, w, torch.ones(2))
    with pytest.raises(TypeError, match="CUDA"):
        embedding.embedding(torch.zeros(2, dtype=torch.long), x)
    with pytest.raises(TypeError, match="CUDA"):
        embedding.embedding_backward(x, torch.zeros(2, dtype=torch.long), 4)
    with pytest.raises(TypeError, match="CUDA"):
        dense_optim.adamw_step([x], [x], torch.zeros(256), torch.zeros(256), step=1, lr=1e-3)
    with pytest.raises(TypeError, match="CUDA"):
        dense_optim.AdamW({"w": torch.nn.Parameter(w)})


def test_argument_checks_come_before_the_device():
    from usaf_b200 import dense_optim, embedding, norms
    x, w = torch.ones(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="shape"):
        norms.rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="at most"):
        norms.rms_norm(torch.ones(1, 40000), torch.ones(40000))
    with pytest.raises(TypeError, match="weight"):
        norms.rms_norm(x, w.half())
    with pytest.raises(TypeError, match="ids"):
        embedding.embedding(torch.zeros(2), x)
    with pytest.raises(ValueError, match="padding_idx"):
        embedding.embedding(torch.zeros(2, dtype=torch.long), x, padding_idx=2)
    with pytest.raises(ValueError, match="gradients for"):
        dense_optim.adamw_step([x], [], torch.zeros(256), torch.zeros(256), step=1, lr=1e-3)
    with pytest.raises(ValueError, match="step"):
        dense_optim.adamw_step([x], [x], torch.zeros(256), torch.zeros(256), step=0, lr=1e-3)


def test_sizes_beyond_the_call_are_refused():
    """Widths and step numbers that the C interface's 32 bits would cut off."""
    from usaf_b200 import dense_optim, embedding
    wide, ids = torch.empty(1, embedding.MAX_WIDTH + 1), torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError, match="at most"):
        embedding.embedding(ids, wide)
    with pytest.raises(ValueError, match="at most"):
        embedding.embedding_backward(wide, ids, 4)
    x = torch.ones(2, 8)
    with pytest.raises(ValueError, match="step"):
        dense_optim.adamw_step([x], [x], torch.zeros(256), torch.zeros(256), step=1 << 32 | 1, lr=1e-3)


def test_model_glue(monkeypatch):
    """use_dense_kernels on a model without MoE blocks, the kernels replaced by
    their formulas: same logits and gradients as the modules, to the rounding of
    64-bit arithmetic."""
    from transformers.models.qwen3_moe.configuration_qwen3_moe import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeForCausalLM
    from usaf_b200 import embedding, norms, qwen3moe
    used = []

    def rms_norm(x, w, eps=1e-6, residual=None):
        used.append("residual" if residual is not None else "norm")
        total = x if residual is None else x + residual
        y = total / torch.sqrt(total.square().mean(-1, keepdim=True) + eps) * w
        return y if residual is None else (y, total)

    def lookup(ids, table, scale=1.0, padding_idx=None, err=None, into_grad=False):
        used.append("embedding")
        assert err.dtype == torch.int32 and not into_grad
        return torch.nn.functional.embedding(ids, table, padding_idx) * scale

    monkeypatch.setattr(norms, "rms_norm", rms_norm)
    monkeypatch.setattr(embedding, "embedding", lookup)
    cfg = Qwen3MoeConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=2,
                         num_attention_heads=2, num_key_value_heads=1, head_dim=16, moe_intermediate_size=16,
                         num_experts=4, num_experts_per_tok=2, max_position_embeddings=64, mlp_only_layers=[0, 1])
    out = []
    for dense in (False, True):
        torch.manual_seed(3)
        m = Qwen3MoeForCausalLM(cfg).double()
        if dense:
            assert qwen3moe.use_dense_kernels(m) is m
        ids = torch.arange(24).view(2, 12) % 64
        logits = m(input_ids=ids).logits
        logits.square().mean().backward()
        out.append((logits.detach(), {n: p.grad for n, p in m.named_parameters()}))
    assert used.count("embedding") == 1 and used.count("residual") == 2 and used.count("norm") == 2 * 3 + 1
    # the modules' norms compute in fp32
    assert float((out[0][0] - out[1][0]).norm()) <= 1e-5 * float(out[0][0].norm())
    for n, g in out[0][1].items():
        assert float((out[1][1][n] - g).norm()) <= 1e-4 * float(g.norm()), n
    assert qwen3moe.embeddings(m) == [m.model.embed_tokens] and len(qwen3moe.error_words(m)) == 1
