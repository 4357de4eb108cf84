"""The dense tensors of a Qwen3-MoE language model trained around the sparse
experts: embedding and norms on the device kernels (qwen3moe.use_dense_kernels)
and SparseTrainer's AdamW over them, as they are used together.

* the model's loss and every dense gradient against the same model on torch's
  own norms and embedding, both in fp32: the norm of the difference within 2e-4
  of the gradient's (each of ~25 operations in a row rounds its sums of up to
  512 terms by (512/32 + 60) 2^-24 = 5e-6 of their size, and the sizes exceed
  the results by a small factor);
* a step's update equals AdamW's, bit for bit, on the gradients it was given;
* micro-batches accumulate in the embedding's gradient as autograd adds them;
* skips, checkpoints, tokens outside the table, activation recompute.
"""
import pytest
import torch

from test_gpu_dense_optim import Plain

pytestmark = pytest.mark.gpu

E, K, H, I, LAYERS, VOCAB = 16, 4, 512, 256, 2, 521


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import usaf_b200  # noqa: F401
    return torch.device("cuda:0")


def make(dev, dtype, tie=False, dense=True):
    from transformers.models.qwen3_moe.configuration_qwen3_moe import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeForCausalLM
    from usaf_b200 import qwen3moe
    from usaf_b200.engine import Projection
    from usaf_b200.quantization import quantize_4bit
    qwen3moe.patch_qwen3moe_for_b200()
    torch.manual_seed(0)
    cfg = Qwen3MoeConfig(vocab_size=VOCAB, hidden_size=H, intermediate_size=1024, num_hidden_layers=LAYERS,
                         num_attention_heads=4, num_key_value_heads=2, head_dim=128, moe_intermediate_size=I,
                         num_experts=E, num_experts_per_tok=K, norm_topk_prob=True, max_position_embeddings=256,
                         tie_word_embeddings=tie, pad_token_id=3)
    m = Qwen3MoeForCausalLM(cfg).to(device=dev, dtype=dtype)
    for p in m.parameters():
        p.requires_grad_(False)
    g = torch.Generator(device=dev).manual_seed(1)
    for layer in m.model.layers:
        layer.mlp.gate.weight.data = (torch.randn(E, H, device=dev, generator=g) * 0.05).to(dtype)
        layer.mlp.gate.weight.requires_grad_(True)
        projs = []
        for shape in ((E, 2 * I, H), (E, H, I)):
            q, s, z, _ = quantize_4bit(torch.randn(*shape, device=dev, generator=g) * 0.02, 128)
            projs.append(Projection(q, s, z, shape, 128, dtype))
        qwen3moe.attach_int4_experts(layer.mlp.experts, *projs)
    for n, p in m.named_parameters():
        if "norm" in n:
            p.data = (1 + 0.2 * torch.randn(p.shape, device=dev, generator=g)).to(dtype)
    return qwen3moe.use_dense_kernels(m) if dense else m


def dense_names(m):
    return [n for n, _ in m.named_parameters() if "norm" in n or "embed_tokens" in n or n.endswith("gate.weight")]


def batch(seed, rows=2):
    return torch.randint(0, VOCAB, (rows, 64), generator=torch.Generator().manual_seed(seed)).cuda()


def lm_loss(model, ids):
    return model(input_ids=ids, labels=ids).loss


def trainer(m, **kw):
    from usaf_b200.trainer import SparseTrainer
    args = dict(steps=20, lr_peak=1e-3, accum=2, frac=0.01, reselect_every=100, dense_names=dense_names(m))
    args.update(kw)
    tr = SparseTrainer(m, **args)
    tr.init_selection(tr.importance(batch(99), lm_loss))
    return tr


@pytest.mark.parametrize("tie,recompute", [(False, False), (True, False), (False, True)])
def test_gradients_against_the_modules(dev, tie, recompute):
    grads, losses, calls = [], [], {}
    for dense in (False, True):
        m = make(dev, torch.float32, tie, dense)
        if recompute and dense:
            m.gradient_checkpointing_enable(gradient_checkpointing_kwargs={"use_reentrant": False})
            m.train()
        for n, p in m.named_parameters():
            p.requires_grad_(n in dense_names(m))
        if dense:       # the kernels run: counted at the library's entry points
            from usaf_b200 import embedding, norms
            kept = norms.call_on

            def counted(dev, name, *a):
                calls[name] = calls.get(name, 0) + 1
                kept(dev, name, *a)

            norms.call_on = embedding.call_on = counted
        try:
            loss = lm_loss(m, batch(5))
            loss.backward()
        finally:
            if dense:
                norms.call_on = embedding.call_on = kept
        losses.append(float(loss.detach()))
        grads.append({n: p.grad.double() for n, p in m.named_parameters() if p.grad is not None})
    twice = 2 if recompute else 1
    assert calls["usaf_rms_norm_fwd"] == 1 + 4 * LAYERS * twice and calls["usaf_rms_norm_bwd"] == 1 + 4 * LAYERS
    assert calls["usaf_embedding_fwd"] == calls["usaf_embedding_bwd"] == 1
    assert abs(losses[0] - losses[1]) <= 2e-5 * abs(losses[0])
    assert grads[0].keys() == grads[1].keys() and len(grads[0]) == 2 + 5 * LAYERS
    for n, want in grads[0].items():
        assert float((grads[1][n] - want).norm()) <= 2e-4 * float(want.norm()), n
    if not tie:
        assert not bool(grads[1]["model.embed_tokens.weight"][3].any())       # the padding's row


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 32), (torch.bfloat16, 8)])
def test_steps(dev, dtype, bits):
    m = make(dev, dtype)
    tr = trainer(m, dense_state_bits=bits)
    names = list(tr.dense_params)
    assert not tr.router_params and tr.router_opt is None
    master = dtype != torch.float32
    plain = {n: Plain(p.detach(), bits, master) for n, p in tr.dense_params.items()}
    seen, kept = {}, tr.dense_opt.step

    def step(grads=None, grad_div=1.0):
        seen.update(div=grad_div, grads={n: p.grad.detach().clone() for n, p in tr.dense_params.items()})
        kept(grads, grad_div)

    tr.dense_opt.step = step
    masters = {n: t.data.clone() for n, t in tr.masters.items()}
    for t in (1, 2):
        out = tr.train_step([batch(10 * t), batch(10 * t + 1)], lm_loss)
        assert out["finite"] and seen["div"] == 4096.0 * 2
        assert all(p.grad is None for p in tr.dense_params.values())
        for n in names:
            wd = tr.weight_decay if tr.dense_params[n].dim() == 2 else 0.0
            plain[n].step(seen["grads"][n], t, out["lr"], 0.9, 0.999, 1e-8, wd, seen["div"])
            assert torch.equal(tr.dense_params[n].detach().cpu(), plain[n].p), (t, n)
            assert bool(seen["grads"][n].any()), n
    assert any(not torch.equal(masters[n], tr.masters[n].data) for n in masters)     # the experts step beside them
    # a loss that is not finite: nothing moves
    before = {n: p.detach().clone() for n, p in tr.dense_params.items()}
    state = tr.dense_opt.state_dict()
    out = tr.train_step([batch(50), batch(51)], lambda mdl, ids: lm_loss(mdl, ids) * float("inf"))
    assert not out["finite"]
    assert all(torch.equal(before[n], p) for n, p in tr.dense_params.items())
    assert tr.dense_opt.state_dict()["step"] == state["step"] == 2
    assert all(torch.equal(tr.dense_opt.state_dict()["m"][n], state["m"][n]) for n in names)


def test_micro_batches_add_to_the_embedding(dev):
    """The gradient that the trainer's loop accumulates equals autograd's sum of
    the micro-batches (scale 1: one addition a row either way)."""
    m = make(dev, torch.float32)
    w = m.model.embed_tokens.weight.requires_grad_(True)
    got = []
    for into in (False, True):
        w.grad = None
        m.model.embed_tokens._usaf_into_grad = into
        for k in (1, 2, 3):
            lm_loss(m, batch(k)).backward()
        got.append(w.grad.clone())
    m.model.embed_tokens._usaf_into_grad = False
    # attention's backward pass may add in any order: an ulp or so of the terms
    assert float((got[0] - got[1]).norm()) <= 1e-5 * float(got[0].norm())
    tr = trainer(m)
    seen, kept = [], m.model.embed_tokens.forward
    m.model.embed_tokens.forward = lambda ids: (seen.append(m.model.embed_tokens._usaf_into_grad), kept(ids))[1]
    tr.train_step([batch(1), batch(2)], lm_loss)
    assert seen == [True, True] and not m.model.embed_tokens._usaf_into_grad


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint(dev, tmp_path, bits):
    m = make(dev, torch.bfloat16)
    tr = trainer(m, dense_state_bits=bits)
    tr.train_step([batch(1), batch(2)], lm_loss)
    path = tr.save_checkpoint(str(tmp_path / "c.pt"))
    m2 = make(dev, torch.bfloat16)
    tr2 = trainer(m2, dense_state_bits=bits)
    tr2.load_checkpoint(path)
    for n, p in tr.dense_params.items():
        assert torch.equal(p, tr2.dense_params[n]), n
        a, b = tr.dense_opt.state(n), tr2.dense_opt.state(n)
        assert all(torch.equal(a[k], b[k]) for k in ("m", "v", "master"))
    assert tr2.dense_opt.state_dict()["step"] == 1 and tr2.step_num == 1
    with pytest.raises(ValueError, match="dense tensors"):
        trainer(make(dev, torch.bfloat16), dense_names=()).load_checkpoint(path)
    from usaf_b200.checkpoint import get_checkpoint_metadata
    assert get_checkpoint_metadata(path)["format"] == "usaf-sparse-v1"


def test_tokens_outside_the_table_and_refusals(dev):
    from usaf_b200._lib import UsafError
    from usaf_b200.trainer import SparseTrainer
    m = make(dev, torch.bfloat16)
    tr = trainer(m)
    before = {n: p.detach().clone() for n, p in tr.dense_params.items()}

    def bad(mdl, ids):
        out = ids.clone()
        out[0, 5] = VOCAB + 7
        return mdl(input_ids=out, labels=ids).loss

    with pytest.raises(UsafError, match="outside"):
        tr.train_step([batch(1), batch(2)], bad)
    assert tr.step_num == 0 and all(torch.equal(before[n], p) for n, p in tr.dense_params.items())
    assert tr.train_step([batch(1), batch(2)], lm_loss)["finite"]
    with pytest.raises(ValueError, match="no parameter"):
        SparseTrainer(m, steps=5, dense_names=["model.nothing"])
    with pytest.raises(ValueError, match="leaf"):
        from usaf_b200 import embedding
        embedding.embedding(batch(1), m.model.embed_tokens.weight * 1.0, into_grad=True)


@pytest.mark.parametrize("into", [False, True])
def test_captured_forward_and_backward(dev, into):
    """Lookup, norm with residual and their backward pass through autograd as one
    graph (warmed up on a side stream, as torch asks): a replay with other
    tokens gives what the eager pass gives."""
    from usaf_b200 import embedding, norms
    V, W = 300, 256
    g = torch.Generator(device=dev).manual_seed(4)
    table = torch.randn(V, W, device=dev, generator=g).requires_grad_(True)
    weight = torch.rand(W, device=dev, generator=g).requires_grad_(True)
    ids = torch.randint(0, V, (3, 50), device=dev, generator=g)
    other = torch.randint(0, V, (3, 50), device=dev, generator=g)

    def run():
        x = embedding.embedding(ids, table, 2.0, padding_idx=1, into_grad=into)
        y, total = norms.rms_norm(x, weight, 1e-6, residual=x.detach())
        (y.square().sum() + total.sum()).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            table.grad = weight.grad = None
            run()
    torch.cuda.current_stream().wait_stream(side)
    if into:
        table.grad.zero_()
        weight.grad.zero_()
    else:
        table.grad = weight.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    ids.copy_(other)
    if into:
        table.grad.zero_()
        weight.grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    got = table.grad.clone(), weight.grad.clone()
    table.grad = weight.grad = None
    run()
    torch.cuda.synchronize()
    assert torch.equal(got[0], table.grad) and torch.equal(got[1], weight.grad)


def test_token_by_token_with_a_cache(dev):
    """Single tokens through the patched layers and the model's cache: the
    logits of the modules, within the rounding of ~25 operations (2e-4)."""
    ids = batch(7)
    out = []
    for dense in (False, True):
        m = make(dev, torch.float32, dense=dense).eval()
        with torch.no_grad():
            first = m(input_ids=ids[:, :40], use_cache=True)
            logits, past = [first.logits[:, -1]], first.past_key_values
            for t in range(40, 44):
                step = m(input_ids=ids[:, t:t + 1], past_key_values=past, use_cache=True)
                logits.append(step.logits[:, -1])
                past = step.past_key_values
        out.append(torch.stack(logits).double())
    assert float((out[0] - out[1]).norm()) <= 2e-4 * float(out[0].norm())
