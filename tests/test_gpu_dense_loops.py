"""SparseTrainer's steps with dense tensors (usaf_b200.trainer) where a loss
function or a gradient does something of its own."""
import pytest
import torch

from test_gpu_dense_train import batch, dev, lm_loss, make, trainer  # noqa: F401  (dev: a fixture)

pytestmark = pytest.mark.gpu


def test_a_loss_that_asks_for_the_embeddings_gradient(dev):  # noqa: F811
    """``torch.autograd.grad`` inside the loss function gives the gradient in every
    micro-batch and leaves ``.grad`` alone (1e-5: attention's backward pass may add in
    any order)."""
    m = make(dev, torch.float32)
    tr = trainer(m)
    w = m.model.embed_tokens.weight
    asked, held, kept = [], {}, tr.dense_opt.step

    def loss(mdl, ids):
        before = None if w.grad is None else w.grad.clone()
        asked.append(torch.autograd.grad(lm_loss(mdl, ids), w)[0])
        assert (w.grad is None) if before is None else torch.equal(w.grad, before)
        return lm_loss(mdl, ids)

    def step(grads=None, grad_div=1.0):
        held.update(grad=w.grad.clone(), div=grad_div)
        kept(grads, grad_div)

    tr.dense_opt.step = step
    assert tr.train_step([batch(1), batch(2)], loss)["finite"]
    assert len(asked) == 2 and all(bool(g.any()) for g in asked)
    want = (asked[0] + asked[1]) * (held["div"] / 2)
    assert float((held["grad"] - want).norm()) <= 1e-5 * float(want.norm())


@pytest.mark.parametrize("name", ["model.norm.weight", "model.embed_tokens.weight"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_dense_gradient_that_is_not_finite_skips_the_step(dev, name, value):  # noqa: F811
    """One value of one dense gradient, all expert gradients finite: nothing moves."""
    m = make(dev, torch.float32)
    tr = trainer(m)
    p = tr.dense_params[name]
    experts = {n: t.data.clone() for n, t in tr.masters.items()}
    dense = {n: t.detach().clone() for n, t in tr.dense_params.items()}

    def loss(mdl, ids):
        if p.grad is not None:      # in front of the last micro-batch's backward pass
            p.grad.view(-1)[-1] = value
        return lm_loss(mdl, ids)

    out = tr.train_step([batch(1), batch(2)], loss)
    assert not out["finite"] and tr.dense_opt.state_dict()["step"] == 0
    assert all(bool(torch.isfinite(g).all()) for g in tr.store.compact.values())
    assert all(torch.equal(experts[n], t.data) for n, t in tr.masters.items())
    assert all(torch.equal(dense[n], t) for n, t in tr.dense_params.items())
    assert tr.train_step([batch(1), batch(2)], lm_loss)["finite"]
    assert not any(torch.equal(dense[n], t) for n, t in tr.dense_params.items())
