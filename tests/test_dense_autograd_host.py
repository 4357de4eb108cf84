"""What autograd is told by the dense operators, on the CPU: the host code decides
it, so the library's entry points are replaced by their formulas."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture
def formulas(monkeypatch):
    """The norm and the lookup with their gradients by torch's operations."""
    from usaf_b200 import embedding, norms

    def norm_fwd(x, weight, eps=1e-6, residual=None, want_rstd=True):
        total = x.detach() if residual is None else x.detach() + residual.detach()
        rstd = 1 / torch.sqrt(total.square().mean(-1) + eps)
        return total * rstd[..., None] * weight.detach(), rstd.reshape(-1), x if residual is None else total

    def norm_bwd(dy, x, weight, rstd, dsum=None, want_dw=True):
        r, w = rstd.view(*x.shape[:-1], 1), weight.detach()
        hat = x.detach() * r
        dx = r * (dy * w - hat * (dy * w * hat).mean(-1, keepdim=True)) + (0 if dsum is None else dsum)
        return dx, (dy * hat).reshape(-1, x.shape[-1]).sum(0) if want_dw else None

    monkeypatch.setattr(norms, "rms_norm_forward", norm_fwd)
    monkeypatch.setattr(norms, "rms_norm_backward", norm_bwd)
    monkeypatch.setattr(embedding, "embedding_forward",
                        lambda ids, table, scale=1.0, err=None: table.detach()[ids] * scale)


@pytest.mark.parametrize("grads", [True, False])
@pytest.mark.parametrize("leaf", [True, False])
def test_forward_mode_is_refused(formulas, grads, leaf):
    """A tangent would be lost: the call is refused instead, whichever input has one,
    with or without backward mode beside it."""
    from usaf_b200 import embedding, norms
    x, w, res = torch.randn(3, 8), torch.randn(8), torch.randn(3, 8)
    table, ids = torch.randn(5, 8), torch.tensor([1, 4])
    with torch.set_grad_enabled(grads), fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))

        for call in (lambda: norms.rms_norm(dual(x), w), lambda: norms.rms_norm(x, dual(w)),
                     lambda: norms.rms_norm(x, w, residual=dual(res)),
                     lambda: norms.rms_norm(dual(x), w, residual=res), lambda: embedding.embedding(ids, dual(table))):
            with pytest.raises(RuntimeError, match="jvp"):
                call()
        # no tangent: nothing to lose
        assert torch.equal(embedding.embedding(ids, table), table[ids])
        y, total = norms.rms_norm(x, w, residual=res)
        assert torch.equal(total, x + res) and not y.requires_grad
    assert torch.equal(embedding.embedding(ids, table), table[ids])
