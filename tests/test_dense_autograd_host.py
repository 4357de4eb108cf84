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


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors pass for the device's; the entry points only record their names."""
    from usaf_b200 import dense_optim, embedding
    names = []
    for mod in (embedding, dense_optim):
        monkeypatch.setattr(mod, "ptr", lambda t: None if t is None else t.data_ptr())
        monkeypatch.setattr(mod, "call_on", lambda index, name, *a: names.append(name))
    return names


def saved_by_a_graph(t):
    """A loss whose backward pass reads ``t`` as it is now."""
    x = torch.ones_like(t, requires_grad=True)
    return (x * t).sum()


def test_a_gradient_added_to_in_place_counts_as_changed(launches):
    from usaf_b200 import embedding
    grad, ids, dout = torch.zeros(5, 8), torch.tensor([1, 4]), torch.ones(2, 8)
    loss = saved_by_a_graph(grad)
    embedding.embedding_backward(dout, ids, 5, grad=grad)
    assert launches == ["usaf_embedding_bwd"] and grad._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # a new gradient is nobody's yet
    assert embedding.embedding_backward(dout, ids, 5)._version == 0


def test_the_tables_gradient_counts_as_changed(formulas, launches):
    """The same where the lookup adds to ``table.grad`` itself."""
    from usaf_b200 import embedding
    table = torch.zeros(5, 8, requires_grad=True)
    table.grad = torch.zeros(5, 8)
    held = table.grad
    loss = saved_by_a_graph(held)
    embedding.embedding_backward(torch.ones(2, 8), torch.tensor([1, 4]), 5, grad=table.grad)
    assert table.grad is held and held._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_states_and_masters_count_as_changed(launches, bits):
    """The step writes them in place as it does the parameters."""
    from usaf_b200 import dense_optim
    p, g, master = torch.ones(300), torch.ones(300), torch.zeros(512)
    m, v = torch.zeros(512), torch.zeros(512)
    if bits == 8:
        m, v = ((torch.zeros(512, dtype=torch.float8_e4m3fn), torch.zeros(2)) for _ in range(2))
    held = [p, master, *(m if bits == 8 else (m,)), *(v if bits == 8 else (v,))]
    loss = saved_by_a_graph(master)
    dense_optim.adamw_step([p], [g], m, v, step=1, lr=1e-3, masters=master)
    assert launches == ["usaf_adamw"] and [t._version for t in held] == [1] * len(held) and g._version == 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_into_grad_leaves_autograd_grad_its_gradient(formulas, monkeypatch):
    """A backward pass that does not add to the leaves' gradients gets the table's
    as any other, and ``.grad`` stays; ``backward()`` adds."""
    from usaf_b200 import embedding
    added = []

    def backward(dout, ids, V, scale=1.0, padding_idx=None, grad=None, err=None):
        g = torch.zeros(V, dout.shape[-1]) if grad is None else grad
        return g.index_add_(0, ids, dout * scale)

    def add(table, dout, ids, *args):
        added.append(1)
        backward(dout, ids, *args, grad=table.grad)

    monkeypatch.setattr(embedding, "embedding_backward", backward)
    monkeypatch.setattr(embedding, "_add_at_the_end", add)
    table, other = torch.randn(5, 8, requires_grad=True), torch.ones(2, 8, requires_grad=True)
    table.grad = torch.ones(5, 8)
    ids = torch.tensor([1, 4])
    err = torch.zeros(1, dtype=torch.int32)
    want = torch.zeros(5, 8).index_fill_(0, ids, 2.0)

    def loss():
        return (embedding.embedding(ids, table, 2.0, err=err, into_grad=True) * other).sum()

    for inputs in (table, [other, table]):
        got = torch.autograd.grad(loss(), inputs)
        assert torch.equal(got[-1], want) and not added and torch.equal(table.grad, torch.ones(5, 8))
    loss().backward(inputs=[other])
    assert not added and torch.equal(table.grad, torch.ones(5, 8))
    loss().backward()
    assert added == [1] and torch.equal(table.grad, 1 + want)
    loss().backward(inputs=[table])
    assert added == [1, 1] and torch.equal(table.grad, 1 + 2 * want)
    # a second derivative's pass inside another
    g, = torch.autograd.grad(loss(), table)
    (loss() + g.detach().sum()).backward()
    assert torch.equal(table.grad, 1 + 3 * want)
