"""AdamW over many steps (usaf_b200.dense_optim): what a refused call leaves
behind, parameters that skip steps, and 8-bit states over thousands of steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
BLOCK = 256


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import usaf_b200  # noqa: F401
    return torch.device("cuda:0")


def parameter(t):
    return torch.nn.Parameter(t, requires_grad=False)


def test_a_refused_step_changes_nothing(dev):
    """One launch a type of parameter or gradient: all are checked before the first."""
    from usaf_b200 import dense_optim
    named = {"a": parameter(torch.ones(300, device=dev)), "b": parameter(torch.ones(70, device=dev).bfloat16()),
             "c": parameter(torch.ones(70, device=dev).bfloat16())}
    opt = dense_optim.AdamW(named, lr=1e-2)
    good = {"a": torch.ones(300, device=dev), "b": torch.ones(70, device=dev), "c": torch.ones(70, device=dev).bfloat16()}
    for bad in (dict(good, b=torch.ones(69, device=dev)), dict(good, c=torch.ones(70, device=dev).half()),
                dict(good, b=torch.ones(70))):
        before = {n: (p.clone(), {k: t.clone() for k, t in opt.state(n).items()}) for n, p in named.items()}
        with pytest.raises((ValueError, TypeError)):
            opt.step(bad)
        for n, (p, state) in before.items():
            assert torch.equal(named[n], p) and all(torch.equal(opt.state(n)[k], t) for k, t in state.items()), n
    want = {n: p.clone() for n, p in named.items()}
    fresh = dense_optim.AdamW({n: parameter(p) for n, p in want.items()}, lr=1e-2)
    fresh.step(good)
    opt.step(good)
    assert all(torch.equal(named[n], p) for n, p in want.items())
