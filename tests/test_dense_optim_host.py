"""AdamW's checks on the CPU, the library's entry point replaced: which memory
the tensors of a step may share."""
import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    from usaf_b200 import dense_optim
    names = []
    monkeypatch.setattr(dense_optim, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(dense_optim, "call_on", lambda index, name, *a: names.append(name))
    return names


def test_states_that_overlap_are_refused(launches):
    """Not only where they begin at the same place: two launches' threads would write
    the same values."""
    from usaf_b200.dense_optim import adamw_step
    hold = torch.zeros(4096)
    p, g = [torch.ones(300), torch.ones(0), torch.ones(200)], [torch.ones(300), torch.ones(0), torch.ones(200)]
    kw = dict(step=1, lr=1e-3)
    m, v, masters = hold[:768], hold[768:1536], hold[1536:2304]
    adamw_step(p, g, m, v, masters=masters, **kw)
    assert len(launches) == 1
    for bad in (dict(v=hold[512:1280]), dict(v=hold[764:1532]), dict(masters=hold[1280:2048]), dict(m=hold[1532:2300])):
        args = dict(dict(m=m, v=v, masters=masters), **bad)
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(p, g, args["m"], args["v"], masters=args["masters"], **kw)
    # with a parameter
    inside = [hold[700:1000], torch.ones(0), torch.ones(200)]
    behind = [torch.ones(300), torch.ones(0), hold[2303:2503]]
    beside = [hold[2304:2604], hold[1000:1000], hold[2604:2804]]
    for params in (inside, behind):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step(params, g, m, v, masters=masters, **kw)
    assert len(launches) == 1
    adamw_step(beside, g, m, v, masters=masters, **kw)
    # 8 bits: values and scales
    q = hold[2816:3200].view(torch.float8_e4m3fn)          # 1536 bytes, 384 values of 4 bytes
    codes = (q[:768], torch.zeros(3)), (q[768:1536], torch.zeros(3))
    adamw_step(p, g, *codes, **kw)
    over = (codes[0][0], codes[0][1]), (q[752:1520], codes[1][1])
    with pytest.raises(ValueError, match="share memory"):
        adamw_step(p, g, *over, **kw)
    assert len(launches) == 3
