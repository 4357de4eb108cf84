"""Embedding lookup and the table's gradient (usaf_b200.embedding) against 64
bits: from one token to many, equal tokens in runs longer than any split, odd
and unaligned widths, padding, tokens outside the table, accumulation.

Tolerances, u = finfo(type).eps / 2 and e = 2^-24: the lookup is one product
in fp32 and one rounding, |y| (u + e); a gradient row of n tokens is n + 1
additions, one product and one rounding, u |G| + (n + 3) e (|scale| sum|dy| + |G0|).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import usaf_b200  # noqa: F401
    return torch.device("cuda:0")


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def tokens(dev, n, V, law, seed=0):
    u = torch.rand(n, device=dev, generator=gen(dev, seed), dtype=torch.float64)
    if law == "uniform":
        return (u * V).long().clamp_(max=V - 1)
    if law == "rank":
        return (float(V) ** u).long().clamp_(1, V) - 1
    if law == "one":
        return torch.full((n,), V // 2, device=dev)
    assert law == "runs"            # long runs, one after another
    return (torch.arange(n, device=dev) // 100) % V


def check_grad(got, dy, ids, V, scale, pad=None, start=None):
    H = dy.shape[-1]
    ids, dy = ids.reshape(-1), dy.reshape(-1, H).double()
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    ids, dy = ids[keep].long(), dy[keep]
    want = torch.zeros(V, H, dtype=torch.float64, device=dy.device).index_add_(0, ids, dy) * scale
    size = torch.zeros_like(want).index_add_(0, ids, dy.abs()) * abs(scale)
    n = torch.bincount(ids, minlength=V).view(V, 1)
    if start is not None:
        want, size = want + start.double() * (n > 0), size + start.double().abs()
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + (n + 3) * E * size + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134)
    err = (got.double() - want).abs()
    if start is not None:
        rest = (n == 0).view(-1)
        assert torch.equal(got[rest], start[rest])
        err[rest] = 0
    else:
        assert not bool(got[(n == 0).view(-1)].any())
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = [(1, 1, 1), (1, 50, 7), (2, 3, 64), (16, 1000, 2048), (33, 40, 129), (300, 77, 1000), (511, 90, 40), (512, 3000, 72), (513, 90, 40), (1025, 5000, 256),
         (4097, 300, 96), (9000, 70000, 40), (3001, 2, 2048), (20000, 1, 24),
         (100, 2 ** 23 + 5, 2), (3000, 2 ** 18 + 1, 4)]


@pytest.mark.parametrize("n,V,H", CASES)
@pytest.mark.parametrize("law", ["uniform", "rank", "one", "runs"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_against_64_bits(dev, n, V, H, law, dt):
    from usaf_b200 import embedding
    ids = tokens(dev, n, V, law, n)
    table = torch.empty(V, H, device=dev, dtype=dt).normal_(generator=gen(dev, 1))
    dy = torch.empty(n, H, device=dev, dtype=dt).normal_(generator=gen(dev, 2))
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    for scale in (1.0, 22.627):
        y = embedding.embedding(ids, table, scale, err=err)
        want = table.double()[ids] * scale
        assert bool(((y.double() - want).abs() <= want.abs() * (torch.finfo(dt).eps / 2 + E)).all())
        if scale == 1.0:
            assert torch.equal(y, table[ids])
        check_grad(embedding.embedding_backward(dy, ids, V, scale, err=err), dy, ids, V, scale)
    for g_dt in {dt, torch.float32}:
        start = torch.empty(V, H, device=dev, dtype=g_dt).normal_(generator=gen(dev, 3))
        got = embedding.embedding_backward(dy, ids, V, 0.5, padding_idx=V - 1, grad=start.clone(), err=err)
        check_grad(got, dy, ids, V, 0.5, V - 1, start)
    assert int(err) == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_ids_of_32_bits_shapes_and_repeats(dev, dt):
    from usaf_b200 import embedding
    V, H = 321, 520
    ids = tokens(dev, 4 * 700, V, "rank", 3).view(4, 700)
    table = torch.empty(V, H, device=dev, dtype=dt).normal_(generator=gen(dev, 1))
    dy = torch.empty(4, 700, H, device=dev, dtype=dt).normal_(generator=gen(dev, 2))
    y = embedding.embedding(ids.int(), table)
    assert y.shape == (4, 700, H) and torch.equal(y, table[ids])
    got = embedding.embedding_backward(dy, ids, V, 2.0, padding_idx=-V)
    check_grad(got, dy, ids, V, 2.0, 0)
    for _ in range(5):
        assert torch.equal(got, embedding.embedding_backward(dy, ids.int(), V, 2.0, padding_idx=0))
    # a transposed batch and a transposed gradient
    yt = embedding.embedding(ids.t(), table)
    assert torch.equal(yt, table[ids.t()])
    check_grad(embedding.embedding_backward(dy.transpose(0, 1), ids.t(), V), dy.transpose(0, 1), ids.t(), V, 1.0)


def test_many_tokens_in_order(dev):
    """More tokens than one pass of any part takes at once; rows of equal tokens
    are added in ascending position: 2^24 + 1 + ... in that order only."""
    from usaf_b200 import embedding
    n, V, H = 150000, 151936, 8
    ids = tokens(dev, n, V, "rank", 5)
    dy = torch.empty(n, H, device=dev).normal_(generator=gen(dev, 6))
    check_grad(embedding.embedding_backward(dy, ids, V), dy, ids, V, 1.0)
    a = torch.tensor([2.0 ** 24, 1.0, 1.0, -2.0 ** 24, 3.0], device=dev)
    ids = torch.tensor([4, 9, 4, 9, 4, 4, 9, 4], device=dev)
    dy = torch.zeros(8, 4, device=dev)
    dy[[0, 2, 4, 5, 7]] = a.view(-1, 1)
    want = torch.zeros((), device=dev)
    for v in a:
        want = want + v
    got = embedding.embedding_backward(dy, ids, 10)
    assert torch.equal(got[4], want.expand(4)) and float(want) == 3.0


def test_tokens_outside_the_table(dev):
    from usaf_b200 import embedding
    from usaf_b200._lib import ERR_BAD_INDEX
    V, H = 50, 96
    for dt in (torch.int64, torch.int32):
        ids = torch.tensor([3, -1, 49, 50, 7, -100, 2 ** 31 - 1, 3], device=dev, dtype=dt)
        table = torch.empty(V, H, device=dev).normal_(generator=gen(dev, 1))
        dy = torch.empty(8, H, device=dev).normal_(generator=gen(dev, 2))
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        y = embedding.embedding(ids, table, err=err)
        assert int(err) == ERR_BAD_INDEX
        ok = torch.tensor([0, 2, 4, 7], device=dev)
        assert torch.equal(y[ok], table[ids[ok].long()])
        y[ok] = 0
        assert not bool(y.any())
        err.zero_()
        got = embedding.embedding_backward(dy, ids, V, err=err)
        assert int(err) == ERR_BAD_INDEX
        check_grad(got, dy, ids, V, 1.0)
        assert torch.equal(got, embedding.embedding_backward(dy, ids, V))      # no error word: the same
    far = torch.tensor([2 ** 40 + 3, 3], device=dev)
    assert not bool(embedding.embedding(far, table)[0].any())
    assert torch.equal(embedding.embedding_backward(dy[:2], far, V)[3], dy[1])


def test_empty(dev):
    from usaf_b200 import embedding
    table = torch.ones(5, 8, device=dev)
    ids = torch.zeros(2, 0, dtype=torch.long, device=dev)
    assert embedding.embedding(ids, table).shape == (2, 0, 8)
    g = embedding.embedding_backward(torch.zeros(2, 0, 8, device=dev), ids, 5)
    assert g.shape == (5, 8) and not bool(g.any())
    # the zeros come after what ran before, a short sum just launched among it
    a = embedding.embedding_backward(torch.ones(1, 8, device=dev), ids.new_zeros(1), 5)
    b = embedding.embedding_backward(torch.zeros(2, 0, 8, device=dev), ids, 5)
    assert float(a.sum()) == 8.0 and not bool(b.any())
    start = torch.ones(5, 8, device=dev)
    assert torch.equal(embedding.embedding_backward(torch.zeros(2, 0, 8, device=dev), ids, 5, grad=start),
                       torch.ones(5, 8, device=dev))


def test_unaligned_and_around(dev):
    """A table, rows and a gradient at odd addresses; memory around the
    gradient keeps its values."""
    from usaf_b200 import embedding
    V, H, n = 60, 72, 500
    ids = tokens(dev, n, V, "rank", 1)
    table = torch.empty(V * H + 1, device=dev, dtype=torch.bfloat16).normal_(generator=gen(dev, 1))[1:].view(V, H)
    dy = torch.empty(n * H + 1, device=dev, dtype=torch.bfloat16).normal_(generator=gen(dev, 2))[1:].view(n, H)
    assert torch.equal(embedding.embedding(ids, table), table[ids])
    held = torch.full((V * H + 9,), 7.0, device=dev, dtype=torch.bfloat16)
    grad = held[1:V * H + 1].view(V, H)
    start = grad.clone()
    embedding.embedding_backward(dy, ids, V, grad=grad)
    check_grad(grad, dy, ids, V, 1.0, None, start)
    assert float(held[0]) == 7.0 and bool((held[V * H + 1:] == 7.0).all())


def test_autograd_streams_and_graph(dev):
    from usaf_b200 import embedding
    V, H, n = 700, 256, 3000
    ids = tokens(dev, n, V, "rank", 1)
    table = torch.empty(V, H, device=dev).normal_(generator=gen(dev, 1)).requires_grad_(True)
    dy = torch.empty(n, H, device=dev).normal_(generator=gen(dev, 2))
    embedding.embedding(ids, table, 3.0, padding_idx=0).backward(dy)
    check_grad(table.grad, dy, ids, V, 3.0, 0)
    # against a difference: the lookup is linear in the table
    d = torch.empty(V, H, device=dev).normal_(generator=gen(dev, 3))
    d[0] = 0
    num = (3.0 * d[ids].double() * dy.double()).sum()
    assert abs(float(num - (table.grad.double() * d.double()).sum())) <= \
        (n + 3) * E * 3.0 * float((d[ids].double() * dy.double()).abs().sum())
    want = embedding.embedding_backward(dy, ids, V)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = embedding.embedding_backward(dy, ids, V)
    side.synchronize()
    assert torch.equal(want, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = embedding.embedding_backward(dy, ids, V)
    ids.copy_(tokens(dev, n, V, "uniform", 9))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, embedding.embedding_backward(dy, ids, V))


@pytest.mark.parametrize("kept", [False, True])
def test_into_grad_of_lookups_on_other_streams(dev, kept):
    """The gradient is whole on the stream that backward() was called on, of two
    lookups on streams of their own and of the table's use beside them, also where
    an earlier graph keeps the leaf's accumulator on that stream."""
    from usaf_b200.embedding import embedding
    V, H = 1000, 256
    table = torch.randn(V, H, device=dev, generator=gen(dev, 1), requires_grad=True)
    table.grad = torch.ones_like(table)
    earlier = (table * 2).sum() if kept else None
    here = torch.cuda.current_stream(dev)
    loss, want = (table * 3).sum(), torch.full((V, H), 4.0, device=dev)
    for k in range(2):
        side = torch.cuda.Stream(dev)
        side.wait_stream(here)
        ids = tokens(dev, 500, V, "uniform", 2 + k)
        with torch.cuda.stream(side):
            y = embedding(ids, table, into_grad=True)
            y.register_hook(lambda g: torch.cuda._sleep(100_000_000))      # 50 ms, in front of the node
        here.wait_stream(side)
        loss = loss + y.sum()
        want += torch.bincount(ids, minlength=V).float()[:, None]         # whole numbers: exact
    loss.backward()
    got = table.grad.clone()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del earlier


def test_refusals(dev):
    from usaf_b200 import embedding
    table = torch.ones(5, 8, device=dev)
    ids = torch.zeros(3, dtype=torch.long, device=dev)
    dy = torch.ones(3, 8, device=dev)
    with pytest.raises(TypeError, match="ids"):
        embedding.embedding(ids.float(), table)
    with pytest.raises(ValueError, match="ids"):
        embedding.embedding(ids.cpu(), table)
    with pytest.raises(ValueError, match="contiguous"):
        embedding.embedding(ids, table.t())
    with pytest.raises(ValueError, match="rows, width"):
        embedding.embedding(ids, table[0])
    with pytest.raises(TypeError, match="unsupported dtype"):
        embedding.embedding(ids, table.double())
    with pytest.raises(ValueError, match="padding_idx"):
        embedding.embedding(ids, table, padding_idx=5)
    with pytest.raises(ValueError, match="err"):
        embedding.embedding(ids, table, err=torch.zeros(1, device=dev))
    with pytest.raises(ValueError, match="dout"):
        embedding.embedding_backward(dy[:2], ids, 5)
    with pytest.raises(ValueError, match="grad"):
        embedding.embedding_backward(dy, ids, 5, grad=torch.zeros(4, 8, device=dev))
    with pytest.raises(TypeError, match="grad"):
        embedding.embedding_backward(dy, ids, 5, grad=torch.zeros(5, 8, device=dev, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        embedding.embedding_backward(dy, ids, 5, grad=torch.zeros(8, 5, device=dev).t())
