"""The order in which the embedding's gradient adds equal tokens' rows, bit for
bit: the stable sort by token, chunks of 32 sorted positions added one after
another, a token's chunks added in order (of more than 17, eight contiguous
parts first).  Another order of any two rows gives other bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CHUNK = 32


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import usaf_b200  # noqa: F401
    return torch.device("cuda:0")


def in_order(rows):
    total = torch.zeros(rows.shape[1])
    for r in rows:
        total = total + r
    return total


def expected(dy, ids, V):
    """fp32 additions on the CPU, each rounded by itself as on the device."""
    out = torch.zeros(V, dy.shape[1])
    place = torch.argsort(ids, stable=True)
    tokens, counts = torch.unique_consecutive(ids[place], return_counts=True)
    a = 0
    for token, n in zip(tokens.tolist(), counts.tolist()):
        parts, i = [], a
        while i < a + n:
            e = min(a + n, i // CHUNK * CHUNK + CHUNK)
            parts.append(in_order(dy[place[i:e]]))
            i = e
        if len(parts) > 17:
            each = -(-len(parts) // 8)
            parts = [in_order(torch.stack(parts[k:k + each])) for k in range(0, len(parts), each)]
        out[token] = in_order(torch.stack(parts))
        a += n
    return out


@pytest.mark.parametrize("n,V", [(600, 7), (5000, 90), (5000, 3), (20000, 1), (9000, 70000), (3000, 2 ** 18 + 1)])
def test_rows_are_added_in_their_order(dev, n, V):
    from usaf_b200 import embedding
    g = torch.Generator().manual_seed(n + V)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    ids = (float(V) ** u).long().clamp_(1, V) - 1
    if V > 2 ** 17:
        ids = ids % 50 * (V // 50) + (ids > 0)         # equal tokens that differ in the high digits
    H = 4
    dy = torch.randn(n, H, generator=g) * torch.exp(3 * torch.randn(n, 1, generator=g))
    want = expected(dy, ids, V)
    got = embedding.embedding_backward(dy.to(dev), ids.to(dev), V).cpu()
    assert torch.equal(got, want)
    # the test itself: the same rows of one token in another order show
    swapped = dy.clone()
    token = ids.mode().values
    at = (ids == token).nonzero().view(-1)
    order = at[torch.randperm(len(at), generator=g)]
    swapped[at] = dy[order]
    assert not torch.equal(expected(swapped, ids, V), want)
