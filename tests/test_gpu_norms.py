"""RMS norm and its backward pass (usaf_b200.norms) against the formulas in 64
bits, from one row to many, odd and wide rows, strided rows, each type.

Tolerances, with u = finfo(type).eps / 2 (one rounding) and e = 2^-24:
* y = s r w: r carries the error of the sum of squares (a chain of at most
  H/32 + 32 additions of positive values, halved by the root) and of a division,
  a root and a reciprocal; then two products and the last rounding:
  |y| (u + (H/32 + 40) e);
* dx = r (g - hat c) + dsum: the same for each term, no smaller than the terms
  it is the difference of: u |dx| + (H/32 + 60) e (r |g| + r |hat| mean|g hat| + |dsum|);
* dw: rows + 60 additions at most: u |dw| + (rows + H/32 + 60) e sum|dy hat|;
* values below the type's normal range: half of its smallest step.
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


def small(dt):
    """Half of the type's smallest step."""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dt]


def rand(dev, seed, *shape):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))


def inputs(dev, rows, H, dt, wdt, seed=0):
    x = (rand(dev, seed, rows, H) * torch.exp(rand(dev, seed + 1, rows, 1))).to(dt)
    res = rand(dev, seed + 2, rows, H).to(dt)
    w = (1 + 0.3 * rand(dev, seed + 3, H)).to(wdt)
    dy, dsum = rand(dev, seed + 4, rows, H).to(dt), rand(dev, seed + 5, rows, H).to(dt)
    return x, res, w, dy, dsum


def close(name, got, want, tol, dt):
    err = (got.double() - want).abs()
    bad = ~(err <= tol + small(dt))
    assert not bool(bad.any()), (name, float((err / (tol + small(dt))).max()), int(bad.sum()))


def check(total, w, y, rstd, eps, dy=None, dsum=None, dx=None, dw=None):
    """``total`` is the stored sum (or x): everything after it in 64 bits."""
    dt, wdt, (rows, H) = y.dtype, w.dtype, y.shape
    u, uw = torch.finfo(dt).eps / 2, torch.finfo(wdt).eps / 2
    s, wd = total.double(), w.double()
    r = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    k = (H / 32 + 40) * E
    want = s * r * wd
    close("y", y, want, want.abs() * (u + k), dt)
    if rstd is not None:
        close("rstd", rstd.view(-1, 1), r, r * k, torch.float32)
    if dx is None:
        return
    g, hat = dy.double() * wd, s * r
    c = (g * hat).mean(1, keepdim=True)
    size = r * g.abs() + r * hat.abs() * (g * hat).abs().mean(1, keepdim=True)
    want = r * (g - hat * c)
    if dsum is not None:
        want, size = want + dsum.double(), size + dsum.double().abs()
    close("dx", dx, want, u * want.abs() + (k + 20 * E) * size, dt)
    if dw is not None:
        t = dy.double() * hat
        want = t.sum(0)
        close("dw", dw, want, uw * want.abs() + (rows * E + k + 20 * E) * t.abs().sum(0), wdt)


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32)]
SIZES = [(1, 1), (1, 2048), (3, 7), (700, 4), (513, 8), (300, 16), (77, 24), (9, 72), (5, 128), (4099, 35), (777, 61), (515, 131), (130, 2050), (1, 35), (8, 771), (9, 771), (1000, 128), (17, 771), (33, 1000), (300, 2048), (700, 520),
         (9, 6144), (65, 8192), (4, 9000), (3, 16384), (2, 32768), (2, 32767)]


@pytest.mark.parametrize("rows,H", SIZES)
@pytest.mark.parametrize("dt,wdt", TYPES)
def test_against_64_bits(dev, rows, H, dt, wdt):
    from usaf_b200 import norms
    x, res, w, dy, dsum = inputs(dev, rows, H, dt, wdt, rows + H)
    y, rstd, total = norms.rms_norm_forward(x, w, 1e-6)
    assert total is x
    dx, dw = norms.rms_norm_backward(dy, x, w, rstd)
    assert dw.dtype == wdt
    check(x, w, y, rstd, 1e-6, dy, None, dx, dw)
    # with the residual addition: the sum is rounded once, the norm is the rounded sum's
    y, rstd, total = norms.rms_norm_forward(x, w, 1e-3, residual=res)
    assert torch.equal(total, (x.float() + res.float()).to(dt))
    dx, dw = norms.rms_norm_backward(dy, total, w, rstd, dsum=dsum)
    check(total, w, y, rstd, 1e-3, dy, dsum, dx, dw)
    # without the weight's gradient: the same dx
    dx2, none = norms.rms_norm_backward(dy, total, w, rstd, dsum=dsum, want_dw=False)
    assert none is None and torch.equal(dx2, dx)


@pytest.mark.parametrize("rows,H", [(70000, 128), (20011, 96), (5000, 2048), (3001, 771), (1500, 6144), (50001, 35), (9001, 131)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_many_rows_repeat_bit_for_bit(dev, rows, H, dt):
    from usaf_b200 import norms
    x, _, w, dy, _ = inputs(dev, rows, H, dt, dt, 5)
    y, rstd, _ = norms.rms_norm_forward(x, w)
    dx, dw = norms.rms_norm_backward(dy, x, w, rstd)
    check(x, w, y, rstd, 1e-6, dy, None, dx, dw)
    for _ in range(5):
        y2, r2, _ = norms.rms_norm_forward(x, w)
        dx2, dw2 = norms.rms_norm_backward(dy, x, w, rstd)
        assert torch.equal(y, y2) and torch.equal(rstd, r2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("H,step,skip", [(128, 136, 0), (128, 131, 3), (2048, 2064, 8), (768, 2304, 768), (40, 41, 1)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_rows(dev, H, step, skip, dt):
    """Rows that are a slice of wider ones, at any offset, and rows of stride 0
    (an expanded gradient): what lies around them is not touched or read."""
    from usaf_b200 import norms
    rows = 37
    wide = [torch.full((rows, step + skip), float("nan"), device=dev, dtype=dt) for _ in range(3)]
    x, res, dy = (t[:, skip:skip + H] for t in wide)
    for i, t in enumerate((x, res, dy)):
        t.copy_(rand(dev, i, rows, H))
    w = (1 + 0.3 * rand(dev, 9, H + 1))[1:].to(dt)      # an odd address
    y, rstd, total = norms.rms_norm_forward(x, w, residual=res)
    dx, dw = norms.rms_norm_backward(dy, total, w, rstd, dsum=dy)
    check(total, w, y, rstd, 1e-6, dy, dy, dx, dw)
    y, rstd, _ = norms.rms_norm_forward(x, w)
    one = dy[:1].expand(rows, H)
    dx, dw = norms.rms_norm_backward(one, x, w, rstd)
    check(x, w, y, rstd, 1e-6, one, None, dx, dw)
    # transposed rows are copied
    xt = rand(dev, 4, H, rows).to(dt).t()
    y, rstd, _ = norms.rms_norm_forward(xt, w)
    check(xt, w, y, rstd, 1e-6)


def test_leading_dimensions_and_empty(dev):
    from usaf_b200 import norms
    x, _, w, dy, _ = inputs(dev, 24, 128, torch.bfloat16, torch.bfloat16)
    y, rstd, _ = norms.rms_norm_forward(x, w)
    y4 = norms.rms_norm(x.view(2, 3, 4, 128), w)
    assert y4.shape == (2, 3, 4, 128) and torch.equal(y4.view(24, 128), y)
    heads = torch.randn(6, 4, 2, 128, device=dev, dtype=torch.bfloat16)[:, :, 1]      # [6, 4, 128], one stride
    check(heads.reshape(24, 128), w, norms.rms_norm(heads, w).view(24, 128), None, 1e-6)
    assert torch.equal(norms.rms_norm(x[0], w), y[0])
    e = x[:0]
    y0, r0, _ = norms.rms_norm_forward(e, w)
    dx0, dw0 = norms.rms_norm_backward(e, e, w, r0)
    assert y0.shape == dx0.shape == (0, 128) and r0.numel() == 0 and not bool(dw0.any())


def test_rows_of_zeros_and_of_bad_values(dev):
    """A row of zeros is zeros; infinities and NaN stay in their rows."""
    from usaf_b200 import norms
    for H in (128, 771, 2048):
        x, _, w, dy, _ = inputs(dev, 64, H, torch.bfloat16, torch.bfloat16, 3)
        clean, r0, _ = norms.rms_norm_forward(x, w)
        dx0, _ = norms.rms_norm_backward(dy, x, w, r0)
        x[5] = 0
        x[9, H // 2] = float("nan")
        x[11, 3] = float("inf")
        y, rstd, _ = norms.rms_norm_forward(x, w)
        dx, _ = norms.rms_norm_backward(dy, x, w, rstd)
        keep = torch.ones(64, dtype=torch.bool, device=dev)
        keep[[5, 9, 11]] = False
        assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], dx0[keep])
        assert not bool(y[5].any()) and bool(torch.isfinite(dx[5]).all())
        assert bool(torch.isnan(y[9]).all())


@pytest.mark.parametrize("H", [128, 771, 2048, 40000 // 8])
def test_rows_near_the_ends_of_the_range(dev, H):
    """Rows of 1e-20 with their rstd of 1e20, and of 1e15: no intermediate value
    leaves the range that the result has."""
    from usaf_b200 import norms
    w, dy = 1 + 0.3 * rand(dev, 1, H), rand(dev, 2, 6, H)
    x = rand(dev, 3, 6, H) * torch.tensor([1e-20, 1e-17, 1e-10, 1.0, 1e10, 1e15], device=dev).view(6, 1)
    rstd = (1 / x.double().square().mean(1).sqrt()).float()
    dx, dw = norms.rms_norm_backward(dy, x, w, rstd)
    r = rstd.double().view(6, 1)
    g, hat = dy.double() * w.double(), x.double() * r
    c = (g * hat).mean(1, keepdim=True)
    tol = (H / 32 + 60) * E * r * (g.abs() + hat.abs() * (g * hat).abs().mean(1, keepdim=True))
    assert bool(((dx.double() - r * (g - hat * c)).abs() <= tol).all())
    t = dy.double() * hat
    assert bool(((dw.double() - t.sum(0)).abs() <= (66 + H / 32) * E * t.abs().sum(0)).all())


def test_autograd_and_differences(dev):
    """The gradients of the differentiable form against the formulas' and
    against central differences of the 64-bit function."""
    from usaf_b200 import norms
    rows, H = 19, 384
    x, res, w, dy, dsum = inputs(dev, rows, H, torch.float32, torch.float32, 8)
    for t in (x, res, w):
        t.requires_grad_(True)
    y, total = norms.rms_norm(x, w, 1e-5, residual=res)
    ((y * dy).sum() + (total * dsum).sum()).backward()
    check(total.detach(), w.detach(), y.detach(), None, 1e-5, dy, dsum, x.grad, w.grad)
    assert torch.equal(x.grad, res.grad)

    def f(xd, wd):
        s = xd + res.detach().double()
        return ((s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5) * wd) * dy.double()).sum() \
            + (s * dsum.double()).sum()

    xd, wd = x.detach().double(), w.detach().double()
    h = 1e-5
    for k in range(3):
        d = rand(dev, 20 + k, rows, H).double()
        num = (f(xd + h * d, wd) - f(xd - h * d, wd)) / (2 * h)
        # fp32 gradients: (H/32 + 60) e of each term's size; the difference's own error is O(h^2)
        assert abs(float(num - (x.grad.double() * d).sum())) <= 1e-5 * float((x.grad.double() * d).abs().sum())
        d = rand(dev, 30 + k, H).double()
        num = (f(xd, wd + h * d) - f(xd, wd - h * d)) / (2 * h)
        assert abs(float(num - (w.grad.double() * d).sum())) <= 1e-5 * float((w.grad.double() * d).abs().sum())
    # frozen weight: no gradient for it, the same for x
    x2, w2 = x.detach().clone().requires_grad_(True), w.detach()
    y2, t2 = norms.rms_norm(x2, w2, 1e-5, residual=res.detach())
    ((y2 * dy).sum() + (t2 * dsum).sum()).backward()
    assert torch.equal(x2.grad, x.grad) and w2.grad is None
    # only the norm is used, or only the sum
    x4 = x.detach().clone().requires_grad_(True)
    w4 = w.detach().clone().requires_grad_(True)
    y4, t4 = norms.rms_norm(x4, w4, 1e-5, residual=res.detach())
    (y4 * dy).sum().backward()
    check(t4.detach(), w4.detach(), y4.detach(), None, 1e-5, dy, None, x4.grad, w4.grad)
    x3 = x.detach().clone().requires_grad_(True)
    _, t3 = norms.rms_norm(x3, w2, 1e-5, residual=res.detach())
    (t3 * dsum).sum().backward()
    assert torch.equal(x3.grad, dsum)
    with pytest.raises(RuntimeError):       # no second derivatives: refused, not wrong
        g, = torch.autograd.grad((norms.rms_norm(x4, w4) * dy).sum(), x4, create_graph=True)
        g.sum().backward()


def test_other_stream_and_graph(dev):
    """On a stream of its own, and captured with other inputs at the replay."""
    from usaf_b200 import norms
    x, res, w, dy, dsum = inputs(dev, 130, 2048, torch.bfloat16, torch.bfloat16, 12)

    def step():
        y, rstd, total = norms.rms_norm_forward(x, w, residual=res)
        return (y, total, *norms.rms_norm_backward(dy, total, w, rstd, dsum=dsum))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(rand(dev, 77, 130, 2048))
    dy.copy_(rand(dev, 78, 130, 2048))
    for _ in range(3):
        graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_refusals(dev):
    from usaf_b200 import norms
    from usaf_b200._lib import UsafError
    x, _, w, dy, _ = inputs(dev, 4, 64, torch.bfloat16, torch.bfloat16)
    y, rstd, _ = norms.rms_norm_forward(x, w)
    with pytest.raises(ValueError, match="shape"):
        norms.rms_norm(x, w[:32])
    with pytest.raises(TypeError, match="weight"):
        norms.rms_norm(x, w.half())
    with pytest.raises(TypeError, match="unsupported dtype"):
        norms.rms_norm(x.double(), w.double())
    with pytest.raises(ValueError, match="contiguous"):
        norms.rms_norm(x, torch.ones(128, device=dev, dtype=torch.bfloat16)[::2])
    with pytest.raises(ValueError, match="device"):
        norms.rms_norm(x, w.cpu())
    with pytest.raises(TypeError, match="residual"):
        norms.rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError, match="residual"):
        norms.rms_norm(x, w, residual=x[:2])
    with pytest.raises(ValueError, match="eps"):
        norms.rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="at most"):
        norms.rms_norm(torch.zeros(1, 32769, device=dev), torch.ones(32769, device=dev))
    with pytest.raises(ValueError, match="rstd"):
        norms.rms_norm_backward(dy, x, w, rstd[:3])
    with pytest.raises(ValueError, match="dy"):
        norms.rms_norm_backward(dy[:3], x, w, rstd)
    assert issubclass(UsafError, RuntimeError)
