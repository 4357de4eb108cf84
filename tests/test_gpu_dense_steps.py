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


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_are_counted_per_parameter(dev, bits):
    """A parameter whose gradients come late, or not always, takes the steps that
    it would take alone: bias corrections follow its own count."""
    from usaf_b200 import dense_optim
    shapes = {"always": (300,), "late": (70, 8), "gaps": (513,)}
    due = {"always": range(1, 8), "late": (5, 6, 7), "gaps": (1, 2, 5, 7)}
    gen = torch.Generator(device=dev).manual_seed(1)
    start = {n: torch.randn(s, device=dev, generator=gen) for n, s in shapes.items()}
    named = {n: parameter(t.clone()) for n, t in start.items()}
    alone = {n: parameter(t.clone()) for n, t in start.items()}
    opt = dense_optim.AdamW(named, lr=1e-2, state_bits=bits)
    opts = {n: dense_optim.AdamW({n: p}, lr=1e-2, state_bits=bits) for n, p in alone.items()}
    for t in range(1, 8):
        grads = {n: torch.randn(s, device=dev, generator=gen) for n, s in shapes.items() if t in due[n]}
        opt.step(grads)
        for n, g in grads.items():
            opts[n].step({n: g})
        assert all(torch.equal(named[n], alone[n]) for n in shapes), t
        if t == 5:      # the first step of a parameter: lr times the gradient's sign, and the decay
            move = (named["late"] - start["late"] * (1 - 1e-2 * 0.01)).abs()
            assert bool((move <= 1e-2 * (1 + 2.0 ** -18)).all()) and float(move.median()) > 0.99e-2
        if t == 6:      # counts travel with the state
            sd = opt.state_dict()
            assert sd["step"] == 6 and sd["steps"] == {"always": 6, "late": 2, "gaps": 3}
            opt = dense_optim.AdamW(named, lr=1e-2, state_bits=bits)
            opt.load_state_dict(sd)
    # a state without counts is one whose parameters took every step
    sd = opts["always"].state_dict()
    del sd["steps"]
    opts["always"].load_state_dict(sd)
    assert opts["always"].state_dict()["steps"] == {"always": 7}


def test_late_parameters_follow_torch(dev):
    """Against torch.optim.AdamW in 64 bits, gradients missing now and then: the update
    is a chain of ~24 fp32 operations on lr-sized values (24 E lr a step), the
    weight's own roundings 3 E |p| a step."""
    from usaf_b200 import dense_optim
    gen = torch.Generator(device=dev).manual_seed(2)
    start = [torch.randn(400, device=dev, generator=gen) for _ in range(3)]
    named = {str(i): parameter(t.clone()) for i, t in enumerate(start)}
    ref = [torch.nn.Parameter(t.double().clone()) for t in start]
    opt = dense_optim.AdamW(named, lr=1e-2, weight_decay=0.1)
    want = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    steps = 30
    for t in range(steps):
        grads = {}
        for i, p in enumerate(ref):
            p.grad = None
            if (t + 1) % (i + 1) == 0 and t >= 4 * i:
                g = torch.randn(400, device=dev, generator=gen) * torch.exp(torch.randn(400, device=dev, generator=gen))
                grads[str(i)], p.grad = g, g.double()
        opt.step(grads)
        want.step()
    for i, p in enumerate(ref):
        size = 1.0 + p.detach().abs() + steps * 1e-2
        # |update| <= 10 lr (Cauchy-Schwarz: m / (1 - b1^t) over the root of v is at most that)
        tol = steps * (24 * E * 10 * 1e-2 + 3 * E * size)
        assert bool(((named[str(i)].double() - p.detach()).abs() <= tol).all()), i


def same(a, b):
    """Equal values, NaN where the other has one."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0.0, 1e38, -1e38), b.nan_to_num(0.0, 1e38, -1e38))


@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("eps", [1e-8, 1e-20, 0.0])
@pytest.mark.parametrize("size", [1e-35, 1e-26, 1e-22, 1e-18, 1e-14, 1e-10, 1e8, 1e15, 1e17])
def test_8_bit_states_at_the_ends_of_the_range(dev, size, eps, master):
    """Second moments down to the smallest numbers (gradients of 1e-35 have none) and
    up to the largest, eps that does not hide the root: states as by the single
    operations, bit for bit, and the weights too where eps is small.  Else the step's
    quotient is within 2^-22 of itself (its reciprocal within 2^-23, a product and a
    sum, where the residual is too small to correct them), so a step moves the weight by
    2^-22 of its size u more or less, and two roundings of both weights are 2^-22 |p|.
    Weights start at zero, so that small steps show."""
    from test_gpu_dense_optim import Plain
    from usaf_b200 import dense_optim
    gen = torch.Generator(device=dev).manual_seed(5)
    n, dt = 3000, torch.bfloat16 if master else torch.float32
    p = torch.zeros(n, device=dev, dtype=dt)
    plain = Plain(p, 8, master)
    opt = dense_optim.AdamW({"w": parameter(p)}, lr=1e-2, eps=eps, state_bits=8, master_weights=master)
    tol, last = torch.full((n,), 2.0 ** -148, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    for t in (1, 2, 3):
        # values of one block 10 powers of e apart, some zeros; a block of zeros; the tail within a block
        g = size * torch.randn(n, device=dev, generator=gen) * torch.exp(3 * torch.randn(n, device=dev, generator=gen))
        g[torch.rand(n, device=dev, generator=gen) < 0.1] = 0
        g[512:768] = 0
        g.clamp_(-1e18, 1e18)          # v stays finite
        opt.step({"w": g})
        plain.step(g, t, 1e-2, 0.9, 0.999, eps, 0.01, 1.0)
        sd = opt.state_dict()
        got, want = (sd["master"]["w"], plain.master) if master else (p.cpu(), plain.p)
        if eps < 1e-8:
            assert same(got, want), t
        else:
            u = (want.double() - last * (1 - 1e-4)).abs()
            tol += 2.0 ** -22 * (u + want.double().abs())
            assert bool(((got.double() - want.double()).abs() <= tol).all()), t
        last = want.double()
        assert same(p.cpu(), got.to(dt))
        for k, (q, s) in (("m", plain.m), ("v", plain.v)):
            assert torch.equal(sd[k]["w"], q.view(torch.uint8)[:n]) and torch.equal(sd[k + "_scale"]["w"], s), (t, k)


def test_a_second_moment_beyond_the_range(dev):
    """A finite gradient whose square is not: that value takes no step (its root is
    infinite), stays finite, and its moment is kept as the largest there is."""
    from usaf_b200 import dense_optim
    for bits in (8, 32):
        p, g = torch.ones(2000, device=dev), torch.full((2000,), 1e-3, device=dev)
        q = p.clone()
        bad = g.clone()
        bad[600] = 1e22
        for w, first in ((p, g), (q, bad)):
            opt = dense_optim.AdamW({"w": parameter(w)}, state_bits=bits, weight_decay=0.0, lr=1e-2)
            opt.step({"w": first})
            if first is bad:
                assert float(w[600]) == 1.0
                if bits == 8:
                    assert 3e38 < float(opt.state("w")["v"][600]) < float("inf")
            opt.step({"w": g})
        assert bool(torch.isfinite(q).all())
        keep = torch.ones(2000, dtype=torch.bool, device=dev)
        keep[512:768] = bits == 32        # in 8 bits the block's other values have its scale
        keep[600] = False
        assert torch.equal(p[keep], q[keep])


# ---- 8-bit states over many steps -----------------------------------------------------
# A value's code may only stand for a part of a step (beta2 = 0.999 moves the root of v by
# 0.05 % at most while codes lie 6 to 12 % apart), so from the step on where the new
# gradient's weight (1 - b) / (1 - b^t) is below 1/8, the scaled value q between two codes
# becomes the upper one where its fraction and a number of the step and the place, spread
# evenly over [0, 1), reach 1.

def reversed16(x):
    for a, b in ((0x5555, 1), (0x3333, 2), (0x0f0f, 4), (0x00ff, 8)):
        x = (x & a) << b | (x >> b) & a
    return x


def spread_numbers(n, t, lo, hi):
    return numbers_at(torch.arange(n), t, lo, hi)


def numbers_at(i, t, lo, hi):
    """The numbers of a step's values at places i, in 2^-16."""
    h = (i // 4) * 0x9E3779B1 & 0xffffffff      # places of up to 2^32 here: no overflow of 64 bits
    h = h ^ h >> 15
    h = h ^ ((t * lo & 0xffff) | (t * hi & 0xffff) << 16)
    half = torch.where(i % 4 < 2, h & 0xffff, h >> 16)
    return torch.where(i % 2 == 0, half, reversed16(half))


def pack_spread(x, least, numbers):
    """Codes and scales, as test_gpu_dense_optim.pack but for the rounding."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    live = top >= 1e-30
    q = (b * torch.where(live, (1 / top) * 448.0, 0.0)).view(-1)
    if least:
        q = torch.maximum(q, torch.where((b > 0) & live, 2.0 ** -9, 0.0).view(-1))
    size = q.abs().double()
    step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)
    low = torch.floor(size / step)
    code = (low + ((size / step - low) + numbers / 65536.0 >= 1)) * step
    code = torch.copysign(code.clamp_max(448.0), q.double()).float().to(torch.float8_e4m3fn)
    return code, torch.where(live, top * torch.tensor(1 / 448.0, dtype=torch.float32), 0.0).view(-1)


@pytest.mark.parametrize("dt,master", [(torch.float32, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("b1", [0.9, 0.98])
def test_codes_bit_for_bit_over_many_steps(dev, dt, master, b1):
    """States of 24 steps, nearest codes first, then spread: bit for bit, in whole blocks
    and in a tensor's tail, wherever the tensor lies in the buffers.  (The weights may
    differ by the last bit of the step's quotient; the states do not depend on them.)"""
    import test_gpu_dense_optim as plain_form
    from usaf_b200 import dense_optim
    gen = torch.Generator(device=dev).manual_seed(9)
    sizes, b2 = (1, 255, 256, 5000, 8192), 0.98
    params = [(torch.randn(n, device=dev, generator=gen)).to(dt) for n in sizes]
    plain = [plain_form.Plain(p, 8, master) for p in params]
    opt = dense_optim.AdamW({str(i): parameter(p) for i, p in enumerate(params)}, betas=(b1, b2), state_bits=8,
                            master_weights=master)
    spread = 0
    for t in range(1, 25):
        grads = [(1e-3 * torch.randn(n, device=dev, generator=gen)
                  * torch.exp(2 * torch.randn(n, device=dev, generator=gen))).to(dt) for n in sizes]
        if t == 20:
            grads = [g * 0 for g in grads]
        opt.step({str(i): g for i, g in enumerate(grads)})
        sd = opt.state_dict()
        kept = plain_form.pack
        for i, (pl, g) in enumerate(zip(plain, grads)):
            n = -(-sizes[i] // BLOCK) * BLOCK

            def pack(x, least):
                b, lo, hi = (b2, 0x9E37, 0xC13F) if least else (b1, 0x91E1, 0x9E37)
                if (1 - b) / (1 - b ** t) >= 0.125:
                    return kept(x, least)
                return pack_spread(x, least, spread_numbers(n, t, lo, hi))

            plain_form.pack = pack
            try:
                pl.step(g, t, 1e-4, b1, b2, 1e-8, 0.01, 1.0)
            finally:
                plain_form.pack = kept
            for k, (q, s) in (("m", pl.m), ("v", pl.v)):
                assert torch.equal(sd[k][str(i)], q.view(torch.uint8)[:sizes[i]]), (t, i, k)
                assert torch.equal(sd[k + "_scale"][str(i)], s), (t, i, k)
        spread += (1 - b2) / (1 - b2 ** t) < 0.125
    assert spread == 16


@pytest.mark.parametrize("case", ["stationary", "falls", "stops"])
def test_the_second_moment_follows_beta2(dev, case):
    """sqrt(v) in 8 bits beside 32 after thousands of steps with beta2 = 0.999, also where
    the gradients of every other value of a block fall 30-fold, or stop.

    The mean of the ratios is 1 within 0.15: a rounding is right in the mean, and its variance
    (p (1 - p) s^2 with p s = x / 2000 a step's move, s <= x / 8) adds at most x s / 2000 a step
    to the mean of x^2, which decays by x^2 / 1000: 1/16 of x^2 in equilibrium and 1/32 of x,
    and as much again on the way down; sampling noise of 8192 values at most 60 % wide is
    0.7 %.  The spread is sqrt(s / 2x) = 0.25 of a value in equilibrium, so 5 % to 95 % lie
    within 0.4 of the median; on the way down it doubles at most."""
    from usaf_b200 import dense_optim
    n = 16384
    gen = torch.Generator(device=dev).manual_seed(11)
    size = torch.exp(0.7 * torch.randn(n, device=dev, generator=gen))
    other = torch.ones(n, device=dev)
    other[::2] = {"stationary": 1.0, "falls": 1 / 30, "stops": 0.0}[case]
    opts = [dense_optim.AdamW({"w": parameter(torch.zeros(n, device=dev))}, lr=0.0, weight_decay=0.0, state_bits=bits)
            for bits in (32, 8)]
    for t in range(6000):
        g = size * torch.randn(n, device=dev, generator=gen)
        if t >= 2000:
            g *= other
        for opt in opts:
            opt.step({"w": g})
    want, got = (opt.state("w")["v"].sqrt() for opt in opts)
    ratio = (got / want).double()
    for part in (ratio[::2], ratio[1::2]):
        assert abs(float(part.mean()) - 1) <= 0.15, float(part.mean())
        lo, mid, hi = (float(torch.quantile(part, q)) for q in (0.05, 0.5, 0.95))
        wide = 0.4 if case == "stationary" else 0.8
        assert 1 - wide <= lo and hi <= 1 + wide and abs(mid - 1) <= 0.25, (lo, mid, hi)


def test_the_first_moment_follows_beta1(dev):
    """beta1 = 0.99 moves m by 1 % of its way a step: constant gradients are reached, and
    where they stop (beside others of the block that go on) m goes to zero.  The mean of
    8192 values, each within 25 % of the mean it has in equilibrium: 1 % and a half for
    what of the start is left (0.99^800); afterwards 0.99^1500 = 3e-7 of it and
    roundings of the lowest codes, 2^-9 of 448 of the block's largest (3e-6)."""
    from usaf_b200 import dense_optim
    n = 16384
    g = torch.exp(0.5 * torch.randn(n, device=dev, generator=torch.Generator(device=dev).manual_seed(12)))
    g[1::4] *= -1
    opt = dense_optim.AdamW({"w": parameter(torch.zeros(n, device=dev))}, lr=0.0, betas=(0.99, 0.999), state_bits=8)
    for _ in range(800):
        opt.step({"w": g})
    ratio = (opt.state("w")["m"] / g).double()
    assert abs(float(ratio.mean()) - 1) <= 0.015 and float(ratio.min()) > 0.2, (float(ratio.mean()), float(ratio.min()))
    half = g.clone()
    half[::2] = 0
    for _ in range(1500):
        opt.step({"w": half})
    m = opt.state("w")["m"].abs()
    assert float(m[::2].mean()) <= 1e-5 * float(m.max()), float(m[::2].mean() / m.max())


def test_long_runs_of_blocks(dev):
    """A tensor so large that a warp steps 16 blocks one after another: as in parts of
    which each block has a warp, also where blocks in between are at the ends of the
    range; and the spread codes of its blocks are those of their places."""
    import test_gpu_dense_optim as plain_form
    from usaf_b200 import dense_optim
    n = 256 * 480000                     # 123 M values
    gen = torch.Generator(device=dev).manual_seed(21)
    p = torch.empty(n, device=dev, dtype=torch.bfloat16).normal_(generator=gen)
    g = torch.empty(n, device=dev, dtype=torch.bfloat16).normal_(0, 1e-3, generator=gen)
    kind = torch.randint(0, 8, (n // 256, 1), device=dev, generator=gen)
    g = (g.view(-1, 256) * torch.where(kind == 0, 1e-20, torch.where(kind == 1, 1e24, torch.where(kind == 2, 0.0, 1.0)))
         ).to(torch.bfloat16).view(-1)

    def states(k):
        return [(torch.zeros(k, dtype=torch.float8_e4m3fn, device=dev), torch.zeros(k // 256, device=dev)) for _ in range(2)]

    def bits(ms):
        return [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for pair in ms for t in pair]

    q, whole = p.clone(), states(n)
    dense_optim.adamw_step([q], [g], *whole, step=1, lr=1e-2)
    part = 256 * 12000
    for a in range(0, n, part):
        r, st = p[a:a + part].clone(), states(part)
        dense_optim.adamw_step([r], [g[a:a + part]], *st, step=1, lr=1e-2)
        assert torch.equal(q[a:a + part], r)
        for t, w, width in zip(bits(st), bits(whole), (256, 1, 256, 1)):
            assert torch.equal(w[a // 256 * width:(a + part) // 256 * width], t)
    assert bool(torch.isfinite(q.float()).all())
    # a late step: 400 blocks anywhere, operation by operation
    before = [t.clone() for t in bits(whole)]
    dense_optim.adamw_step([q], [g], *whole, step=1000, lr=1e-2)
    pick = torch.randperm(n // 256, generator=torch.Generator().manual_seed(3))[:400].sort().values
    at = (pick.view(-1, 1) * 256 + torch.arange(256)).view(-1)
    on = at.to(dev)
    pl = plain_form.Plain(p[on], 8, False)
    pl.m, pl.v = ((before[i][on].cpu().view(torch.float8_e4m3fn), before[i + 1][pick.to(dev)].cpu()) for i in (0, 2))
    kept = plain_form.pack
    plain_form.pack = lambda x, least: pack_spread(
        x, least, numbers_at(at, 1000, *((0x9E37, 0xC13F) if least else (0x91E1, 0x9E37))))
    try:
        pl.step(g[on], 1000, 1e-2, 0.9, 0.999, 1e-8, 0.0, 1.0)
    finally:
        plain_form.pack = kept
    after = bits(whole)
    # (blocks of infinite moments have scales that the plain form does not bound)
    fine = ((kind[pick.to(dev), 0] != 1).cpu()).repeat_interleave(256)
    assert int(fine.sum()) > 300 * 256
    for i, (codes, scales) in ((0, pl.m), (2, pl.v)):
        assert torch.equal(after[i][on].cpu()[fine], codes.view(torch.uint8)[fine])
        assert torch.equal(after[i + 1][pick.to(dev)].cpu()[fine[::256]], scales[fine[::256]])
