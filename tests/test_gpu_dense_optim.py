"""AdamW over many tensors (usaf_b200.dense_optim).

* against the same fp32 operations done one by one by torch on the CPU: each
  is correctly rounded there and on the device, so every output is equal bit
  for bit, states in 32 and in 8 bits, over several steps;
* against the formulas in 64 bits: with e = 2^-24, m and v are two products
  (three) and an addition of rounded constants, 6 e of the terms' sizes; the
  step is a root, two products, a division and two additions more, 24 e of
  lr |update| and 3 e of |p|; then the parameter's rounding.
"""
import math

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


def pack(x, least):
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    live = top >= 1e-30
    q = (b * torch.where(live, (1 / top) * 448.0, 0.0)).to(torch.float8_e4m3fn)
    if least:
        q = torch.where((q.float() == 0) & (b > 0) & live, 2.0 ** -9, q.float()).to(torch.float8_e4m3fn)
    return q.view(-1), torch.where(live, top * torch.tensor(1 / 448.0, dtype=torch.float32), 0.0).view(-1)


def f32(v):
    return torch.tensor(v, dtype=torch.float32)


class Plain:
    """One tensor's step, operation by operation in fp32 on the CPU."""

    def __init__(self, p, bits, master):
        self.p, self.bits, n = p.cpu().clone(), bits, -(-p.numel() // BLOCK) * BLOCK
        self.master = p.cpu().float().reshape(-1) if master else None
        self.m, self.v = torch.zeros(n), torch.zeros(n)
        if bits == 8:
            self.m, self.v = pack(self.m, False), pack(self.v, True)

    def step(self, g, t, lr, b1, b2, eps, wd, div):
        n = self.p.numel()
        g = torch.cat([g.cpu().float().reshape(-1), torch.zeros(-n % BLOCK)]) * f32(1 / div)
        p = self.master if self.master is not None else self.p.float().reshape(-1)
        if self.bits == 8:
            m, r = (((q.float().view(-1, BLOCK)) * s.view(-1, 1)).view(-1) for q, s in (self.m, self.v))
            v = r * r
        else:
            m, v = self.m, self.v
        m = m * f32(b1) + g * f32(1 - b1)
        v = v * f32(b2) + (g * f32(1 - b2)) * g
        # torch's fp32 root on the CPU is not always the nearest value; the 64-bit one, rounded, is
        root = torch.sqrt(v.double()).float()
        up = m / (root * f32(1 / math.sqrt(1 - b2 ** t)) + f32(eps))
        p = p * f32(1 - lr * wd) - up[:n] * f32(lr / (1 - b1 ** t))
        if self.master is not None:
            self.master = p
        self.p = p.to(self.p.dtype).view(self.p.shape)
        self.m, self.v = (pack(m, False), pack(root, True)) if self.bits == 8 else (m, v)


def tensors(dev, shapes, dt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(s, device=dev, generator=g) * 0.05).to(dt) for s in shapes]


def gradients(dev, shapes, dt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for s in shapes:
        t = torch.randn(s, device=dev, generator=g) * torch.exp(2 * torch.randn(s, device=dev, generator=g)) * 1e-3
        out.append(torch.where(torch.rand(s, device=dev, generator=g) < 0.1, 0.0, t).to(dt))
    return out


SHAPES = [(1,), (255,), (256,), (257,), (128, 96), (3, 5, 7), (0,), (1000, 77), (2048,), (4099,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt,gdt,master", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, True),
                                           (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, True),
                                           (torch.float16, torch.float16, True), (torch.float16, torch.float32, False)])
def test_bit_for_bit(dev, bits, dt, gdt, master):
    from usaf_b200 import dense_optim
    params = tensors(dev, SHAPES, dt, 1)
    plain = [Plain(p, bits, master) for p in params]
    opt = dense_optim.AdamW({str(i): torch.nn.Parameter(p, requires_grad=False) for i, p in enumerate(params)},
                            lr=3e-3, betas=(0.9, 0.98), eps=1e-7, weight_decay=0.1, no_decay=("2", "7"),
                            state_bits=bits, master_weights=master)
    for t in range(1, 5):
        grads = gradients(dev, SHAPES, gdt, 10 + t)
        if t == 3:
            grads = [g * 0 for g in grads]       # a step of zeros
        opt.step({str(i): g for i, g in enumerate(grads)}, grad_div=6.0)
        for i, (pl, g) in enumerate(zip(plain, grads)):
            pl.step(g, t, 3e-3, 0.9, 0.98, 1e-7, 0.0 if i in (2, 7) else 0.1, 6.0)
        sd = opt.state_dict()
        for i, pl in enumerate(plain):
            n, k = pl.p.numel(), str(i)
            assert torch.equal(params[i].cpu(), pl.p), (t, i)
            if master:
                assert torch.equal(sd["master"][k], pl.master), (t, i)
            if bits == 8:
                for nm, (q, s) in (("m", pl.m), ("v", pl.v)):
                    assert torch.equal(sd[nm][k], q.view(torch.uint8)[:n]), (t, i, nm)
                    assert torch.equal(sd[nm + "_scale"][k], s), (t, i, nm)
            else:
                assert torch.equal(sd["m"][k], pl.m[:n]) and torch.equal(sd["v"][k], pl.v[:n]), (t, i)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 700, 100003])
def test_against_64_bits(dev, bits, n):
    from usaf_b200 import dense_optim
    (p,), (g,) = tensors(dev, [(n,)], torch.float32, 2), gradients(dev, [(n,)], torch.float32, 3)
    opt = dense_optim.AdamW({"w": torch.nn.Parameter(p, requires_grad=False)}, lr=1e-2, weight_decay=0.05,
                            state_bits=bits)
    for t in range(1, 4):
        st, p0 = opt.state("w"), p.double()
        m = 0.9 * st["m"].double() + 0.1 * g.double()
        v = 0.999 * st["v"].double() + 0.001 * g.double().square()
        msize = 0.9 * st["m"].double().abs() + 0.1 * g.double().abs()
        den = torch.sqrt(v / (1 - 0.999 ** t)) + 1e-8
        up, usize = (x / (1 - 0.9 ** t) / den for x in (m, msize))
        want = p0 * (1 - 1e-2 * 0.05) - 1e-2 * up
        opt.step({"w": g})
        assert bool(((p.double() - want).abs() <= 24 * E * 1e-2 * usize + 3 * E * p0.abs() + 2.0 ** -140).all())
        new = opt.state("w")
        if bits == 32:
            assert bool(((new["m"].double() - m).abs() <= 6 * E * msize + 2.0 ** -140).all())
            assert bool(((new["v"].double() - v).abs() <= 6 * E * v + 2.0 ** -140).all())
        else:
            # e4m3: half a step of 2^-4 of the value, or of 2^-9 of the block's largest / 448; the lowest
            # code in place of zero for the root
            def top(x):
                b = torch.cat([x.abs(), x.new_zeros(-n % BLOCK)]).view(-1, BLOCK).amax(1)
                return b.repeat_interleave(BLOCK)[:n] / 448
            assert bool(((new["m"].double() - m).abs() <= m.abs() * (2.0 ** -4 + 8 * E) + 8 * E * msize
                         + top(m) * 2.0 ** -10).all())
            r, nr = v.sqrt(), new["v"].double().sqrt()
            assert bool(((nr - r).abs() <= r * (2.0 ** -4 + 16 * E) + top(r) * 2.0 ** -9).all())
            assert bool((nr > 0)[r > 0].all())


def test_more_tensors_than_one_launch_holds(dev):
    from usaf_b200 import dense_optim
    shapes = [(1 + i % 300,) for i in range(1500)]
    params = tensors(dev, shapes, torch.float32, 4)
    grads = gradients(dev, shapes, torch.float32, 5)
    one = [p.clone() for p in params]
    starts, total = dense_optim.state_layout(p.numel() for p in params)
    m, v = torch.zeros(total, device=dev), torch.zeros(total, device=dev)
    dense_optim.adamw_step(params, grads, m, v, step=1, lr=1e-2, weight_decay=0.1)
    for p, g, q in zip(one, grads, params):
        n = -(-p.numel() // BLOCK) * BLOCK
        dense_optim.adamw_step([p], [g], torch.zeros(n, device=dev), torch.zeros(n, device=dev), step=1, lr=1e-2,
                               weight_decay=0.1)
        assert torch.equal(p, q)


def test_unaligned_tensors_and_around(dev):
    """Parameters and gradients at odd addresses; memory around them and the
    states between tensors keep their values."""
    from usaf_b200 import dense_optim
    for dt in (torch.float32, torch.bfloat16):
        held = torch.full((5000,), 3.0, device=dev, dtype=dt)
        ghold = torch.randn(5000, device=dev).to(dt)
        places = [(1, 700), (703, 1024), (1729, 255), (1985, 2049)]
        params, grads = ([t[a:a + n] for a, n in places] for t in (held, ghold))
        ref = [(p.clone(), g.clone()) for p, g in zip(params, grads)]
        starts, total = dense_optim.state_layout(n for _, n in places)
        m, v = torch.full((total,), 9.0, device=dev), torch.full((total,), 9.0, device=dev)
        rm, rv = m.clone(), v.clone()
        dense_optim.adamw_step(params, grads, m, v, step=2, lr=1e-2)
        dense_optim.adamw_step([p for p, _ in ref], [g for _, g in ref], rm, rv, step=2, lr=1e-2)
        inside = torch.zeros(5000, dtype=torch.bool, device=dev)
        for (a, n), p, (q, _), s in zip(places, params, ref, starts):
            assert torch.equal(p, q)
            inside[a:a + n] = True
            end = s + -(-n // BLOCK) * BLOCK
            assert bool((m[s + n:end] == 9.0).all()) and bool((v[s + n:end] == 9.0).all())
        assert torch.equal(m, rm) and torch.equal(v, rv)
        assert bool((held[~inside] == 3.0).all())


def test_states_stay_apart_and_parts_of_them(dev):
    """A parameter without a gradient keeps everything; the others step as if
    alone; gradients of two types in one step."""
    from usaf_b200 import dense_optim
    for bits in (8, 32):
        params = tensors(dev, [(300,), (500, 3), (70,)], torch.bfloat16, 6)
        g = gradients(dev, [(300,), (500, 3), (70,)], torch.float32, 7)
        named = {k: torch.nn.Parameter(p, requires_grad=False) for k, p in zip("abc", params)}
        opt = dense_optim.AdamW(named, state_bits=bits)
        opt.step({"a": g[0], "b": g[1].bfloat16(), "c": g[2]})
        before = {k: {n: t.clone() for n, t in opt.state(k).items()} for k in "abc"}
        b0 = params[1].clone()
        opt.step({"a": g[0], "c": g[2].bfloat16()})
        assert all(torch.equal(opt.state("b")[n], t) for n, t in before["b"].items()) and torch.equal(params[1], b0)
        assert not torch.equal(opt.state("a")["m"], before["a"]["m"])
        assert not torch.equal(opt.state("c")["m"], before["c"]["m"])


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_round_trip(dev, bits, tmp_path):
    from usaf_b200 import dense_optim
    shapes = [(300,), (64, 33)]

    def make():
        ps = tensors(dev, shapes, torch.bfloat16, 8)
        return ps, dense_optim.AdamW({str(i): torch.nn.Parameter(p, requires_grad=False) for i, p in enumerate(ps)},
                                     state_bits=bits, lr=1e-2)

    a, opt_a = make()
    for t in range(3):
        opt_a.step({str(i): g for i, g in enumerate(gradients(dev, shapes, torch.bfloat16, t))})
    torch.save(opt_a.state_dict(), tmp_path / "s.pt")
    b, opt_b = make()
    opt_b.load_state_dict(torch.load(tmp_path / "s.pt", weights_only=True))
    for x, y in zip(a, b):
        y.copy_(x)
    g = {str(i): g for i, g in enumerate(gradients(dev, shapes, torch.bfloat16, 50))}
    opt_a.step(g)
    opt_b.step(g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(opt_a.state(k)[n], opt_b.state(k)[n]) for k in "01" for n in ("m", "v", "master"))
    with pytest.raises(ValueError, match="bits"):
        sd = dict(opt_a.state_dict(), state_bits=40 - bits)
        opt_b.load_state_dict(sd)
    sd = opt_a.state_dict()
    sd["m"]["1"] = sd["m"]["1"][:-1]
    before = opt_b.state("0")["m"].clone()
    with pytest.raises(ValueError, match="no m"):
        opt_b.load_state_dict(sd)
    assert torch.equal(opt_b.state("0")["m"], before)
    # masters follow weights that are loaded anew
    a[0].fill_(0.25)
    opt_a.refresh_masters()
    assert bool((opt_a.state("0")["master"] == 0.25).all())


def test_inf_stays_in_its_place(dev):
    """A gradient with an infinity or NaN spoils its own value (in 8 bits its
    block), no other."""
    from usaf_b200 import dense_optim
    for bits in (8, 32):
        (p,), (g,) = tensors(dev, [(2000,)], torch.float32, 1), gradients(dev, [(2000,)], torch.float32, 2)
        q, bad = p.clone(), g.clone()
        bad[600], bad[1500] = float("inf"), float("nan")
        for w, d in ((p, g), (q, bad)):
            opt = dense_optim.AdamW({"w": torch.nn.Parameter(w, requires_grad=False)}, state_bits=bits)
            opt.step({"w": d})
            opt.step({"w": g})
        same = torch.ones(2000, dtype=torch.bool, device=dev)
        if bits == 8:
            same[512:768] = False
            same[1280:1536] = False
        else:
            same[600] = same[1500] = False
        assert torch.equal(p[same], q[same])


def test_captured_step(dev):
    """The step itself can be captured: replays step the buffers again, with
    the gradients of the time."""
    from usaf_b200 import dense_optim
    shapes = [(300,), (64, 33)]
    ps, gs = tensors(dev, shapes, torch.float32, 8), gradients(dev, shapes, torch.float32, 1)
    qs = [p.clone() for p in ps]
    _, total = dense_optim.state_layout(p.numel() for p in ps)
    sa, sb = ([torch.zeros(total, device=dev) for _ in range(2)] for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense_optim.adamw_step(ps, gs, *sa, step=5, lr=1e-2)
    for t in range(3):
        for g, new in zip(gs, gradients(dev, shapes, torch.float32, 20 + t)):
            g.copy_(new)
        graph.replay()
        dense_optim.adamw_step(qs, gs, *sb, step=5, lr=1e-2)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps + sa, qs + sb))
    opt = dense_optim.AdamW({"w": torch.nn.Parameter(ps[0], requires_grad=False)})
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step({"w": gs[0]})


def test_a_graph_that_saved_the_weights_notices_the_step(dev):
    from usaf_b200 import dense_optim
    w = torch.nn.Parameter(torch.ones(64, device=dev))
    x = torch.ones(64, device=dev, requires_grad=True)
    loss = (x * w).sum()
    loss.backward(retain_graph=True)
    dense_optim.AdamW({"w": w}).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals(dev):
    from usaf_b200 import dense_optim
    p, g = torch.ones(300, device=dev), torch.ones(300, device=dev)
    m, v = torch.zeros(512, device=dev), torch.zeros(512, device=dev)
    q = (torch.zeros(512, dtype=torch.float8_e4m3fn, device=dev), torch.zeros(2, device=dev))
    kw = dict(step=1, lr=1e-3)
    step = dense_optim.adamw_step
    with pytest.raises(ValueError, match="gradients for"):
        step([p], [], m, v, **kw)
    with pytest.raises(ValueError, match="step"):
        step([p], [g], m, v, step=0, lr=1e-3)
    with pytest.raises(ValueError, match="grad_div"):
        step([p], [g], m, v, grad_div=0.0, **kw)
    with pytest.raises(ValueError, match="betas"):
        step([p], [g], m, v, betas=(0.9, 1.0), **kw)
    with pytest.raises(ValueError, match="16-byte"):
        step([p[:256]], [g[:256]], torch.zeros(257, device=dev)[1:], v[:256], **kw)
    with pytest.raises(TypeError, match="both"):
        step([p], [g], m, q, **kw)
    with pytest.raises(TypeError, match="gradients"):
        step([p], [g.bfloat16()], m, v, **kw)
    with pytest.raises(TypeError, match="tensor 1"):
        step([p, p.bfloat16()], [g, g.bfloat16()], m, v, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        step([torch.ones(600, device=dev)[::2]], [g], m, v, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        step([p], [g[:299]], m, v, **kw)
    with pytest.raises(ValueError, match="m: expected"):
        step([p], [g], m[:300], v, **kw)
    with pytest.raises(ValueError, match="v scales"):
        step([p], [g], q, (q[0], q[1][:1]), **kw)
    with pytest.raises(ValueError, match="masters"):
        step([p], [g], m, v, masters=p, **kw)
    with pytest.raises(ValueError, match="must not share"):
        step([p], [g], m, m, **kw)
    with pytest.raises(ValueError, match="must not share"):
        step([p], [g], m, v, masters=v, **kw)
    with pytest.raises(ValueError, match="must not share"):
        step([p], [g], q, (q[0].clone(), q[1]), **kw)
    with pytest.raises(ValueError, match="twice"):
        step([p, p], [g, g], torch.zeros(1024, device=dev), torch.zeros(1024, device=dev), **kw)
    with pytest.raises(ValueError, match="share memory"):
        step([p[:200], p[100:]], [g[:200], g[:200]], torch.zeros(512, device=dev), torch.zeros(512, device=dev), **kw)
    for starts in ([3], [256], [-256], [0, 0]):
        with pytest.raises(ValueError, match="starts"):
            step([p], [g], m, v, starts=starts, **kw)
    with pytest.raises(ValueError, match="starts"):
        step([p, p.clone()], [g, g], torch.zeros(1024, device=dev), torch.zeros(1024, device=dev), starts=[0, 256], **kw)
    with pytest.raises(ValueError, match="state_bits"):
        dense_optim.AdamW({"w": torch.nn.Parameter(p)}, state_bits=16)
    with pytest.raises(ValueError, match="no_decay"):
        dense_optim.AdamW({"w": torch.nn.Parameter(p)}, no_decay=("x",))
    with pytest.raises(TypeError, match="CUDA"):
        dense_optim.AdamW({"w": torch.nn.Parameter(p.cpu())})
