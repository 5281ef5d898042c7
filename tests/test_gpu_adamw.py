"""AdamW against a restatement in numpy: the moments bit for bit in fp32 (every operation is rounded on its
own), and against 64 bits with a tolerance counted in roundings."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F = np.float32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.999, 1e-8, 0.02


def encode(x, signed):
    """Codes and scales of a vector, blocks of 256."""
    shift, top = (20, 127) if signed else (19, 255)
    n = len(x)
    x = np.concatenate([x, np.zeros(-n % 256, F)]).reshape(-1, 256)
    scale = np.abs(x).max(1)
    fine = scale >= F(2.0 ** -126)
    with np.errstate(divide="ignore"):
        r = np.where(fine, F(1) / scale, F(0)).astype(F)
    y = (x * r[:, None]).astype(F)
    bits = np.abs(y).view(np.int32)
    code = ((bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift) - ((0x3F800000 >> shift) - top)
    code = np.where(bits == 0, 0, np.clip(code, 0 if signed else 1, top))
    code = np.where(fine[:, None], code, 0)
    if signed:
        code = code + 128 * ((y < 0) & (code > 0))
    return code.reshape(-1)[:n].astype(np.uint8), np.where(fine, scale, F(0)).astype(F)


def decode(codes, scale, signed):
    shift, top = (20, 127) if signed else (19, 255)
    low = codes.astype(np.int32)
    sign = low >= 128 if signed else np.zeros(len(low), bool)
    low = low & 127 if signed else low
    y = np.where(low > 0, ((low + ((0x3F800000 >> shift) - top)) << shift).astype(np.int32).view(F), F(0))
    y = np.where(sign, -y, y)
    return (y * np.repeat(scale, 256)[:len(codes)]).astype(F)


def step_f32(p, g, m, v, t, lr=LR):
    """One step in fp32, one rounding an operation: (p, m, v, root of v)."""
    c1, c2 = 1.0 - B1 ** t, 1.0 - B2 ** t
    m = m * F(B1) + g * F(1.0 - B1)
    v = v * F(B2) + (g * g) * F(1.0 - B2)
    root = np.sqrt(v)
    return p * F(1.0 - lr * WD) - (m * F(lr / c1)) / (root * F(1.0 / np.sqrt(c2)) + F(EPS)), m, v, root


def make(sizes, ptype, gtype, seed):
    gen = torch.Generator().manual_seed(seed)
    ps = [(torch.randn(n, generator=gen) * 0.4).to(TYPES[ptype]) for n in sizes]
    gs = [(torch.randn(n, generator=gen) * torch.exp(-8 * torch.rand(n, generator=gen))).to(TYPES[gtype])
          for n in sizes]
    return ps, gs


def f32(x):
    return x.detach().float().cpu().numpy().reshape(-1)


SIZES = [[1], [255, 256, 257], [0, 5, 1000], [70001], [7 + 13 * i for i in range(40)], [3] * 300]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                         ("f16", "f32")])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_steps_match_the_restatement(bits, ptype, gtype, sizes):
    from bidmach_b200 import AdamW
    ps, _ = make(sizes, ptype, gtype, 1)
    dev = [p.cuda() for p in ps]
    opt = AdamW(dev, AdamW.Opts(lrate=LR, beta1=B1, beta2=B2, eps=EPS, wdecay=WD, bits=bits))
    p = [f32(x) for x in ps]
    m, v = [np.zeros(n, F) for n in sizes], [np.zeros(n, F) for n in sizes]
    for t in (1, 2, 3):
        gs = make(sizes, ptype, gtype, 10 + t)[1]
        opt.step([g.cuda() for g in gs])
        for i, g in enumerate(gs):
            old = p[i]
            new, m[i], v[i], root = step_f32(old, f32(g), m[i], v[i], t)
            if bits == 8:
                mc, ms = encode(m[i], True)
                vc, vs = encode(root, False)
                np.testing.assert_array_equal(opt.m[i].cpu().numpy(), mc)
                np.testing.assert_array_equal(opt.v[i].cpu().numpy(), vc)
                np.testing.assert_array_equal(opt.mscale[i].cpu().numpy(), ms[:(sizes[i] + 255) // 256])
                m[i], v[i] = decode(mc, ms, True), decode(vc, vs, False) ** 2
            # the quotient is good to two units of its last place (2^-22), and what is then subtracted
            # and rounded may land one unit of the parameter's type further
            p[i] = f32(dev[i])
            unit = torch.finfo(TYPES[ptype]).eps * np.abs(new) + (2.0 ** -24 if ptype == "f16" else 0)
            assert np.all(np.abs(p[i] - new) <= 2.0 ** -22 * (np.abs(old) + np.abs(new - old)) + unit)
        got = opt.moments()
        for i in range(len(sizes)):
            np.testing.assert_array_equal(f32(got[0][i]), m[i])
            np.testing.assert_array_equal(f32(got[1][i]), v[i])


@pytest.mark.parametrize("ptype", list(TYPES))
def test_step_against_64_bits(ptype):
    """m is two products and a sum of rounded constants: 4 roundings of its terms.  The step has 14
    (m 4, root 5 / 2 + 1, product, sum, product, quotient 4); p is off by 2 roundings of its own
    terms, 16 of the step's and the rounding to its type."""
    from bidmach_b200 import AdamW
    u = 2.0 ** -24
    (p,), (g,) = make([10007], ptype, "f32", 5)
    rng = np.random.default_rng(2)
    m0 = rng.standard_normal(10007).astype(F)
    v0 = np.square(rng.standard_normal(10007)).astype(F)
    dp, dm, dv = p.cuda(), torch.from_numpy(m0).cuda(), torch.from_numpy(v0).cuda()
    opt = AdamW([dp], AdamW.Opts(lrate=LR, beta1=B1, beta2=B2, eps=EPS, wdecay=WD),
                state={"t": 6, "m": [dm], "v": [dv]})
    opt.step([g.cuda()])
    g, p = g.double().numpy(), p.double().numpy()
    m = B1 * m0.astype(np.float64) + (1 - B1) * g
    v = B2 * v0.astype(np.float64) + (1 - B2) * g ** 2
    step = LR / (1 - B1 ** 7) * m / (np.sqrt(v / (1 - B2 ** 7)) + EPS)
    terms = np.abs(B1 * m0) + np.abs((1 - B1) * g)
    want = p * (1 - LR * WD) - step
    assert np.all(np.abs(dm.cpu().numpy() - m) <= 4 * u * terms)
    assert np.all(np.abs(dv.cpu().numpy() - v) <= 5 * u * v)
    size = LR / (1 - B1 ** 7) * terms / np.sqrt(v / (1 - B2 ** 7))
    half = torch.finfo(TYPES[ptype]).eps / 2
    assert np.all(np.abs(dp.double().cpu().numpy() - want) <= 3 * u * np.abs(p) + 16 * u * size +
                  (half + u) * (np.abs(want) + size) + (2.0 ** -25 if ptype == "f16" else 0))


@pytest.mark.parametrize("bits", [32, 8])
def test_any_alignment(bits):
    """Views at odd offsets of one buffer: the same bits as separate tensors."""
    from bidmach_b200 import AdamW
    o = AdamW.Opts(bits=bits)
    for off, n in [(1, 777), (3, 256), (2, 513)]:
        (p,), (g,) = make([n], "f32", "f32", off)
        flat, gflat = torch.zeros(2000, device="cuda"), torch.zeros(2000, device="cuda")
        flat[off:off + n] = p.cuda()
        gflat[off:off + n] = g.cuda()
        flat[off + n] = 7.0
        q = p.cuda()
        a, b = AdamW([flat[off:off + n]], o), AdamW([q], o)
        for _ in range(2):
            a.step([gflat[off:off + n]])
            b.step([g.cuda()])
        assert torch.equal(flat[off:off + n], q)
        assert torch.equal(a.m[0], b.m[0]) and torch.equal(a.v[0], b.v[0])
        assert flat[off + n] == 7.0 and flat[:off].abs().sum() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients(bits):
    """A NaN or an infinity spoils its element (with 8 bits the moments of its 256), nothing else."""
    from bidmach_b200 import AdamW
    p = torch.ones(1024, device="cuda")
    opt = AdamW([p], AdamW.Opts(bits=bits))
    g = torch.full((1024,), 0.5, device="cuda")
    g[300], g[900] = float("nan"), float("inf")
    opt.step([g])
    bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
    bad[300] = bad[900] = True
    assert torch.isnan(p[bad]).all() and torch.isfinite(p[~bad]).all()
    m, v = opt.moments()
    if bits == 8:
        bad[256:512] = True
        bad[768:] = True
        assert torch.isnan(m[0][bad]).all()
    assert torch.isfinite(m[0][~bad]).all() and torch.isfinite(v[0][~bad]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_and_zero_gradients(bits):
    """No step is larger than lrate / (1 - beta1) whatever the gradients' size; zeros move nothing."""
    from bidmach_b200 import AdamW
    for size in (0.0, 1e-30, 1e-38, 1e-42, 1e30 ** 0.5):
        p = torch.zeros(600, device="cuda")
        g = torch.linspace(-1, 1, 600, device="cuda") * size
        opt = AdamW([p], AdamW.Opts(lrate=0.1, bits=bits))
        for _ in range(4):
            opt.step([g])
        assert torch.isfinite(p).all() and float(p.abs().max()) <= 4 * 1.0
        if size == 0.0:
            assert float(p.abs().max()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count(bits):
    """A captured step, replayed, does what as many calls do, with a rate read from the device."""
    from bidmach_b200 import AdamW
    (p,), (g,) = make([5000], "f32", "f32", 3)
    a, b, g = p.cuda(), p.cuda(), g.cuda()
    rate = torch.tensor([0.01], device="cuda")
    oa, ob = AdamW([a], AdamW.Opts(bits=bits)), AdamW([b], AdamW.Opts(bits=bits))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ob.step([g], rate)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        ob.step([g], rate)
    oa.step([g], 0.01)
    for r in (0.01, 0.02, 0.005):
        rate.fill_(r)
        graph.replay()
        oa.step([g], float(torch.tensor(r)))
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(oa.m[0], ob.m[0]) and torch.equal(oa.v[0], ob.v[0])


def test_refusals_on_the_device():
    from bidmach_b200 import AdamW
    p = torch.zeros(512, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        AdamW([p[:300], p[200:]])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([p.view(2, 256).t()])
    opt = AdamW([p])
    for g in (torch.zeros(511, device="cuda"), torch.zeros(512), torch.zeros(512, device="cuda", dtype=torch.float16),
              torch.zeros(1024, device="cuda")[::2]):
        with pytest.raises(ValueError):
            opt.step([g])
    with pytest.raises(ValueError):
        opt.step([])
    with pytest.raises(ValueError):
        opt.step([p], torch.zeros(1))
    with pytest.raises(ValueError, match="state"):
        AdamW([p], state={"t": 0, "m": [torch.zeros(511, device="cuda")], "v": [p.clone()]})
    with pytest.raises(ValueError):
        opt.moments(mout=[p.clone()])


def test_moments_that_share_memory_are_refused():
    from bidmach_b200 import AdamW
    p = torch.zeros(300, device="cuda")
    x = torch.zeros(300, device="cuda")
    for m, v in ((x, x), (p, x), (x, p)):
        with pytest.raises(ValueError, match="overlaps"):
            AdamW([p], state=dict(t=0, m=[m], v=[v]))


@pytest.mark.parametrize("bits", [32, 8])
def test_smallest_eps(bits):
    """An eps that fp32 does not hold: an element without a gradient only decays."""
    from bidmach_b200 import AdamW
    p = torch.ones(300, device="cuda")
    opt = AdamW([p], AdamW.Opts(lrate=0.5, eps=1e-60, wdecay=0.5, bits=bits))
    g = torch.zeros(300, device="cuda")
    g[7] = 2.0
    opt.step([g])
    want = torch.full((300,), 0.75)
    want[7] = 0.25      # the first step is lrate in the gradient's direction
    # m / c1 and sqrt(v / c2): six roundings each and three of the step, below 2^-19 in all
    assert torch.allclose(p.cpu(), want, rtol=0, atol=2.0 ** -19)
    assert torch.equal(p.cpu()[8:], want[8:])


def mix32(x):
    x = np.asarray(x, np.uint32)
    x = ((x ^ x >> 16) * np.uint32(0x85ebca6b)).astype(np.uint32)
    x = ((x ^ x >> 13) * np.uint32(0xc2b2ae35)).astype(np.uint32)
    return x ^ x >> 16


def encode_random(x, signed, key, first):
    """Codes rounded at random; `first` is the place of x[0] among the random bits."""
    shift, top = (20, 127) if signed else (19, 255)
    n = len(x)
    x = np.concatenate([x, np.zeros(-n % 256, F)]).reshape(-1, 256)
    scale = np.abs(x).max(1)
    y = (x * np.where(scale >= F(2.0 ** -126), F(1) / np.maximum(scale, F(2.0 ** -126)), F(0)).astype(F)[:, None]).reshape(-1)
    bits = np.abs(y).view(np.uint32)
    h = mix32((first + np.arange(len(y))).astype(np.uint32) ^ key)
    if signed:
        code = (bits + (h & np.uint32(0xfffff))) >> 20
    else:
        f, m = (bits & np.uint32(2 ** 19 - 1)).astype(F) * F(2.0 ** -19), (32 + (bits >> 18 & 30)).astype(F)
        up = (f * (m + f)) * (F(1) / (m + F(1)))
        code = (bits >> 19) + (((up * F(2.0 ** 19)).astype(np.uint32) + (h >> 13)) >> 19)
    code = np.minimum(code.astype(np.int64), 0x3F800000 >> shift) - ((0x3F800000 >> shift) - top)
    code = np.where(bits == 0, 0, np.maximum(code, 0 if signed else 1))
    if signed:
        code = code + 128 * ((y < 0) & (code > 0))
    return code[:n].astype(np.uint8), scale.astype(F)


@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [0, 5, 1000], [70001], [3] * 300], ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("ptype", list(TYPES))
def test_random_rounding_matches_the_restatement(ptype, sizes):
    from bidmach_b200 import AdamW
    seed = 0x123456789
    ps, _ = make(sizes, ptype, "f32", 1)
    opt = AdamW([p.cuda() for p in ps], AdamW.Opts(lrate=LR, beta1=B1, beta2=B2, eps=EPS, wdecay=WD, bits=8,
                                                  rounding="random", seed=seed))
    m, v = [np.zeros(n, F) for n in sizes], [np.zeros(n, F) for n in sizes]
    with np.errstate(over="ignore"):
        for t in range(3):
            gs = make(sizes, ptype, "f32", 10 + t)[1]
            opt.step([g.cuda() for g in gs])
            unit, launch = 0, 0
            for i, g in enumerate(gs):
                if i == 256:          # the tensors of a launch
                    unit, launch = 0, 1
                key = mix32(mix32(np.uint32(seed & 0xffffffff) + mix32(np.uint32((seed >> 32) + launch * 0x9e3779b9))) +
                            np.uint32(t * 0x9e3779b9 & 0xffffffff))
                _, m[i], v[i], root = step_f32(np.zeros(sizes[i], F), f32(g), m[i], v[i], t + 1)
                mc, ms = encode_random(m[i], True, key, unit * 256)
                vc, vs = encode_random(root, False, key, unit * 256)
                np.testing.assert_array_equal(opt.m[i].cpu().numpy(), mc)
                np.testing.assert_array_equal(opt.v[i].cpu().numpy(), vc)
                np.testing.assert_array_equal(opt.vscale[i].cpu().numpy(), vs[:(sizes[i] + 255) // 256])
                m[i], v[i] = decode(mc, ms, True), decode(vc, vs, False) ** 2
                unit += (sizes[i] + 255) // 256


@pytest.mark.parametrize("beta1", [0.9, 0.99])
@pytest.mark.parametrize("case", ["falling", "rising", "sparse"])
def test_moments_in_8_bits_over_thousands_of_steps(case, beta1):
    """Gradients whose size changes, beside 32-bit moments: the mean over 8160 elements of the stored v is the
    32-bit one.  The first element of each block keeps gradients of size 1, so the others are relative to it.

    Tolerance.  Rounding is right in the mean, so what is left is chance.  A code is at most 1/16 above the one
    before, so a step that changes sqrt(v) relative to its scale by d adds at most 4 d / 16 to the relative
    variance of v.  The 8000 steps of `falling` change it by 4.6 of its own and about 1e-3 a step with
    the scale, 13 in all: the relative variance of an element is at most exp(13 / 4) - 1 = 25, the standard
    deviation of the mean of 8160 is 0.055, and 0.3 is more than five times that.  The sums of m have
    a spread of their own: they are compared as m against 32 bits in norm over one step's rounding,
    below 1/8 each over about 1 / (1 - beta1) steps, in quadrature with weights beta1^k."""
    from bidmach_b200 import AdamW
    n = 32 * 256
    gen = torch.Generator(device="cuda").manual_seed(7)
    first = torch.zeros(n, dtype=torch.bool, device="cuda")
    first[::256] = True
    o = dict(lrate=0.0, beta1=beta1, beta2=0.999, wdecay=0.0)
    a = AdamW([torch.zeros(n, device="cuda")], AdamW.Opts(bits=32, **o))
    b = AdamW([torch.zeros(n, device="cuda")], AdamW.Opts(bits=8, rounding="random", seed=3, **o))
    size = {"falling": (1.0, 0.01), "rising": (0.2, 1.0), "sparse": (1.0, 1.0)}[case]
    for t in range(10000):
        g = torch.randn(n, generator=gen, device="cuda")
        scale = size[0] if t < 2000 else size[1]
        if case == "sparse":
            scale = (torch.rand(n, generator=gen, device="cuda") < 0.01).float()
        g = torch.where(first, g, g * scale)
        a.step([g])
        b.step([g])
    (ma,), (va,) = a.moments()
    (mb,), (vb,) = b.moments()
    rest = ~first
    ratio = float(vb[rest].double().mean() / va[rest].double().mean())
    assert 0.7 <= ratio <= 1.3, ratio
    off = float((mb - ma)[rest].double().norm() / ma[rest].double().norm())
    # each step's rounding is below 1/8 of a code's value of m, whose size stays about that of the last one
    assert off <= 0.125 / (1 - beta1 ** 2) ** 0.5, off


def test_random_rounding_repeats_and_is_asked_for():
    from bidmach_b200 import AdamW
    (p,), (g,) = make([5000], "f32", "f32", 3)
    g = g.cuda()

    def after(seed, steps=3, start=0):
        opt = AdamW([p.cuda()], AdamW.Opts(bits=8, rounding="random", seed=seed))
        for _ in range(steps):
            opt.step([g])
        return torch.cat([opt.m[0], opt.v[0]])

    assert torch.equal(after(5), after(5)) and not torch.equal(after(5), after(6)) and not torch.equal(after(5), after(5 + 2 ** 32))
    # a captured step draws other bits in each replay, those of as many calls
    q = p.cuda()
    opt = AdamW([q], AdamW.Opts(bits=8, rounding="random", seed=5))
    opt.step([g])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    graph.replay()
    graph.replay()
    assert torch.equal(torch.cat([opt.m[0], opt.v[0]]), after(5))
    # a step count that goes on draws on
    t2 = AdamW([p.cuda()], AdamW.Opts(bits=8, rounding="random", seed=5),
               state=dict(t=3, m=[opt.m[0].clone()], v=[opt.v[0].clone()], mscale=[opt.mscale[0].clone()],
                          vscale=[opt.vscale[0].clone()]))
    t2.step([g])
    assert torch.equal(torch.cat([t2.m[0], t2.v[0]]), after(5, 4))
    with pytest.warns(UserWarning, match="rounding"):
        AdamW([p.cuda()], AdamW.Opts(bits=8))


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_move(bits):
    """After p.data = ... or p.set_ a step works on the new memory and leaves the old alone."""
    from bidmach_b200 import AdamW
    ps, gs = make([700, 300], "f32", "f32", 4)
    gs = [g.cuda() for g in gs]
    a, b = [p.cuda() for p in ps], [p.cuda() for p in ps]
    o = AdamW.Opts(bits=bits, rounding="random")
    oa, ob = AdamW(a, o), AdamW(b, o)
    oa.step(gs)
    ob.step(gs)
    for change in (lambda x: setattr(x, "data", x.clone()), lambda x: x.set_(x.clone()),
                   lambda x: setattr(x, "data", torch.cat([x.new_zeros(5), x])[5:])):
        old = b[1].detach()
        kept = old.clone()
        change(b[1])
        assert b[1].data_ptr() != old.data_ptr()
        oa.step(gs)
        ob.step(gs)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(old, kept)
    for bad, match in ((lambda: setattr(b[1], "data", torch.zeros(301, device="cuda")), "size"),
                       (lambda: setattr(b[1], "data", b[0].data[:300]), "overlap"),
                       (lambda: setattr(b[1], "data", torch.zeros(600, device="cuda")[::2]), "contiguous")):
        good = b[1].data
        bad()
        with pytest.raises(ValueError, match=match):
            ob.step(gs)
        b[1].data = good
    oa.step(gs)
    ob.step(gs)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_state_that_is_given_other_memory():
    """The updater goes on with the moments that it was given."""
    from bidmach_b200 import AdamW
    p, m, v = (torch.zeros(300, device="cuda") for _ in range(3))
    opt = AdamW([p], state=dict(t=0, m=[m], v=[v]))
    was = m.detach()
    m.set_(torch.zeros(300, device="cuda"))
    opt.step([torch.ones(300, device="cuda")])
    assert torch.equal(opt.m[0], was) and not m.any()
    assert abs(float(was[0]) - 0.1) <= 2.0 ** -24


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_in_the_state_are_refused(bits):
    from bidmach_b200 import AdamW
    buf = torch.zeros(2048, device="cuda")
    p, g = buf[:512], buf[512:1024]
    opt = AdamW([p], AdamW.Opts(bits=bits, rounding="random"))
    state = opt.m[0] if bits == 32 else opt.mscale[0]
    opt.step([g])
    before = [x.clone() for x in (p, opt.m[0], opt.v[0])]
    for bad in ([p], [buf[256:768]], [opt.m[0]] if bits == 32 else [opt.m[0].view(torch.float32)]):
        if bad[0].numel() == 512:
            with pytest.raises(ValueError, match="shares memory"):
                opt.step(bad)
    assert all(torch.equal(x, y) for x, y in zip(before, (p, opt.m[0], opt.v[0])))
    # one tensor for several parameters is fine, next to the parameters too
    two = AdamW([buf[:512], buf[1024:1536]], AdamW.Opts(bits=bits, rounding="random"))
    two.step([g, g])
    two.step([g, g])
    with pytest.raises(ValueError, match="shares memory"):
        two.step([g, buf[1000:1512]])
    assert state.is_cuda


def test_moments_into_shared_memory_are_refused():
    from bidmach_b200 import AdamW
    ps = [torch.zeros(n, device="cuda") for n in (600, 256)]
    opt = AdamW(ps, AdamW.Opts(bits=8, rounding="random"))
    opt.step([torch.randn(n, device="cuda") for n in (600, 256)])
    want = opt.moments()
    x, y, z = (torch.zeros(n, device="cuda") for n in (600, 256, 1000))
    for m, v in (([x, y], [x, y]), ([x, z[:256]], [z[200:800], y]), ([ps[0], y], [x, z[:256]]),
                 ([x, y], [z[:600], ps[1]]), ([x, z[:256]], [z[400:], z[100:356]])):
        with pytest.raises(ValueError, match="overlap|shares memory"):
            opt.moments(m, v)
    got = opt.moments([x, y], [z[:600], z[600:856]])
    for _ in range(2):
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
        got = opt.moments([x, y], [z[:600], z[600:856]])


def test_moments_over_a_parameter_that_moved_are_refused():
    from bidmach_b200 import AdamW
    p, out = torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda")
    opt = AdamW([p], AdamW.Opts(bits=8, rounding="random"))
    opt.moments([out], [torch.zeros(256, device="cuda")])
    p.data = out
    with pytest.raises(ValueError, match="shares memory"):
        opt.moments([out], [torch.zeros(256, device="cuda")])
