"""Softmax cross entropy over the vocabulary and its gradients against 64 bits.

Tolerances.  u = 2^-24.  A logit is a sum of dim products; with |h|.|w| the sum of their magnitudes it is
off by at most (dim u + 2^-20) |h|.|w|: fp32 accumulation, which the tensor cores truncate (twice a
rounding, hence dim u for the whole sum of the usual dim u / 2), and, for fp32 operands, 22 bits of each
and the product of the two remainders.  So lse is off by that plus 2^-21 of its terms (an exponential is
good to 2^-22, its argument to a rounding of numbers below 64, the logarithm and the result to u each):
`E` below.  A gradient is off by E + 2^-20 relative in every probability, by a half step of the type that
d is rounded to, by accumulation, and by a half step of its own type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def inputs(n, vocab, dim, labels, t, seed=0, size=1.0):
    gen = torch.Generator().manual_seed(seed + n + vocab + dim)
    hidden = (torch.randn(n, dim, generator=gen) * size).to(TYPES[t])
    weight = (torch.randn(vocab, dim, generator=gen) * (2.0 / dim ** 0.5)).to(TYPES[t])
    targets = torch.randint(-1, vocab + 1, (n, labels), generator=gen, dtype=torch.int32)   # -1 and vocab: none
    if n > 2:
        targets[n // 2] = -1
        targets[0] = vocab - 1      # the same word in every slot
    gloss = torch.rand(n, generator=gen) / n
    return hidden, weight, targets, gloss


def formula(hidden, weight, targets, gloss):
    h, w, g = hidden.double(), weight.double(), gloss.double()
    vocab = w.shape[0]
    there = (targets >= 0) & (targets < vocab)
    at = targets.long().clamp(0, vocab - 1)
    x = h @ w.T
    lse = torch.logsumexp(x, 1)
    loss = torch.where(there, lse[:, None] - x.gather(1, at), 0.0).sum(1)
    k = there.sum(1).double()
    prob = torch.exp(x - lse[:, None]) * (g * k)[:, None]
    hit = torch.zeros_like(x).scatter_add_(1, at, torch.where(there, g[:, None], 0.0))
    d = prob - hit
    return {"loss": loss, "lse": lse, "dh": d @ w, "dw": d.T @ h, "d": d, "prob": prob, "hit": hit, "k": k}


def hold(got, hidden, weight, targets, gloss, t):
    """Asserts that (loss, lse, dh, dw) are within the bounds above."""
    f = formula(hidden, weight, targets, gloss)
    h, w = hidden.double().abs(), weight.double().abs()
    n, dim = h.shape
    vocab = w.shape[0]
    e = (dim * U + 2.0 ** -20) * (h @ w.T).amax(1)
    lse_off = e + 2.0 ** -20 * (1 + f["lse"].abs())
    loss, lse, dh, dw = (x.double().to(h.device) for x in got)
    assert torch.all((lse - f["lse"]).abs() <= lse_off)
    assert torch.all((loss - f["loss"]).abs() <= f["k"] * (lse_off + e) + f["k"] * U * f["loss"].abs())
    # what d may be off by: its probabilities, then its rounding (fp32 keeps 22 bits of it)
    half = torch.finfo(TYPES[t]).eps / 2
    rel = (e + lse_off + 2.0 ** -20)[:, None]
    off = 1.001 * rel * f["prob"].abs() + (half if t != "f32" else 2.0 ** -21) * f["d"].abs() + U * f["hit"].abs()
    top = (gloss.double().abs() * f["k"]).amax()
    off = off + 2.0 ** -126 * top     # an exponential below the smallest normal number is zero
    if t != "bf16":    # fp16 parts of d: steps of 2^-25 where the largest row's is 2^14 to 2^15
        off = off + 2.0 ** (-38 if t == "f16" else -48) * top
    grow = 2 * U       # truncated accumulation, and the joining of pieces
    for got_g, want, other, terms, count in ((dh, f["dh"], w, f["d"].abs(), vocab), (dw, f["dw"], h, f["d"].abs().T, n)):
        o = off if other is w else off.T
        size = terms @ other
        bound = o @ other + (grow * (count + 64) + 2.0 ** -20) * size
        bound = bound + (half + U) * (want.abs() + bound) + (2.0 ** -25 if t == "f16" else 2.0 ** -126)
        assert torch.all((got_g - want).abs() <= bound)


def run(hidden, weight, targets, gloss):
    from bidmach_b200 import Softmax
    h, w, y, g = hidden.cuda(), weight.cuda(), targets.cuda(), gloss.cuda()
    loss, lse = Softmax.loss(h, w, y)
    return (loss, lse, *Softmax.grad(h, w, y, lse, g))


SIZES = [(1, 1, 1), (1, 1000, 256), (2, 33, 7), (3, 257, 300), (5, 1001, 64), (8, 4097, 100), (9, 1, 1), (9, 255, 64),
         (16, 300, 301), (17, 300, 100), (4, 999, 96), (12, 60, 513), (127, 256, 128), (128, 513, 37), (129, 1000, 16), (200, 5003, 300), (300, 777, 1000),
         (515, 2049, 520), (64, 40, 4096)]


@pytest.mark.parametrize("n,vocab,dim", SIZES)
@pytest.mark.parametrize("labels", [1, 5])
@pytest.mark.parametrize("t", list(TYPES))
def test_against_64_bits(n, vocab, dim, labels, t):
    x = inputs(n, vocab, dim, labels, t)
    hold(run(*x), *x, t)


@pytest.mark.parametrize("n,vocab,dim,t", [(8500, 12000, 24, "f32"), (8500, 21000, 24, "bf16"), (16600, 300, 16, "f16"),
                                           (8193, 1000, 300, "f32"), (700, 40000, 40, "f16")])
def test_several_pieces(n, vocab, dim, t):
    """More rows or words than one piece holds: sums go on over pieces, the last one smaller."""
    x = inputs(n, vocab, dim, 2, t)
    got = run(*x)
    hold([g.cuda() for g in got], *[v.cuda() for v in x], t)


@pytest.mark.parametrize("n", [5, 100])
@pytest.mark.parametrize("t", list(TYPES))
def test_one_factor_for_all_rows(n, t):
    hidden, weight, targets, _ = inputs(n, 700, 48, 3, t)
    for g in (1.0, -0.375, 1e-6, 3e4):
        if t == "f16" and g == 3e4:
            continue     # the gradients themselves leave the type's range
        one = torch.tensor([g])
        got = run(hidden, weight, targets, one)
        f = formula(hidden, weight, targets, one.expand(n))
        for have, want in ((got[2], f["dh"]), (got[3], f["dw"])):
            half = torch.finfo(TYPES[t]).eps / 2
            terms = (f["d"].abs() @ weight.double().abs()).amax() if want is f["dh"] else \
                (f["d"].abs().T @ hidden.double().abs()).amax()
            # d and the result are rounded, the rest is fp32: four half steps of the largest sum of terms
            bound = 4 * max(half, 2.0 ** -18) * terms + (2.0 ** -25 if t == "f16" else 0)
            assert (have.double().cpu() - want).abs().amax() <= bound


@pytest.mark.parametrize("n", [4, 60])
@pytest.mark.parametrize("t", list(TYPES))
def test_weights_of_rows_over_decades(n, t):
    """Zero, negative and tiny factors of single rows beside large ones."""
    hidden, weight, targets, gloss = inputs(n, 333, 40, 2, t)
    gloss = gloss * torch.logspace(0, -5, n)
    gloss[1] = 0.0
    gloss[2] = -gloss[2]
    got = run(hidden, weight, targets, gloss)
    hold(got, hidden, weight, targets, gloss, t)
    assert not got[2][1].any()


@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("t", list(TYPES))
def test_rows_inside_wider_matrices(n, t):
    """Any leading dimension and alignment, of the operands and of the results; what lies between stays."""
    from bidmach_b200 import Softmax
    for off, dim in ((0, 64), (8, 56), (3, 61), (1, 16)):
        hidden, weight, targets, gloss = inputs(n, 515, dim, 1, t)
        base_h, base_w = torch.zeros(n, 80, dtype=TYPES[t], device="cuda"), torch.zeros(515, 88, dtype=TYPES[t], device="cuda")
        h, w = base_h[:, off:off + dim], base_w[:, off:off + dim]
        h.copy_(hidden)
        w.copy_(weight)
        y, g = targets[:, 0].contiguous().cuda(), gloss.cuda()
        loss, lse = Softmax.loss(h, w, y)
        dbase_h, dbase_w = torch.full_like(base_h, 9.0), torch.full_like(base_w, 9.0)
        dh, dw = Softmax.grad(h, w, y, lse, g, dhidden=dbase_h[:, off:off + dim], dweight=dbase_w[:, off:off + dim])
        hold((loss, lse, dh, dw), hidden, weight, targets, gloss, t)
        for base in (dbase_h, dbase_w):
            keep = torch.ones(base.shape[1], dtype=torch.bool)
            keep[off:off + dim] = False
            assert (base[:, keep] == 9.0).all()


@pytest.mark.parametrize("n", [6, 150])
@pytest.mark.parametrize("t", list(TYPES))
def test_large_and_small_logits(n, t):
    """Logits up to a few hundred (all but one word at probability zero) and logits of nearly zero."""
    for size in (30.0, 2.0 ** -12):
        x = inputs(n, 400, 64, 2, t, size=size)
        hold(run(*x), *x, t)


@pytest.mark.parametrize("n", [5, 90])
@pytest.mark.parametrize("t", list(TYPES))
def test_not_finite_rows(n, t):
    """An infinity or a NaN in a row of hidden spoils that row's lse and loss, no other's."""
    from bidmach_b200 import Softmax
    hidden, weight, targets, _ = inputs(n, 300, 32, 1, t)
    targets[:] = 7
    want = formula(hidden, weight, targets, torch.ones(n))
    hidden[1, 3], hidden[3, 5] = float("nan"), float("inf")
    loss, lse = Softmax.loss(hidden.cuda(), weight.cuda(), targets.cuda())
    bad = torch.zeros(n, dtype=torch.bool)
    bad[1] = bad[3] = True
    assert torch.isnan(lse.cpu()[bad]).all() and torch.isnan(loss.cpu()[bad]).all()
    assert (lse.cpu().double() - want["lse"])[~bad].abs().max() <= 2.0 ** -14
    assert torch.isfinite(loss.cpu()[~bad]).all()


def test_no_rows_and_no_targets():
    from bidmach_b200 import Softmax
    w = torch.randn(50, 12, device="cuda")
    h, y = torch.empty(0, 12, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda")
    loss, lse = Softmax.loss(h, w, y)
    assert loss.shape == lse.shape == (0,)
    dh, dw = Softmax.grad(h, w, y, lse, torch.ones(1, device="cuda"))
    assert dh.shape == (0, 12) and not dw.any()
    for n in (3, 70):
        h, y = torch.randn(n, 12, device="cuda"), torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
        loss, lse = Softmax.loss(h, w, y)
        dh, dw = Softmax.grad(h, w, y, lse, torch.ones(n, device="cuda"))
        assert not loss.any() and not dh.any() and not dw.any() and torch.isfinite(lse).all()


@pytest.mark.parametrize("n,vocab,dim,t", [(7, 500, 20, "f32"), (130, 900, 33, "f32")])
def test_gradient_against_differences(n, vocab, dim, t):
    """Along a direction, the difference of the kernel's losses over a step and the kernel's gradient.  The
    difference has the formula's own curvature error, taken from the same difference in 64 bits, and
    the losses' rounding over the step."""
    from bidmach_b200 import Softmax
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, t)
    gen = torch.Generator().manual_seed(3)
    u, z, e = torch.randn(n, dim, generator=gen), torch.randn(vocab, dim, generator=gen) / dim ** 0.5, 2.0 ** -6

    def total(s):
        loss, _ = Softmax.loss((hidden + s * u).cuda(), (weight + s * z).cuda(), targets.cuda())
        return float((loss.double().cpu() * gloss.double()).sum())

    def total64(s):
        return float((formula(hidden.double() + s * u, weight.double() + s * z, targets, gloss)["loss"] * gloss.double()).sum())

    _, _, dh, dw = run(hidden, weight, targets, gloss)
    along = float((dh.double().cpu() * u).sum() + (dw.double().cpu() * z).sum())
    f = formula(hidden, weight, targets, gloss)
    exact = float((f["dh"] * u).sum() + (f["dw"] * z).sum())
    curved = abs((total64(e) - total64(-e)) / (2 * e) - exact)
    size = (hidden.abs() + e * u.abs()).double() @ (weight.abs() + e * z.abs()).double().T
    noise = float((gloss.double() * f["k"] * (2 * (dim + 64) * U * size.amax(1) + 2.0 ** -19 * (1 + f["lse"].abs()))).sum()) / e
    assert abs((total(e) - total(-e)) / (2 * e) - along) <= curved + noise + 2.0 ** -16 * abs(exact)


def test_equal_calls_streams_and_graphs():
    """Calls at once on several streams, and captured graphs replayed side by side, give the bits of the call
    alone."""
    from bidmach_b200 import Softmax
    sets = []
    for n, vocab, dim, t in ((300, 3000, 100, "bf16"), (260, 2000, 70, "f32"), (12, 3000, 50, "f32"), (3, 900, 64, "f16")):
        x = [v.cuda() for v in inputs(n, vocab, dim, 2, t)]
        sets.append((x, run(*x)))
    torch.cuda.synchronize()

    def step(x):
        loss, lse = Softmax.loss(*x[:3])
        return (loss, lse, *Softmax.grad(*x[:3], lse, x[3]))

    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(3):
        for s, (x, want) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append((step(x), want))
    torch.cuda.synchronize()
    graphs = []
    for x, want in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x)
        graphs.append(graph)
        got.append((out, want))
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for have, want in got:
        assert all(torch.equal(a, b) for a, b in zip(have, want))


def test_refusals_on_the_device():
    from bidmach_b200 import Softmax
    h, w = torch.zeros(4, 8, device="cuda"), torch.zeros(9, 8, device="cuda")
    y, g = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda")
    for args in [(h.half(), w, y), (h, w[:, :7], y), (h, w, y.long()), (h, w, y[:3]), (h, w, y.cpu()), (h.t(), w, y),
                 (h, w[:0], y), (h, w, y.view(4, 1, 1)), (torch.zeros(4, 5000, device="cuda"), torch.zeros(9, 5000, device="cuda"), y)]:
        with pytest.raises(ValueError):
            Softmax.loss(*args)
    loss, lse = Softmax.loss(h, w, y)
    for bad in [(lse[:3], g), (lse.double(), g), (lse, g[:3]), (lse, g.cpu()), (lse, g.half())]:
        with pytest.raises(ValueError):
            Softmax.grad(h, w, y, *bad)
    with pytest.raises(ValueError):
        Softmax.grad(h, w, y, lse, g, dweight=torch.zeros(8, 8, device="cuda"))


def test_many_short_calls_in_a_row():
    """Passes of about 50 us that nothing waits between, on inputs in turn: the same bits every time."""
    from bidmach_b200 import Softmax
    sets = []
    for seed in (1, 2, 3):
        x = [v.cuda() for v in inputs(1908, 4000, 80, 1, "bf16", seed=seed)]
        sets.append((x, run(*x)))
    last = {}
    for i in range(1500):
        x, want = sets[i % 3]
        loss, lse = Softmax.loss(*x[:3])
        last[i % 3] = (loss, lse, *Softmax.grad(*x[:3], lse, x[3]))
    torch.cuda.synchronize()
    for i, (x, want) in enumerate(sets):
        assert all(torch.equal(a, b) for a, b in zip(last[i], want))


def test_outputs_that_share_memory_are_refused():
    from bidmach_b200 import Softmax
    h, w = (torch.randn(n, 32, device="cuda") for n in (40, 50))
    y = torch.zeros(40, dtype=torch.int32, device="cuda")
    loss, lse = Softmax.loss(h, w, y)
    one = torch.ones((), device="cuda")
    for out in (dict(dhidden=h), dict(dweight=w), dict(dhidden=w[:40]), dict(dhidden=w[10:], dweight=w.clone()),
                dict(zip(("dhidden", "dweight"), (lambda b: (b[:40], b[:50]))(torch.empty(60, 32, device="cuda"))))):
        with pytest.raises(ValueError, match="overlaps"):
            Softmax.grad(h, w, y, lse, one, **out)
    with pytest.raises(ValueError, match="overlaps"):
        Softmax.loss(h, w, y, loss=loss, lse=loss)
    # the gradients beside their operands in one buffer each
    both = torch.zeros(50, 64, device="cuda")
    both[:, :32] = w
    want = Softmax.grad(h, w, y, lse, one)
    got = Softmax.grad(h, both[:, :32], y, lse, one, dweight=both[:, 32:])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(both[:, :32], w)


def test_short_calls_on_two_streams():
    """Kernels of a few tiles from two streams, which follow one another on an SM without a gap: no arrival of
    one reaches the next, so every call gives the bits of the call alone."""
    from bidmach_b200 import Softmax
    sets = []
    for n, vocab, dim, t in ((20, 600, 64, "bf16"), (40, 300, 72, "f32"), (300, 700, 16, "f16"), (17, 260, 320, "bf16")):
        x = [v.cuda() for v in inputs(n, vocab, dim, 1, t, seed=5)]
        sets.append((x, run(*x)))
    torch.cuda.synchronize()
    streams, last = [torch.cuda.Stream(), torch.cuda.Stream()], {}
    for i in range(800):
        k = i % len(sets)
        with torch.cuda.stream(streams[(i // len(sets) + i) % 2]):
            x = sets[k][0]
            loss, lse = Softmax.loss(*x[:3])
            last[k, i % 2] = (loss, lse, *Softmax.grad(*x[:3], lse, x[3]))
    torch.cuda.synchronize()
    for (k, _), got in last.items():
        assert all(torch.equal(a, b) for a, b in zip(got, sets[k][1]))


@pytest.mark.parametrize("n", [9, 90])
@pytest.mark.parametrize("t,size", [("f32", 1.0), ("f32", 1e-4), ("f32", 3e5), ("f16", 1.0), ("bf16", 1e-4)])
@pytest.mark.parametrize("where", ["hidden", "gloss"])
def test_not_finite_numbers_stay_in_their_rows(n, t, size, where):
    """A NaN and an infinity in rows of hidden, or among the rows' factors: loss, lse and dhidden of all other
    rows are within the usual bounds, whatever the size of the numbers beside them."""
    hidden, weight, targets, gloss = inputs(n, 300, 32, 1, t)
    hidden, weight = (hidden.float() * size).to(TYPES[t]), (weight.float() / size).to(TYPES[t])
    gloss = gloss * (1e-3 if t == "f16" else 1.0)     # d of fp16 has to be scaled up
    targets[:, 0] = torch.arange(n, dtype=torch.int32)
    good = torch.ones(n, dtype=torch.bool)
    good[1] = good[3] = False
    broken = [hidden.clone(), weight, targets, gloss.clone()]
    if where == "hidden":
        broken[0][1, 3], broken[0][3, 5] = float("nan"), float("inf")
    else:
        broken[3][1], broken[3][3] = float("nan"), float("inf")
    got = [x.cpu() for x in run(*broken)]
    clean = run(hidden, weight, targets, gloss)      # its dweight stands in for the broken one, which is NaN
    loss, lse, dh = (torch.where(good.view(-1, *[1] * (x.dim() - 1)), x, c.cpu()) for x, c in zip(got[:3], clean))
    assert all(torch.isfinite(x).all() for x in (loss, lse, dh))
    hold((loss, lse, dh, clean[3].cpu()), hidden, weight, targets, gloss, t)
    assert torch.isnan(got[2][~good]).any(1).all()


@pytest.mark.parametrize("n", [1, 4, 16, 200])
@pytest.mark.parametrize("t", list(TYPES))
def test_loss_of_sure_rows_is_not_negative(n, t):
    """Rows whose target has nearly all of the probability: the loss is the difference of two rounded numbers."""
    for seed in range(4):
        hidden, weight, targets, gloss = inputs(n, 700, 96, 3, t, seed=seed, size=12.0)
        top = (hidden.double() @ weight.double().T).argmax(1)
        targets[:] = top[:, None].int()
        got = run(hidden, weight, targets, gloss)
        assert (got[0] >= 0).all()
        hold(got, hidden, weight, targets, gloss, t)


def test_the_next_call_says_that_a_kernel_gave_up():
    """The flag that such a kernel raises, raised here by the host: the next call reports it and is then done with it,
    before it has launched anything."""
    from bidmach_b200 import Softmax, _lib
    hidden, weight, targets, gloss = (x.cuda() for x in inputs(50, 300, 32, 1, "bf16"))
    loss, lse = Softmax.loss(hidden, weight, targets)
    flag, count = _lib.load().w2v_softmax_fault(), _lib.load().w2v_launch_count
    for call in (lambda: Softmax.loss(hidden, weight, targets), lambda: Softmax.grad(hidden, weight, targets, lse, gloss),
                 Softmax.check):
        flag[0], before = 1, count()
        with pytest.raises(RuntimeError, match="702|gave up|timed out|time"):
            call()
        assert count() == before and flag[0] == 0
        call()
    assert torch.equal(Softmax.loss(hidden, weight, targets)[0], loss)


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_no_room_for_copies_that_are_not_made(t):
    """A 200 MB matrix that TMA reads where it lies: the loss allocates its 13 MB of row parts."""
    from bidmach_b200 import Softmax
    hidden = torch.randn(1024, 512, device="cuda").to(TYPES[t])
    weight = torch.zeros(200000, 512, dtype=TYPES[t], device="cuda")
    targets = torch.zeros(1024, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    _, lse = Softmax.loss(hidden, weight, targets)
    assert torch.cuda.max_memory_allocated() - before < 20 << 20
    assert (lse - 12.206072645530174).abs().max() < 1e-5      # log 200000


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("dim", [255, 256, 257, 264, 272])
def test_both_sides_of_the_few_rows_border(n, dim, t):
    """Few rows go one way or another by type, width and alignment; a workspace of the size that is asked for
    without flags is enough for each."""
    from bidmach_b200 import _lib
    x = inputs(n, 900, dim, 2, t)
    hold(run(*x), *x, t)
    h, w, y, g = (v.cuda() for v in x)
    lib, kind = _lib.load(), list(TYPES).index(t)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ok = (h.data_ptr(), dim, w.data_ptr(), dim, y.data_ptr(), n, 900, dim, 2, kind)
    for grad in (0, 1):
        size = lib.w2v_softmax_workspace(n, 900, dim, 2, kind, grad)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.current_stream().cuda_stream
        if grad:
            err = lib.w2v_softmax_grad(*ok, lse.data_ptr(), g.data_ptr(), 1, dh.data_ptr(), dim, dw.data_ptr(), dim,
                                       work.data_ptr(), size, stream)
        else:
            err = lib.w2v_softmax_loss(*ok, loss.data_ptr(), lse.data_ptr(), work.data_ptr(), size, stream)
        assert err == 0
        torch.cuda.synchronize()
    hold((loss, lse, dh, dw), *x, t)


def test_the_first_call_of_a_process_is_captured():
    """What a process sets up once is allowed in a capture too."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from bidmach_b200 import Softmax
h, w = torch.randn(40, 64, device="cuda"), torch.randn(300, 64, device="cuda")
y, one = torch.zeros(40, dtype=torch.int32, device="cuda"), torch.ones((), device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss, lse = Softmax.loss(h, w, y)
    dh, dw = Softmax.grad(h, w, y, lse, one)
graph.replay()
torch.cuda.synchronize()
again = Softmax.loss(h, w, y)
assert torch.equal(loss, again[0]) and all(torch.equal(a, b) for a, b in zip((dh, dw), Softmax.grad(h, w, y, lse, one)))
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]
