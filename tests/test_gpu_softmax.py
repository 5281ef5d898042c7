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
    loss, lse, dh, dw = (x.double().cpu() for x in got)
    assert torch.all((lse - f["lse"]).abs() <= lse_off)
    assert torch.all((loss - f["loss"]).abs() <= f["k"] * (lse_off + e) + f["k"] * U * f["loss"].abs())
    # what d may be off by: its probabilities, then its rounding (fp32 keeps 22 bits of it)
    half = torch.finfo(TYPES[t]).eps / 2
    rel = (e + lse_off + 2.0 ** -20)[:, None]
    off = 1.001 * rel * f["prob"] + (half if t != "f32" else 2.0 ** -21) * f["d"].abs() + U * f["hit"]
    if t != "bf16":    # fp16 parts of d: steps of 2^-25 where the largest row's is 2^14 to 2^15
        top = (gloss.double() * f["k"]).amax()
        off = off + 2.0 ** (-38 if t == "f16" else -48) * top
    grow = 2 * U       # truncated accumulation, and the joining of pieces
    for got_g, want, other, terms, count in ((dh, f["dh"], w, f["d"].abs(), vocab), (dw, f["dw"], h, f["d"].abs().T, n)):
        o = off if other is w else off.T
        size = terms @ other
        bound = o @ other + (grow * (count + 64) + 2.0 ** -20) * size
        bound = bound + (half + U) * (want.abs() + bound) + (2.0 ** -25 if t == "f16" else 0)
        assert torch.all((got_g - want).abs() <= bound)


def run(hidden, weight, targets, gloss):
    from bidmach_b200 import Softmax
    h, w, y, g = hidden.cuda(), weight.cuda(), targets.cuda(), gloss.cuda()
    loss, lse = Softmax.loss(h, w, y)
    return (loss, lse, *Softmax.grad(h, w, y, lse, g))


SIZES = [(1, 1, 1), (1, 1000, 256), (2, 33, 7), (3, 257, 300), (5, 1001, 64), (8, 4097, 100), (9, 1, 1), (9, 255, 64),
         (16, 300, 301), (127, 256, 128), (128, 513, 37), (129, 1000, 16), (200, 5003, 300), (300, 777, 1000),
         (515, 2049, 520), (64, 40, 4096)]


@pytest.mark.parametrize("n,vocab,dim", SIZES)
@pytest.mark.parametrize("labels", [1, 5])
@pytest.mark.parametrize("t", list(TYPES))
def test_against_64_bits(n, vocab, dim, labels, t):
    x = inputs(n, vocab, dim, labels, t)
    hold(run(*x), *x, t)
