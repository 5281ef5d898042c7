"""Softmax in fp32 where rows differ in size by many orders: the results of ordinary rows and words are as good as
without the others.

Tolerances as in test_gpu_softmax.py (E there), from the magnitudes of the rows and words that are looked at: a
row without targets has d = 0 exactly and a word whose logit lies 200 or more below the largest has probability 0
in fp32, so neither adds to the others' errors.  An operand keeps 22 bits of its own row's largest number."""
import pytest
import torch

from test_gpu_softmax import U, formula, inputs, run

pytestmark = pytest.mark.gpu


def hold_some(got, hidden, weight, targets, gloss, rows=None, words=None, half=2.0 ** -21, out=U):
    """Asserts the bounds for some rows of (loss, lse, dh) and, where `words` are given, for these of dw."""
    x = [v.cuda() for v in (hidden, weight, targets, gloss)]
    f = formula(*x)
    n, dim = hidden.shape
    vocab = weight.shape[0]
    rows = torch.ones(n, dtype=torch.bool) if rows is None else rows
    kept = torch.ones(vocab, dtype=torch.bool) if words is None else words
    rows, kept = rows.cuda(), kept.cuda()
    h, w = x[0][rows].double().abs(), x[1][kept].double().abs()
    prob, d, hit, k = f["prob"][rows][:, kept].abs(), f["d"][rows][:, kept].abs(), f["hit"][rows][:, kept].abs(), f["k"][rows]
    loss, lse, dh, dw = (v.double().cuda() for v in got)
    e = (dim * U + 2.0 ** -20) * (h @ w.T).amax(1)
    lse_off = e + 2.0 ** -20 * (1 + f["lse"][rows].abs())
    assert torch.all((lse - f["lse"])[rows].abs() <= lse_off)
    assert torch.all((loss - f["loss"])[rows].abs() <= k * (lse_off + e) + k * U * f["loss"][rows].abs())
    own = x[3][rows].double().abs() * k
    off = 1.001 * (e + lse_off + 2.0 ** -20)[:, None] * prob + half * d + U * hit
    off = off + 2.0 ** -48 * own[:, None]          # smallest step of d beside its own row's factor
    grow = 2 * U
    bound = off @ w + (grow * (vocab + 64) + 2.0 ** -20) * (d @ w)
    bound = bound + 2 * out * (f["dh"][rows].abs() + bound) + 2.0 ** -126
    assert torch.all((dh - f["dh"])[rows].abs() <= bound)
    if words is not None:
        bound = off.T @ h + (grow * (n + 64) + 2.0 ** -20) * (d.T @ h)
        bound = bound + 2 * out * (f["dw"][kept].abs() + bound) + 2.0 ** -126
        assert torch.all((dw - f["dw"])[kept].abs() <= bound)


SIZES = [(12, 300, 64), (17, 300, 100), (100, 513, 64), (129, 1000, 16), (300, 777, 1000), (515, 2049, 520), (700, 40000, 40)]


@pytest.mark.parametrize("size", [2.0 ** 15, 1e6, 1e9, 1e12])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_a_large_row_without_targets(n, vocab, dim, size):
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, "f32")
    hidden[7] *= size
    targets[7] = -1
    rows = torch.ones(n, dtype=torch.bool)
    rows[7] = False
    got = run(hidden, weight, targets, gloss)
    hold_some(got, hidden, weight, targets, gloss, rows, torch.ones(vocab, dtype=torch.bool))
    assert not got[2][7].any()


@pytest.mark.parametrize("size", [1e6, 1e12])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_a_large_row_with_targets(n, vocab, dim, size):
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, "f32")
    hidden[3] *= size
    targets[3] = 5
    rows = torch.ones(n, dtype=torch.bool)
    rows[3] = False
    hold_some(run(hidden, weight, targets, gloss), hidden, weight, targets, gloss, rows)


@pytest.mark.parametrize("size", [1e6, 1e12])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_a_large_word(n, vocab, dim, size):
    """A word of large negative logits: probability zero everywhere."""
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, "f32")
    hidden[:, 0] = hidden[:, 0].abs() + 0.5
    weight[11] = 0.0
    weight[11, 0] = -size
    targets[targets == 11] = 12
    words = torch.ones(vocab, dtype=torch.bool)
    words[11] = False
    got = run(hidden, weight, targets, gloss)
    hold_some(got, hidden, weight, targets, gloss, words=words)
    assert not got[3][11].any()


@pytest.mark.parametrize("size", [1e-6, 1e-12])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_a_small_row_and_a_small_word(n, vocab, dim, size):
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, "f32")
    hidden[5] *= size
    weight[4] *= size
    targets[5], targets[6] = 4, 4
    hold_some(run(hidden, weight, targets, gloss), hidden, weight, targets, gloss, words=torch.ones(vocab, dtype=torch.bool))


def test_several_pieces_of_parts():
    """Row blocks and pieces of the vocabulary, with operands in three parts."""
    hidden, weight, targets, gloss = inputs(8300, 12000, 24, 1, "f32")
    hidden[8299] *= 1e9
    targets[8299] = -1
    rows = torch.arange(8300) < 8299
    hold_some(run(hidden, weight, targets, gloss), hidden, weight, targets, gloss, rows, torch.ones(12000, dtype=torch.bool))


@pytest.mark.parametrize("n", [12, 300])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_factors_over_many_decades(n, t):
    """Each row's gradient is good beside its own factor, not the largest one."""
    hidden, weight, targets, _ = inputs(n, 900, 72, 2, t)
    gloss = torch.logspace(0, -12, n)[torch.randperm(n, generator=torch.Generator().manual_seed(2))]
    half = torch.finfo(torch.bfloat16).eps / 2 if t == "bf16" else 2.0 ** -21
    hold_some(run(hidden, weight, targets, gloss), hidden, weight, targets, gloss, words=torch.ones(900, dtype=torch.bool),
              half=half, out=half if t == "bf16" else U)


@pytest.mark.parametrize("big,small", [(2.0 ** 120, 2.0 ** -118), (2.0 ** -118, 2.0 ** 120)])
def test_operands_at_the_ends_of_the_range(big, small):
    """Products of ordinary size from operands near the largest and the smallest numbers."""
    hidden, weight, targets, gloss = inputs(40, 200, 32, 1, "f32")
    x = (hidden * big, weight * small, targets, gloss)
    got = run(*x)
    f = formula(*x)
    e = (32 * U + 2.0 ** -20) * (x[0].double().abs() @ x[1].double().abs().T).amax(1) + 2.0 ** -20 * (1 + f["lse"].abs())
    assert torch.all((got[1].cpu().double() - f["lse"]).abs() <= e)
    assert torch.isfinite(got[2]).all() and torch.isfinite(got[3]).all()


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 13.5])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_a_large_row_that_one_scale_still_serves(n, vocab, dim, size):
    """Just below the border to three parts.  dw is held to 22 bits of its rows' largest numbers: an element far
    below its row's largest has fewer bits of its own."""
    hidden, weight, targets, gloss = inputs(n, vocab, dim, 2, "f32")
    hidden[7] *= size
    targets[7] = -1
    rows = torch.ones(n, dtype=torch.bool)
    rows[7] = False
    got = run(hidden, weight, targets, gloss)
    hold_some(got, hidden, weight, targets, gloss, rows)
    f = formula(hidden, weight, targets, gloss)
    h = hidden.double().abs()[rows].amax(1, keepdim=True).expand(-1, dim)
    size = f["d"][rows].abs().T @ h
    e = (dim * U + 2.0 ** -20) * (hidden.double().abs()[rows] @ weight.double().abs().T).amax(1) + 2.0 ** -20 * (1 + f["lse"][rows].abs())
    off = (2 * e + 2.0 ** -20)[:, None] * f["prob"][rows].abs()
    bound = 1.001 * off.T @ h + (2 * U * (n + 64) + 2.0 ** -20 + 2.0 ** -22) * size + 2 * U * f["dw"].abs() + 2.0 ** -126
    assert torch.all((got[3].double().cpu() - f["dw"]).abs() <= bound)
