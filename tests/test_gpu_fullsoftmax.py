"""Word2Vec with the softmax over the whole vocabulary: the operators together, as a minibatch uses them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def rows_of(words, lb, ub, nskip):
    ids, targets = [], []
    for k in range(len(words)):
        if words[k] < 0:
            continue
        c = [words[i] for i in range(max(0, k - nskip), min(len(words), k + nskip + 1))
             if i != k and words[i] >= 0 and lb[i] <= k - i <= ub[i]]
        if c:
            ids.append(words[k])
            targets.append(c + [-1] * (2 * nskip - len(c)))
    return np.array(ids, np.int32), np.array(targets, np.int32).reshape(-1, 2 * nskip)


@pytest.mark.parametrize("n", [1, 2, 31, 256, 257, 5000, 300000])
@pytest.mark.parametrize("nskip", [1, 5, 9])
def test_window_rows(n, nskip):
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    if n == 300000 and nskip != 5:
        return
    rng = np.random.default_rng(n + nskip)
    words = rng.integers(0, 50, n).astype(np.int32)
    words[rng.random(n) < 0.5] = -1
    lb = -np.minimum(rng.integers(0, nskip + 1, n), np.arange(n)).astype(np.int32)
    ub = np.minimum(rng.integers(0, nskip + 1, n), n - 1 - np.arange(n)).astype(np.int32)
    m = Word2Vec(Opts(vocabSize=50, dim=4, nskip=nskip))
    ids, targets = m.windowRows(*(torch.from_numpy(x).cuda() for x in (words, lb, ub)))
    want = rows_of(words, lb, ub, nskip)
    np.testing.assert_array_equal(ids.cpu().numpy(), want[0])
    np.testing.assert_array_equal(targets.cpu().numpy(), want[1])
    # the pairs of the positive update
    assert (want[1] >= 0).sum() == sum(words[i] >= 0 and words[i + j] >= 0 for i in range(n)
                                       for j in range(lb[i], ub[i] + 1) if j)


def model_of(vocab, dim, n, **more):
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    # a large eps: the step is then a smooth function of the gradient, so rounding does not turn its sign
    o = Opts(vocabSize=vocab, dim=dim, nskip=5, wsample=1e-2, lrate=0.02, texp=0.5, fullSoftmax=True, adamEps=1e-2,
             wdecay=0.01, seed=5, **more)
    m = Word2Vec(o).init(n)
    gen = torch.Generator(device="cuda").manual_seed(1)
    m.modelmats[0].copy_(torch.randn(vocab, dim, generator=gen, device="cuda") * 0.5)
    m.modelmats[1].copy_(torch.randn(vocab, dim, generator=gen, device="cuda") * 0.5)
    return m


def tokens(vocab, n, seed):
    from bidmach_b200.corpus import zipf_corpus
    return zipf_corpus(vocab, n, 1.0, seed=seed, doc_len=60)


def formula(ids, targets, context, centre):
    """Mean loss over the pairs, its gradients and the magnitudes that they are sums of, in 64 bits."""
    h, w, y = context[ids.long()].double(), centre.double(), targets.long()
    there = y >= 0
    pairs = there.sum().double()
    x = h @ w.T
    lse = torch.logsumexp(x, 1)
    loss = torch.where(there, lse[:, None] - x.gather(1, y.clamp(min=0)), 0.0).sum() / pairs
    d = torch.exp(x - lse[:, None]) * there.sum(1, keepdim=True)
    d = d.scatter_add(1, y.clamp(min=0), -there.double()) / pairs
    dctx, sctx = torch.zeros_like(context.double()), torch.zeros_like(context.double())
    dctx.index_add_(0, ids.long(), d @ w)
    sctx.index_add_(0, ids.long(), d.abs() @ w.abs())
    return float(loss), dctx, d.T @ h, sctx, d.abs().T @ h.abs()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("vocab,dim,n", [(300, 20, 700), (1500, 100, 4096)])
def test_minibatch_against_the_formula(vocab, dim, n, bits):
    """Two training minibatches.  The gradients are good to 2^-16 of the magnitudes they sum (fp32 sums and
    22-bit operands).  The corrected moments are averages of the gradients so far (v of their squares), so m
    and sqrt(v) are off by at most the largest of their errors, that of a step whose own gradient is zero
    included, and the step by 2 lrate / eps times that while sqrt(v) + eps >= eps.  The 8-bit moments of
    the first step put the second off by a 16th of its size."""
    m = model_of(vocab, dim, n, momentBits=bits)
    o = m.opts
    context, centre = (x.double().clone() for x in m.modelmats)
    mom = [[torch.zeros_like(context), torch.zeros_like(context)], [torch.zeros_like(centre), torch.zeros_like(centre)]]
    off = [torch.zeros_like(context), torch.zeros_like(centre)]
    for t, seed in ((1, 3), (2, 4)):
        toks = torch.from_numpy(tokens(vocab, n, seed)).cuda()
        m._batches = 10 * t
        ids, targets, pairs = m._softmaxRows(toks)
        ids, targets = ids.clone(), targets.clone()
        assert pairs == int((targets >= 0).sum())
        start = [x.clone() for x in m.modelmats]
        _, dctx, dcen, sctx, scen = formula(ids, targets, start[0], start[1])
        m._batches = 10 * t
        m.dobatch([toks], 0, 1000 * t)
        lr = o.lrate * (1000 * t / 1000) ** -o.texp
        for i, (g, size) in enumerate(((dctx, sctx), (dcen, scen))):
            mo, ve = mom[i]
            mo.mul_(0.9).add_(0.1 * g)
            ve.mul_(0.999).add_(0.001 * g * g)
            off[i] = torch.maximum(off[i], size)
            step = lr / (1 - 0.9 ** t) * mo / ((ve / (1 - 0.999 ** t)).sqrt() + o.adamEps)
            want = start[i].double() * (1 - lr * o.wdecay) - step
            bound = 2 * lr / o.adamEps * 2.0 ** -16 * off[i] + 2.0 ** -22 * (start[i].double().abs() + step.abs())
            if bits == 8 and t == 2:
                bound = bound + lr * 0.1
            assert torch.all((m.modelmats[i].double() - want).abs() <= bound), (t, i)
    assert m._adam_steps == 2


def test_score_is_the_mean_log_likelihood():
    m = model_of(800, 64, 3000)
    toks = torch.from_numpy(tokens(800, 3000, 9)).cuda()
    m._batches = 4
    score = m.evalbatch([toks], 0, 0)
    m._batches = 4
    ids, targets, _ = m._softmaxRows(toks)
    want = -formula(ids, targets, *m.modelmats)[0]
    assert abs(score - want) <= 2.0 ** -18 * abs(want)
    m._batches = 4
    assert m.evalbatchg([toks.cpu()], 0, 0) == score


def test_learner_runs_and_checkpoints(tmp_path):
    """The learner drives it as it does the sampled objective; both minibatch forms count the same pairs."""
    from bidmach_b200 import Learner, MatSource, Word2Vec
    from bidmach_b200.learner import LearnerOpts
    from bidmach_b200.word2vec import Opts
    o = Opts(vocabSize=500, dim=24, lrate=1e-2, fullSoftmax=True, wsample=1e-2, momentBits=8)
    learner = Learner(MatSource(tokens(500, 20000, 1), 2000), Word2Vec(o), LearnerOpts(npasses=1)).train()
    assert all(np.isfinite(s) and s < 0 for s in learner.reslist)
    m = learner.model
    assert all(torch.isfinite(x).all() for x in m.modelmats)
    m.save(str(tmp_path) + "/")
    other = Word2Vec(Opts(vocabSize=500, dim=24)).load(str(tmp_path) + "/")
    assert other.opts.fullSoftmax and other.opts.momentBits == 8
    assert all(torch.equal(a, b) for a, b in zip(other.modelmats, m.modelmats))


def test_a_minibatch_without_pairs():
    """Sentences of one word: nothing to learn, nothing changes."""
    m = model_of(40, 8, 64)
    toks = torch.stack([torch.arange(64) % 40, torch.arange(64)], 1).int().cuda()
    before = [x.clone() for x in m.modelmats]
    assert m.dobatchg([toks.cpu()], 0, 64) == 0
    assert m.evalbatch([toks], 0, 64) == 0.0
    assert all(torch.equal(a, b) for a, b in zip(before, m.modelmats))


def test_refused_with_slices():
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    with pytest.raises(ValueError, match="nSlices"):
        Word2Vec(Opts(fullSoftmax=True, nSlices=2))


def test_window_rows_refuses():
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    m = Word2Vec(Opts(vocabSize=50, dim=4))
    w = torch.zeros(10, dtype=torch.int32, device="cuda")
    for args in ((w, w[:9], w), (w, w, w[:9]), (w, w, w.cpu()), (w[::2], w[:5], w[:5]), (w, w.float(), w)):
        with pytest.raises(ValueError):
            m.windowRows(*args)
    with pytest.raises(ValueError, match="nskip"):
        Word2Vec(Opts(vocabSize=50, dim=4, nskip=513)).windowRows(w, w, w)
