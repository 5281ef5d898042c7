"""Rows by ids and their gradient against 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ids_of(kind, n, vocab, seed):
    rng = np.random.default_rng(seed)
    if kind == "one":
        ids = np.full(n, vocab // 2)
    elif kind == "zipf":
        ids = np.minimum(np.exp(rng.random(n) * np.log(vocab + 1.0)).astype(int) - 1, vocab - 1)
    elif kind == "none":
        ids = np.full(n, -1)
    elif kind == "distinct":
        ids = rng.permutation(max(n, vocab))[:n] % vocab
    else:      # dropped words and ids behind the matrix among the others
        ids = rng.integers(-3, vocab + 3, n)
    return torch.from_numpy(ids.astype(np.int32))


CASES = [(1, 1, 1), (1, 50, 7), (31, 9, 300), (32, 9, 300), (33, 3, 256), (64, 5, 8), (97, 1000, 301), (1000, 20, 1280),
         (5000, 3000, 100), (20011, 257, 33)]


@pytest.mark.parametrize("kind", ["zipf", "one", "none", "mixed", "distinct"])
@pytest.mark.parametrize("n,vocab,dim", CASES)
@pytest.mark.parametrize("t", list(TYPES))
def test_rows_and_gradient(kind, n, vocab, dim, t):
    from bidmach_b200 import EmbedRows
    ids = ids_of(kind, n, vocab, n + dim)
    gen = torch.Generator().manual_seed(n)
    matrix = torch.randn(vocab, dim, generator=gen).to(TYPES[t])
    grad = torch.randn(n, dim, generator=gen).to(TYPES[t])
    there = (ids >= 0) & (ids < vocab)
    at = ids.long().clamp(0, vocab - 1)
    rows = EmbedRows.forward(ids.cuda(), matrix.cuda())
    assert torch.equal(rows.cpu(), torch.where(there[:, None], matrix[at], torch.zeros((), dtype=TYPES[t])))
    got = EmbedRows.backward(ids.cuda(), grad.cuda(), vocab)
    again = EmbedRows.backward(ids.cuda(), grad.cuda(), vocab)
    assert torch.equal(got, again)
    masked = torch.where(there[:, None], grad.double(), 0.0)
    want = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, at, masked)
    size = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, at, masked.abs())
    count = torch.zeros(vocab, 1, dtype=torch.float64).index_add_(0, at, there.double()[:, None])
    # a sum of k terms has at most k - 1 roundings, each of a partial sum no larger than the terms' sizes
    half = torch.finfo(TYPES[t]).eps / 2
    bound = (count - 1).clamp(min=0) * 2.0 ** -24 * size * 1.001
    if t != "f32":
        bound = bound + half * (want.abs() + bound) + (2.0 ** -25 if t == "f16" else 0)
    assert torch.all((got.double().cpu() - want).abs() <= bound)


def test_strided_and_unaligned():
    """Rows inside wider matrices, at odd offsets: what lies between them stays."""
    from bidmach_b200 import EmbedRows
    ids = ids_of("mixed", 500, 60, 1).cuda()
    for off, dim in [(0, 40), (1, 40), (3, 13), (8, 64)]:
        base = torch.randn(60, 80, device="cuda")
        g = torch.randn(500, 80, device="cuda")
        m, gr = base[:, off:off + dim], g[:, off:off + dim]
        out = torch.full((500, 80), 5.0, device="cuda")
        EmbedRows.forward(ids, m, out=out[:, off:off + dim])
        assert torch.equal(out[:, off:off + dim], EmbedRows.forward(ids, m.contiguous()))
        keep = torch.ones(80, dtype=torch.bool)
        keep[off:off + dim] = False
        assert (out[:, keep] == 5.0).all()
        dm = torch.full((60, 80), 5.0, device="cuda")
        EmbedRows.backward(ids, gr, 60, out=dm[:, off:off + dim])
        assert torch.equal(dm[:, off:off + dim], EmbedRows.backward(ids, gr.contiguous(), 60))
        assert (dm[:, keep] == 5.0).all()


def test_no_tokens():
    from bidmach_b200 import EmbedRows
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert EmbedRows.forward(none, torch.randn(4, 6, device="cuda")).shape == (0, 6)
    assert torch.equal(EmbedRows.backward(none, torch.empty(0, 6, device="cuda"), 4), torch.zeros(4, 6, device="cuda"))


def test_two_streams_and_a_graph():
    from bidmach_b200 import EmbedRows
    ids = [ids_of("zipf", 30000, 500, s).cuda() for s in (1, 2)]
    grads = [torch.randn(30000, 96, device="cuda") for _ in ids]
    want = [EmbedRows.backward(i, g, 500) for i, g in zip(ids, grads)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(EmbedRows.backward(ids[k], grads[k], 500))
    graphs, outs = [], []
    torch.cuda.synchronize()
    for k in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(EmbedRows.backward(ids[k], grads[k], 500))
        graphs.append(graph)
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        assert torch.equal(outs[k], want[k]) and all(torch.equal(x, want[k]) for x in got[k])


def test_refusals_on_the_device():
    from bidmach_b200 import EmbedRows
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    m = torch.zeros(5, 6, device="cuda")
    for bad in [(ids.long(), m), (ids, m.double()), (ids, m.t()), (ids.cpu(), m), (ids[::2], m), (ids, m.cpu())]:
        with pytest.raises(ValueError):
            EmbedRows.forward(*bad)
    with pytest.raises(ValueError):
        EmbedRows.forward(ids, m, out=torch.zeros(3, 6, device="cuda"))
    for args in [(ids, m, 5), (ids, m[:4], 0), (ids, m[:4].expand(4, 6).double(), 5), (ids, m[:1].expand(4, 6), 5)]:
        with pytest.raises(ValueError):
            EmbedRows.backward(*args)


def test_outputs_that_share_memory_are_refused():
    from bidmach_b200 import EmbedRows
    m = torch.randn(9, 8, device="cuda")
    ids = torch.arange(9, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        EmbedRows.forward(ids, m, out=m)
    with pytest.raises(ValueError, match="overlaps"):
        EmbedRows.backward(ids, m, 9, out=m)


def test_more_columns_than_the_kernels_take_are_refused():
    from bidmach_b200 import EmbedRows
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    wide = torch.zeros(3, 65537, device="cuda")
    with pytest.raises(ValueError, match="columns"):
        EmbedRows.forward(ids, wide)
    with pytest.raises(ValueError, match="columns"):
        EmbedRows.backward(ids, wide, 5)
    assert EmbedRows.forward(ids, wide[:, :65536].contiguous()).shape == (3, 65536)
