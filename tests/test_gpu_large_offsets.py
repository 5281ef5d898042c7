"""Matrices of more than 2^31 elements: the rows at their end are computed like those of a small matrix."""
import pytest
import torch

pytestmark = pytest.mark.gpu
ROWS, DIM = 1_100_000, 2048          # 2.25e9 elements
TAIL = 300


@pytest.fixture(scope="module")
def matrix():
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 60 GB")
    m = torch.zeros(ROWS, DIM, dtype=torch.bfloat16, device="cuda")
    m[-TAIL:] = torch.randn(TAIL, DIM, device="cuda") * 0.1
    yield m
    del m
    torch.cuda.empty_cache()


def test_rows_by_ids(matrix):
    from bidmach_b200 import EmbedRows
    ids = torch.randint(ROWS - TAIL, ROWS, (500,), device="cuda").int()
    assert torch.equal(EmbedRows.forward(ids, matrix), matrix[ids.long()])
    grad = torch.randn(500, DIM, device="cuda").bfloat16()
    got = EmbedRows.backward(ids, grad, ROWS)
    assert torch.equal(got[-TAIL:], EmbedRows.backward(ids - (ROWS - TAIL), grad, TAIL))
    assert not got[:1000].any() and not got[ROWS // 2: ROWS // 2 + 1000].any()


@pytest.mark.parametrize("n", [3, 40])
def test_softmax(matrix, n):
    """All words but the last are zero rows, logit 0: lse = log(ROWS - TAIL + sum over the last).  The tolerance
    of a logit is 2^-18 of the magnitudes it sums, which are below 2^9 here; the gradients are held to
    four half steps of their type."""
    from bidmach_b200 import Softmax
    h = torch.randn(n, DIM, device="cuda").bfloat16()
    y = torch.randint(ROWS - TAIL, ROWS, (n, 2), device="cuda").int()
    loss, lse = Softmax.loss(h, matrix, y)
    x = h.double() @ matrix[-TAIL:].double().T
    z = torch.log(ROWS - TAIL + x.exp().sum(1))
    at = (y - (ROWS - TAIL)).long()
    assert (lse.double() - z).abs().max() <= 2.0 ** -9
    assert (loss.double() - (2 * z[:, None] - x.gather(1, at) * 2).mean(1)).abs().max() <= 2.0 ** -7
    g = torch.full((1,), 1.0, device="cuda")
    dh, dw = Softmax.grad(h, matrix, y, lse, g)
    d = 2 * (x - z[:, None]).exp()
    d.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    w = matrix[-TAIL:].double()
    for got, want, size in ((dh, d @ w, d.abs() @ w.abs()), (dw[-TAIL:], d.T @ h.double(), d.abs().T @ h.double().abs())):
        assert ((got.double() - want).abs() <= 4 * 2.0 ** -9 * size + 2.0 ** -20).all()
    del dw


def test_adamw(matrix):
    from bidmach_b200 import AdamW
    o = AdamW.Opts(bits=8)
    p, tail = matrix.view(-1), matrix[-TAIL:].reshape(-1).clone()
    g = torch.zeros_like(p)
    g[-TAIL * DIM:] = torch.randn(TAIL * DIM, device="cuda") * 1e-2
    a, b = AdamW([p], o), AdamW([tail], o)
    for _ in range(2):
        a.step([g])
        b.step([g[-TAIL * DIM:]])
    assert torch.equal(p[-TAIL * DIM:], tail) and torch.equal(a.m[0][-TAIL * DIM:], b.m[0])
    assert not p[:5000].any()
