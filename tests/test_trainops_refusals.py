"""What the training operators refuse before they touch a GPU."""
import ctypes as C

import pytest
import torch

from bidmach_b200 import AdamW, EmbedRows, _lib


def test_adamw_options_and_tensors():
    p = torch.zeros(8)
    for o in (dict(bits=16), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=0.0), dict(wdecay=-1.0)):
        with pytest.raises(ValueError):
            AdamW([p], AdamW.Opts(**o))
    for params in ([], [p], [torch.zeros(3, dtype=torch.int32)], [torch.zeros(3, dtype=torch.float64)]):
        with pytest.raises(ValueError):
            AdamW(params)


def test_embed_wants_device_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        EmbedRows.forward(torch.zeros(3, dtype=torch.int32), torch.zeros(4, 4))
    with pytest.raises(ValueError, match="int32"):
        EmbedRows.backward(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4), 5)


def test_c_entries_refuse_without_a_launch():
    lib = _lib.load()
    before = lib.w2v_launch_count()
    t = (_lib.W2VAdamwTensor * 1)(_lib.W2VAdamwTensor(64, 64, 64, 0, 0, 4, 0))
    g, k = (C.c_void_p * 1)(64), (C.c_int * 1)(0)
    o = _lib.W2VAdamwOpts(1e-3, 0.9, 0.999, 1e-8, 0.0)
    bad = [dict(bits=16), dict(clock=0), dict(clock=4), dict(k=(C.c_int * 1)(2)), dict(bits=8), dict(n=-1),
           dict(g=(C.c_void_p * 1)(0)), dict(o=_lib.W2VAdamwOpts(1e-3, 1.0, 0.999, 1e-8, 0.0))]
    for b in bad:
        assert lib.w2v_adamw_step(t, b.get("g", g), b.get("k", k), b.get("n", 1), b.get("bits", 32),
                                  C.byref(b.get("o", o)), None, b.get("clock", 64), None) == 1
    assert lib.w2v_adamw_clock(0, 0.9, 0.999, 0, None) == 1
    assert lib.w2v_adamw_clock(64, 0.9, 0.999, -1, None) == 1
    assert lib.w2v_adamw_moments(t, None, None, 1, None) == 1
    for n, vocab, dim, kind in [(-1, 5, 4, 0), (1 << 30, 5, 4, 0), (3, 0, 4, 0), (3, 5, 0, 0), (3, 5, 4, 3)]:
        assert lib.w2v_embed_grad_workspace(n, vocab, dim, kind) == -1
        assert lib.w2v_embed_rows(64, n, 64, dim, vocab, dim, kind, 64, dim, None) == 1
    assert lib.w2v_embed_rows(64, 3, 64, 3, 5, 4, 0, 64, 4, None) == 1       # rows overlap
    assert lib.w2v_embed_grad(64, 3, 64, 4, 5, 4, 0, 64, 4, 0, 0, None) == 1   # no workspace
    assert lib.w2v_launch_count() == before


def test_softmax_refuses():
    from bidmach_b200 import Softmax
    lib = _lib.load()
    before = lib.w2v_launch_count()
    for n, vocab, dim, labels, kind in [(-1, 5, 4, 1, 0), (3, 0, 4, 1, 0), (3, 5, 0, 1, 0), (3, 5, 4097, 1, 0),
                                        (3, 5, 4, 0, 0), (3, 5, 4, 1025, 0), (3, 5, 4, 1, 3), (3, 1 << 31, 4, 1, 0),
                                        (1 << 31, 5, 4, 1, 0)]:
        assert lib.w2v_softmax_workspace(n, vocab, dim, labels, kind, 1) == -1
        assert lib.w2v_softmax_loss(64, dim, 64, dim, 64, n, vocab, dim, labels, kind, 64, 64, 256, 1 << 40, None) == 1
    ok = (64, 4, 64, 4, 64, 20, 50, 4, 1, 0)
    for ws, size in [(0, 1 << 40), (64, 1 << 40), (256, 0)]:     # none, not aligned, too small
        assert lib.w2v_softmax_loss(*ok, 64, 64, ws, size, None) == 1
        assert lib.w2v_softmax_grad(*ok, 64, 64, 1, 64, 4, 64, 4, ws, size, None) == 1
    assert lib.w2v_softmax_grad(*ok, 64, 64, 2, 64, 4, 64, 4, 256, 1 << 40, None) == 1     # stride of gloss
    assert lib.w2v_softmax_grad(*ok, 64, 64, 1, 64, 3, 64, 4, 256, 1 << 40, None) == 1     # rows overlap
    assert lib.w2v_softmax_loss(64, 4, 64, 3, *ok[4:], 64, 64, 256, 1 << 40, None) == 1
    assert lib.w2v_launch_count() == before
    with pytest.raises(ValueError, match="CUDA"):
        Softmax.loss(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        Softmax.loss(torch.zeros(3, 4, dtype=torch.float64), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int32))


def test_window_rows_refuses():
    lib = _lib.load()
    assert lib.w2v_window_rows_workspace(-1) == -1
    size = lib.w2v_window_rows_workspace(10)
    for n, nskip, rows, ws, have in [(-1, 5, 64, 64, 1 << 20), (10, 0, 64, 64, size), (10, 513, 64, 64, size),
                                     (10, 5, 0, 64, size), (10, 5, 64, 0, size), (10, 5, 64, 64, size - 1)]:
        assert lib.w2v_window_rows(64, 64, 64, n, nskip, 64, 64, rows, ws, have, None) == 1


def test_outputs_that_share_memory():
    from bidmach_b200.embed import check_apart
    buf = torch.zeros(12, 10)
    a = buf[:, :4]
    for b in (a, buf, buf[:, 3:6], buf[:6, 2:], buf.view(-1)[3:5], buf[5:6, 1:3], buf[3, 2], buf.view(24, 5)[:, :2],
              buf.view(torch.int32)[:, :1]):
        with pytest.raises(ValueError, match="out overlaps x"):
            check_apart("out", a, x=b)
        with pytest.raises(ValueError, match="out overlaps x"):
            check_apart("out", b, x=a)
    # other columns, other rows, nothing, other memory; rows that start in the columns and end in the next row
    for b in (buf[:, 4:8], buf[:, 4:], buf[:0], torch.zeros(5), torch.tensor(1.0)):
        check_apart("out", a, x=b)
        check_apart("out", b, x=a)
    check_apart("out", buf[:6], x=buf[6:])
    wrap = buf.view(-1)[8:108].view(10, 10)[:, :3]      # columns 8, 9 and 0 of the next row
    with pytest.raises(ValueError):
        check_apart("out", a, x=wrap)
    check_apart("out", buf[:, 2:4], x=wrap)


def test_adamw_moments_that_share_memory():
    x = torch.zeros(1024)
    with pytest.raises(ValueError, match="state overlaps"):
        AdamW._apart([x[:8], x[8:16], x[15:20]], "a tensor of the state overlaps")
    AdamW._apart([x[:8], x[8:16], x[8:8]], "")


def test_rounding_is_checked():
    with pytest.raises(ValueError, match="rounding"):
        AdamW([torch.zeros(8)], AdamW.Opts(bits=8, rounding="up"))
    lib, before = _lib.load(), _lib.load().w2v_launch_count()
    t = (_lib.W2VAdamwTensor * 1)(_lib.W2VAdamwTensor(64, 64, 64, 0, 0, 4, 0))     # no scales
    g, k = (C.c_void_p * 1)(64), (C.c_int * 1)(0)
    o = _lib.W2VAdamwOpts(1e-3, 0.9, 0.999, 1e-8, 0.0)
    assert lib.w2v_adamw_step_random(t, g, k, 1, C.byref(o), None, 1, 64, None) == 1
    assert lib.w2v_adamw_step_random(t, g, k, 1, C.byref(o), None, 1, 0, None) == 1
    assert lib.w2v_launch_count() == before


def test_softmax_says_when_a_kernel_gave_up(monkeypatch):
    """The flag that such a kernel raises, raised here on the host."""
    from bidmach_b200 import Softmax, softmax

    class Fake:
        flag = (C.c_int * 1)(0)

        def w2v_softmax_fault(self):
            return self.flag

    fake = Fake()
    monkeypatch.setattr(softmax._lib, "load", lambda: fake)
    Softmax.check()
    fake.flag[0] = 1
    with pytest.raises(RuntimeError, match="gave up"):
        Softmax.check()
    Softmax.check()      # said once
    fake.w2v_softmax_fault = lambda: None      # no pinned memory
    Softmax.check()


def test_window_rows_wants_equal_int32_vectors_of_the_device():
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    m = Word2Vec(Opts(vocabSize=50, dim=4))
    w = torch.zeros(10, dtype=torch.int32)
    for bad, match in ((w.long(), "int32"), (w.view(2, 5), "dimension"), (w, "CUDA"), ([0] * 10, "int32")):
        with pytest.raises(ValueError, match=match):
            m.windowRows(bad, w, w)


def test_fullsoftmax_options_are_checked_when_the_model_is_made():
    from bidmach_b200 import Word2Vec
    from bidmach_b200.word2vec import Opts
    for bad in (dict(dim=4097), dict(nskip=513), dict(nskip=0), dict(momentBits=16), dict(beta1=1.0), dict(beta2=-0.1),
                dict(adamEps=0.0), dict(wdecay=-1.0), dict(nSlices=2)):
        with pytest.raises(ValueError):
            Word2Vec(Opts(fullSoftmax=True, **bad))
    o = Opts(fullSoftmax=True)
    m = Word2Vec(o)
    o.momentBits = 4
    with pytest.raises(ValueError, match="momentBits"):
        m.init(16)


@pytest.mark.parametrize("n,vocab,dim", [(5, 300, 40), (300, 1000, 64), (9000, 50000, 301)])
@pytest.mark.parametrize("grad", [0, 1])
def test_softmax_workspace_without_copies(n, vocab, dim, grad):
    """A 16-bit matrix that is read where it lies takes no room; fp32 ones are always split."""
    size = _lib.load().w2v_softmax_workspace
    width = (dim + 63) // 64 * 64
    for kind in (1, 2):
        full = size(n, vocab, dim, 1, kind, grad)
        for flag, rows in ((2, n), (4, vocab)):
            copy = (rows * width * 2 + 1023) // 1024 * 1024
            assert full - size(n, vocab, dim, 1, kind, grad | flag) == copy - 1024
    assert size(n, vocab, dim, 1, 0, grad | 6) == size(n, vocab, dim, 1, 0, grad)
