"""Softmax cross entropy over a whole vocabulary, with its gradients, without keeping the logits."""
from __future__ import annotations

import torch

from . import _lib
from .adamw import TYPES, check, on_device, stream_of
from .embed import check_apart, check_ids, check_matrix

CUDA_ERROR_LAUNCH_TIMEOUT = 702
GRAD, HIDDEN_IN_PLACE, WEIGHT_IN_PLACE = 1, 2, 4      # flags of w2v_softmax_workspace


def _vector(x, name: str, n: int, device):
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32 or x.dim() != 1 or x.shape[0] != n \
            or x.get_device() != device.index or not x.is_contiguous():
        raise ValueError(f"{name}: contiguous fp32 [{n}] on {device}")


class Softmax:
    """Static methods only.  With the logits ``l = hidden @ weight.T``:

        lse[i]  = log sum_v exp l[i, v]
        loss[i] = sum over the targets y of row i of (lse[i] - l[i, y])

    ``hidden`` is ``[n, dim]``, ``weight`` ``[vocab, dim]``, both fp32, bf16 or fp16, ``dim`` up to 4096;
    ``targets`` int32 ``[n]`` or ``[n, labels]``.  A target outside ``[0, vocab)`` (-1 by convention) stands
    for none; a row may have none (its loss and gradient are zero) or the same word more than once.
    fp32 operands are multiplied to 22 bits, counted from the largest number of each one's row, and accumulated
    in fp32; 16-bit ones are multiplied exactly.  (Rows or factors of very different sizes, beyond 2^14 or 2^12
    between the largest and the smallest that is not zero, take twice the time; what is below 2^-60
    of the largest may be lost.)
    Every row takes part in the products: an infinity or a NaN in a row of ``hidden``, with targets or without,
    or in ``gloss`` spoils that row's results and ``dweight``, one in ``weight`` all rows'.
    Outputs that are given share no memory with the inputs or with each other."""

    @staticmethod
    def _operands(hidden, weight, targets):
        ldh = check_matrix(hidden, "hidden")
        ldw = check_matrix(weight, "weight", hidden.device, hidden.dtype)
        if not isinstance(targets, torch.Tensor) or targets.dim() not in (1, 2):
            raise ValueError("targets is int32 [n] or [n, labels]")
        check_ids(targets, "targets", targets.dim())
        n, dim = hidden.shape
        labels = 1 if targets.dim() == 1 else targets.shape[1]
        if targets.shape[0] != n or targets.get_device() != hidden.get_device():
            raise ValueError(f"targets has {targets.shape[0]} rows on {targets.device}, hidden {n} on {hidden.device}")
        if weight.shape[1] != dim:
            raise ValueError(f"weight has {weight.shape[1]} columns, hidden {dim}")
        if dim > 4096 or not 1 <= labels <= 1024 or weight.shape[0] < 1:
            raise ValueError("need dim <= 4096, 1 <= labels <= 1024 and at least one word")
        return ldh, ldw, n, weight.shape[0], dim, labels

    @staticmethod
    def _workspace(hidden, ldh, weight, ldw, labels, grad):
        flags = GRAD if grad else 0
        if hidden.element_size() == 2:     # matrices that are read where they lie need no room for a copy
            flags |= HIDDEN_IN_PLACE if hidden.data_ptr() % 16 == 0 and ldh % 8 == 0 else 0
            flags |= WEIGHT_IN_PLACE if weight.data_ptr() % 16 == 0 and ldw % 8 == 0 else 0
        (n, dim), vocab = hidden.shape, weight.shape[0]
        size = _lib.load().w2v_softmax_workspace(n, vocab, dim, labels, TYPES[hidden.dtype], flags)
        if size < 0:
            raise ValueError("w2v_softmax_workspace refused the sizes")
        return torch.empty(size, dtype=torch.uint8, device=hidden.device), size

    @staticmethod
    def check():
        """Raises where a kernel of an earlier call gave up waiting for its copies or products (its results
        hold NaN then).  ``loss`` and ``grad`` do the same for the calls before them; this is for the last ones,
        and for replayed graphs, when their stream has been waited for."""
        flag = _lib.load().w2v_softmax_fault()
        if flag and flag[0]:
            flag[0] = 0
            check(CUDA_ERROR_LAUNCH_TIMEOUT, "Softmax: a kernel gave up waiting:")

    @staticmethod
    def loss(hidden, weight, targets, loss=None, lse=None):
        """Returns ``(loss, lse)``, fp32 ``[n]`` each, new or in the given tensors."""
        ldh, ldw, n, vocab, dim, labels = Softmax._operands(hidden, weight, targets)
        dev, kind = hidden.device, TYPES[hidden.dtype]
        if loss is None:
            loss = torch.empty(n, dtype=torch.float32, device=dev)
        else:
            _vector(loss, "loss", n, dev)
            check_apart("loss", loss, hidden=hidden, weight=weight, targets=targets)
        if lse is None:
            lse = torch.empty(n, dtype=torch.float32, device=dev)
        else:
            _vector(lse, "lse", n, dev)
            check_apart("lse", lse, hidden=hidden, weight=weight, targets=targets, loss=loss)
        with on_device(dev):
            work, size = Softmax._workspace(hidden, ldh, weight, ldw, labels, False)
            check(_lib.load().w2v_softmax_loss(hidden.data_ptr(), ldh, weight.data_ptr(), ldw, targets.data_ptr(), n,
                                               vocab, dim, labels, kind, loss.data_ptr(), lse.data_ptr(),
                                               work.data_ptr(), size, stream_of(dev)), "w2v_softmax_loss")
        return loss, lse

    @staticmethod
    def grad(hidden, weight, targets, lse, gloss, dhidden=None, dweight=None):
        """Gradients of ``sum_i gloss[i] loss[i]`` for ``hidden`` and ``weight``, of their type:
        ``(dhidden, dweight)``, new or in the given tensors.  ``lse`` is what ``loss`` returned; ``gloss``
        fp32 ``[n]``, or one element for all rows.

        With 16-bit operands the gradient by the logits is rounded to their type before it meets them (up to four
        rows excepted), which adds about a tenth to the error that rounding the results has.  In fp16, one factor
        a row, its steps are 2^-38 of the largest ``gloss`` times targets of the call: a row whose factor is below
        1e-6 of that keeps little of its probabilities in ``dhidden``.  bf16 and fp32 keep them for any factors."""
        ldh, ldw, n, vocab, dim, labels = Softmax._operands(hidden, weight, targets)
        dev, kind = hidden.device, TYPES[hidden.dtype]
        _vector(lse, "lse", n, dev)
        if not isinstance(gloss, torch.Tensor) or gloss.dtype is not torch.float32 \
                or gloss.get_device() != dev.index:
            raise ValueError(f"gloss is an fp32 tensor on {dev}")
        one = gloss.numel() == 1
        if not one:
            _vector(gloss, "gloss", n, dev)
        lddh = lddw = dim
        given = dhidden is not None, dweight is not None
        if dhidden is None:
            dhidden = torch.empty(n, dim, dtype=hidden.dtype, device=dev)
        else:
            lddh = check_matrix(dhidden, "dhidden", dev, hidden.dtype)
        if dweight is None:
            dweight = torch.empty(vocab, dim, dtype=hidden.dtype, device=dev)
        else:
            lddw = check_matrix(dweight, "dweight", dev, hidden.dtype)
        if tuple(dhidden.shape) != (n, dim) or tuple(dweight.shape) != (vocab, dim):
            raise ValueError(f"dhidden is {(n, dim)} and dweight {(vocab, dim)}")
        inputs = dict(hidden=hidden, weight=weight, targets=targets, lse=lse, gloss=gloss)
        if given[0]:
            check_apart("dhidden", dhidden, **inputs, dweight=dweight)
        if given[1]:
            check_apart("dweight", dweight, **inputs, dhidden=dhidden)
        with on_device(dev):
            work, size = Softmax._workspace(hidden, ldh, weight, ldw, labels, True)
            check(_lib.load().w2v_softmax_grad(hidden.data_ptr(), ldh, weight.data_ptr(), ldw, targets.data_ptr(), n,
                                               vocab, dim, labels, kind, lse.data_ptr(), gloss.data_ptr(),
                                               0 if one else 1, dhidden.data_ptr(), lddh, dweight.data_ptr(), lddw,
                                               work.data_ptr(), size, stream_of(dev)), "w2v_softmax_grad")
        return dhidden, dweight
