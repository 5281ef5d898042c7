"""Rows of a matrix picked by word ids, and the gradient of that."""
from __future__ import annotations

import torch

from . import _lib
from .adamw import TYPES, check, on_device, stream_of


def check_matrix(x, name: str, device=None, dtype=None):
    """A CUDA matrix whose rows are contiguous; returns its leading dimension."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.dtype not in TYPES:
        raise ValueError(f"{name} is a matrix of fp32, bf16 or fp16")
    if dtype is not None and x.dtype is not dtype:
        raise ValueError(f"{name} has type {x.dtype}, expected {dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} is not on a CUDA device")
    if device is not None and x.get_device() != device.index:
        raise ValueError(f"{name} is on {x.device}, expected {device}")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError(f"{name} has no columns")
    if rows <= 1 and (cols == 1 or x.stride(1) == 1):
        return cols
    ld, step = x.stride()
    if (step != 1 and cols > 1) or ld < cols:
        raise ValueError(f"{name}: rows have to be contiguous and must not overlap")
    return ld


def check_ids(x, name: str, dim: int):
    if not isinstance(x, torch.Tensor) or x.dim() != dim or x.dtype is not torch.int32:
        raise ValueError(f"{name} is int32 with {dim} dimension" + ("s" if dim > 1 else ""))
    if not x.is_cuda:
        raise ValueError(f"{name} is not on a CUDA device")
    if not x.is_contiguous():
        raise ValueError(f"{name} is not contiguous")


def _meet(a, b) -> bool:
    """Whether an element of `a` shares memory with one of `b`: contiguous tensors, or matrices with
    contiguous rows.  Two sets of columns of one buffer do not; others whose ranges cross count as met."""
    spans = []
    for x in (a, b):
        if x.numel() == 0:
            return False
        matrix = x.dim() == 2 and x.shape[0] > 1
        row = (x.shape[1] if matrix else x.numel()) * x.element_size()
        ld, rows = (x.stride(0) * x.element_size(), x.shape[0]) if matrix else (row, 1)
        spans.append((x.data_ptr(), x.data_ptr() + (rows - 1) * ld + row, ld, row))
    (a0, a1, lda, rowa), (b0, b1, ldb, rowb) = spans
    if a1 <= b0 or b1 <= a0:
        return False
    if lda != ldb:
        return True
    off = (b0 - a0) % lda
    return off < rowa or off + rowb > lda


def check_apart(name: str, out, **others):
    """Refuses an output that shares memory with another tensor of the call."""
    for other, x in others.items():
        if _meet(out, x):
            raise ValueError(f"{name} overlaps {other}")


class EmbedRows:
    """Static methods only.  ``ids``: int32, one for each row; an id outside the matrix (-1 marks a
    dropped word) gives a row of zeros and takes no part in the gradient.
    ``out``, where one is given, shares no memory with the inputs."""

    @staticmethod
    def forward(ids, matrix, out=None):
        """``out[i] = matrix[ids[i]]``."""
        check_ids(ids, "ids", 1)
        ldm = check_matrix(matrix, "matrix", ids.device)
        n, (vocab, dim) = ids.numel(), matrix.shape
        if not 1 <= vocab < 2 ** 31 - 1 or n >= 2 ** 30 or dim > 65536:
            raise ValueError("need 1 to 2^31 - 2 rows of matrix, fewer than 2^30 ids, at most 65536 columns")
        if out is None:
            out, ldo = torch.empty(n, dim, dtype=matrix.dtype, device=ids.device), dim
        else:
            ldo = check_matrix(out, "out", ids.device, matrix.dtype)
            if tuple(out.shape) != (n, dim):
                raise ValueError(f"out has shape {tuple(out.shape)}, expected {(n, dim)}")
            check_apart("out", out, ids=ids, matrix=matrix)
        with on_device(ids.device):
            check(_lib.load().w2v_embed_rows(ids.data_ptr(), n, matrix.data_ptr(), ldm, vocab, dim,
                                             TYPES[matrix.dtype], out.data_ptr(), ldo, stream_of(ids.device)),
                  "w2v_embed_rows")
        return out

    @staticmethod
    def backward(ids, grad, nrows: int, out=None):
        """Gradient of the matrix, ``[nrows, dim]``: row ``v`` is the sum of the rows of ``grad`` whose
        id is ``v``, added in fp32 and in an order that the ids fix (equal calls give equal bits), zero
        where there is none."""
        check_ids(ids, "ids", 1)
        ldg = check_matrix(grad, "grad", ids.device)
        n, dim, nrows = ids.numel(), grad.shape[1], int(nrows)
        if grad.shape[0] != n:
            raise ValueError(f"grad has {grad.shape[0]} rows for {n} ids")
        if not 1 <= nrows < 2 ** 31 - 1 or n >= 2 ** 30 or dim > 65536:
            raise ValueError("need 1 <= nrows < 2^31 - 1, fewer than 2^30 ids, at most 65536 columns")
        if out is None:
            out, ldo = torch.empty(nrows, dim, dtype=grad.dtype, device=ids.device), dim
        else:
            ldo = check_matrix(out, "out", ids.device, grad.dtype)
            if tuple(out.shape) != (nrows, dim):
                raise ValueError(f"out has shape {tuple(out.shape)}, expected {(nrows, dim)}")
            check_apart("out", out, ids=ids, grad=grad)
        lib, t = _lib.load(), TYPES[grad.dtype]
        with on_device(ids.device):
            size = lib.w2v_embed_grad_workspace(n, nrows, dim, t)
            if size < 0:
                raise RuntimeError("w2v_embed_grad_workspace refused the sizes")
            work = torch.empty(size, dtype=torch.uint8, device=ids.device)
            check(lib.w2v_embed_grad(ids.data_ptr(), n, grad.data_ptr(), ldg, nrows, dim, t, out.data_ptr(), ldo,
                                     work.data_ptr(), size, stream_of(ids.device)), "w2v_embed_grad")
        return out
