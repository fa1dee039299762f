"""Operators around the graph layers, over libpspmm's C ABI: embedding lookup and its gradient, the
root-mean-square norm of a residual stream, and activations held in 8 bits.

They are tensor-level calls like those of ``ops`` (no autograd; ``gnn_conv`` has the layers that train
with them).  Element types: float32, bfloat16 and float16, sums in 32 bits or more.  2-D operands may be
row-strided views; every operand of a call lives on one GPU, which need not be the current one, and the
work goes to that GPU's current stream.  There is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import check, lib
from .ops import _ptr, _scratch, _stream

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PSPMM_F32 / _BF16 / _F16
EIGHT_BLOCK = 128  # columns that share a scale in the 8-bit form
MAX_DIM = 1 << 24


def _check_tensors(**tensors):
    """What is wrong with operands that are not tensors of one GPU (None among them: left out)."""
    gpu = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise RuntimeError("%s must be a tensor" % name)
        if not t.is_cuda:
            raise RuntimeError("%s must be a CUDA tensor" % name)
        if gpu is None:
            gpu = t.get_device()
        elif t.get_device() != gpu:
            raise RuntimeError("%s is on another device than the other operands" % name)


def _gpu(t):
    """The GPU of a tensor; -1 for anything else."""
    return t.get_device() if isinstance(t, torch.Tensor) and t.is_cuda else -1


def _elsewhere(gpu):
    return gpu != torch._C._cuda_getDevice()


def _rows(t, name, dtype=None, shape=None):
    """(rows, columns, leading dimension) of a matrix with unit column stride, or of a contiguous array with more or fewer
    dimensions taken as rows of its last one."""
    if t.dtype not in _DTYPES or (dtype is not None and t.dtype is not dtype):
        raise RuntimeError("%s must have dtype %s, got %s" % (name, dtype or "float32, bfloat16 or float16", t.dtype))
    size = t.shape
    if shape is not None and size != shape:
        raise RuntimeError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(size)))
    dim = size[-1] if size else 0
    if not 0 < dim <= MAX_DIM:
        raise RuntimeError("%s must have between 1 and %d columns" % (name, MAX_DIM))
    if t.is_contiguous():
        return t.numel() // dim, dim, dim
    if t.dim() == 2 and (t.stride(1) == 1 or dim == 1) and t.stride(0) >= dim:
        return size[0], dim, t.stride(0)
    raise RuntimeError("%s must be contiguous, or a matrix whose rows are" % name)


def _empty_like(t):
    """A contiguous array of a tensor's type and shape (a call without sizes takes half the time)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _vector(t, name, dim, dtype):
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != dim or not t.is_contiguous():
        raise RuntimeError("%s must be a contiguous %s vector of %d" % (name, dtype, dim))


# ----------------------------------------------------------------------------- embedding
def _ids(ids):
    if ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("ids must be int32 or int64, got %s" % ids.dtype)
    if not ids.is_contiguous():
        raise RuntimeError("ids must be contiguous")
    return 1 if ids.dtype is torch.int64 else 0


def embedding(ids, table, scale=1.0):
    """``scale * table[ids]``: one row of ``table`` ([rows, dim]) per id, of the table's type, shaped ``ids.shape + (dim,)``.

    An id outside the table gives a row of NaN and sets :func:`embedding_status` (the GPU is not waited for)."""
    gpu = _gpu(table)
    if gpu < 0 or _gpu(ids) != gpu:
        _check_tensors(ids=ids, table=table)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return embedding(ids, table, scale)
    wide = _ids(ids)
    if table.dim() != 2:
        raise RuntimeError("table must be 2-dimensional")
    rows, dim, ld = _rows(table, "table")
    out = table.new_empty((*ids.shape, dim))
    rc = lib().pspmm_embedding(ids.data_ptr(), wide, ids.numel(), table.data_ptr(), _DTYPES[table.dtype], rows, dim, ld, scale,
                               out.data_ptr(), dim, _stream())
    if rc:
        check(rc)
    return out


def embedding_grad(ids, grad, n_rows, scale=1.0, padding_idx=None):
    """Gradient of :func:`embedding` with respect to its table of ``n_rows`` rows: row t is ``scale`` times the sum of the rows of
    ``grad`` whose id is t, of the type of ``grad``; ids equal to ``padding_idx`` and ids outside the table add nothing.

    The sums run in the order of the ids' positions (they are sorted first): equal calls give equal bits."""
    gpu = _gpu(grad)
    if gpu < 0 or _gpu(ids) != gpu:
        _check_tensors(ids=ids, grad=grad)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return embedding_grad(ids, grad, n_rows, scale, padding_idx)
    wide = _ids(ids)
    n, dim, ld = _rows(grad, "grad")
    if n != ids.numel():
        raise RuntimeError("grad must have one row per id")
    if n_rows < 0:
        raise RuntimeError("n_rows must not be negative")
    if padding_idx is not None and not 0 <= padding_idx < n_rows:
        raise RuntimeError("padding_idx must be a row of the table")
    out = grad.new_empty((n_rows, dim))
    scratch, need = _scratch("pspmm_embedding_grad_scratch_bytes", (n, dim), grad.device)
    rc = lib().pspmm_embedding_grad(ids.data_ptr(), wide, n, grad.data_ptr(), _DTYPES[grad.dtype], ld, n_rows, dim, scale,
                                    -1 if padding_idx is None else padding_idx, out.data_ptr(), dim, _ptr(scratch), need, _stream())
    if rc:
        check(rc)
    return out


def embedding_status():
    """1 once an id outside its table has been met in this process on the current GPU, else 0 (synchronises with the device)."""
    v = ctypes.c_int32(0)
    check(lib().pspmm_embedding_status(ctypes.byref(v)))
    return int(v.value)


# ----------------------------------------------------------------------------- rows in 8 bits
class Rows8:
    """Rows held in 8 bits: per row and block of 128 columns with largest magnitude a, ``scale = a / 127`` and whole numbers
    ``q = rint(x * (127 / a))``; ``q * scale`` stands for ``x`` and is off by at most 0.51 scale.  Blocks below 2^-119 are
    zeros, blocks with an infinity or a NaN come back as NaN.

    ``q``: int8 [n, pitch], rows padded to a multiple of 16 bytes; ``scales``: float32 [n, ceil(dim / 128)]; ``shape`` is that of
    the array held."""

    __slots__ = ("q", "scales", "dim", "shape")

    def __init__(self, q, scales, dim, shape=None):
        n = q.shape[0] if q.dim() == 2 else -1
        if (q.dtype is not torch.int8 or n < 0 or not q.is_contiguous() or q.shape[1] < dim or q.shape[1] % 16 or dim < 1
                or q.data_ptr() % 16):
            raise RuntimeError("q must be a contiguous, 16-byte aligned int8 matrix of rows padded to a multiple of 16, at least %d"
                               % dim)
        if (scales.dtype is not torch.float32 or not scales.is_contiguous()
                or scales.shape != (n, (dim + EIGHT_BLOCK - 1) // EIGHT_BLOCK)):
            raise RuntimeError("scales must be a contiguous float32 matrix of a scale per row and block of %d columns" % EIGHT_BLOCK)
        if q.get_device() != scales.get_device():
            raise RuntimeError("scales is on another device than q")
        self.q, self.scales, self.dim = q, scales, dim
        self.shape = torch.Size((n, dim)) if shape is None else torch.Size(shape)
        if self.shape[-1] != dim or self.shape.numel() != n * dim:
            raise RuntimeError("shape must be that of %d rows of %d" % (n, dim))

    def dequantize(self, dtype=torch.float32):
        """The values that the whole numbers stand for."""
        gpu = _gpu(self.q)
        if gpu < 0:
            _check_tensors(q=self.q)
        if _elsewhere(gpu):
            with torch.cuda.device(gpu):
                return self.dequantize(dtype)
        if dtype not in _DTYPES:
            raise RuntimeError("dtype must be float32, bfloat16 or float16, got %s" % dtype)
        out = self.q.new_empty(self.shape, dtype=dtype)
        rc = lib().pspmm_dequantize_rows(self.q.data_ptr(), self.q.shape[1], self.scales.data_ptr(), _DTYPES[dtype], out.data_ptr(),
                                         self.dim, self.q.shape[0], self.dim, _stream())
        if rc:
            check(rc)
        return out

    def weight_grad(self, G):
        """:func:`rows8_mm_t` of these rows and ``G``."""
        return rows8_mm_t(self, G)


def _empty_rows8(x, n, dim):
    """Rows8 of an array like ``x``, yet to be written."""
    kept = Rows8.__new__(Rows8)
    kept.q = x.new_empty((n, dim + -dim % 16), dtype=torch.int8)
    kept.scales = x.new_empty((n, (dim + EIGHT_BLOCK - 1) // EIGHT_BLOCK), dtype=torch.float32)
    kept.dim, kept.shape = dim, x.shape
    return kept


def quantize_rows(x):
    """``x`` in 8 bits (:class:`Rows8`), a scale per row and 128 columns."""
    gpu = _gpu(x)
    if gpu < 0:
        _check_tensors(x=x)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return quantize_rows(x)
    n, dim, ld = _rows(x, "x")
    kept = _empty_rows8(x, n, dim)
    rc = lib().pspmm_quantize_rows(x.data_ptr(), _DTYPES[x.dtype], ld, n, dim, kept.q.data_ptr(), dim + -dim % 16,
                                   kept.scales.data_ptr(), _stream())
    if rc:
        check(rc)
    return kept


def rows8_mm_t(rows, G, out=None):
    """``X^T @ G`` in float32, [dim, cols], from the 8-bit form of X ([n, dim], a :class:`Rows8`) and ``G`` ([n, cols]): the weight
    gradient of a layer that kept its input in 8 bits, on the tensor cores with float32 accuracy."""
    if not isinstance(rows, Rows8):
        raise RuntimeError("rows must be a Rows8")
    gpu = _gpu(G)
    if gpu < 0 or _gpu(rows.q) != gpu or (out is not None and _gpu(out) != gpu):
        _check_tensors(q=rows.q, G=G, out=out)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return rows8_mm_t(rows, G, out)
    n, cols, ld = _rows(G, "G")
    if n != rows.q.shape[0]:
        raise RuntimeError("G must have one row per row held, %d, got %d" % (rows.q.shape[0], n))
    if out is None:
        out = G.new_empty((rows.dim, cols), dtype=torch.float32)
    elif (out.dtype is not torch.float32 or out.shape != (rows.dim, cols) or out.stride(1) != 1 or out.stride(0) < cols):
        raise RuntimeError("out must be a float32 matrix of %d rows of %d with unit column stride" % (rows.dim, cols))
    aligned = 1 if (ld * G.element_size()) % 16 == 0 and G.data_ptr() % 16 == 0 else 0
    try:
        scratch, need = _scratch("pspmm_rows8_mm_t_scratch_bytes", (n, rows.dim, cols, _DTYPES[G.dtype], aligned), G.device)
    except torch.cuda.OutOfMemoryError:
        if aligned:
            raise
        # without the copy of G on aligned rows
        scratch, need = _scratch("pspmm_rows8_mm_t_scratch_bytes", (n, rows.dim, cols, _DTYPES[G.dtype], 1), G.device)
    rc = lib().pspmm_rows8_mm_t(rows.q.data_ptr(), rows.q.shape[1], rows.scales.data_ptr(), n, rows.dim, G.data_ptr(),
                                _DTYPES[G.dtype], ld, cols, out.data_ptr(), out.stride(0), _ptr(scratch), need, _stream())
    if rc:
        check(rc)
    return out


def rows8_mm_status():
    """1 once a bounded wait of :func:`rows8_mm_t` has run out in this process on the current GPU, else 0 (synchronises with the
    device).  What was not computed of the result is NaN then."""
    v = ctypes.c_int32(0)
    check(lib().pspmm_rows8_mm_status(ctypes.byref(v)))
    return int(v.value)


# ----------------------------------------------------------------------------- norm
def rms_norm(x, weight, residual=None, eps=1e-6, relu=False, values=True, eight_bit=False):
    """Root-mean-square norm of ``h = x + residual`` over the last dimension: ``y = h * rstd * weight`` with
    ``rstd = (mean(h^2) + eps)^-1/2``, negative ``y`` set to 0 with ``relu``.

    Returns ``(y, h, rstd, kept)``: ``h`` is the residual stream (``x`` itself without a ``residual``), ``rstd`` (float32, one per
    row) what :func:`rms_norm_backward` needs, ``kept`` the :class:`Rows8` of ``y`` with ``eight_bit`` (else None), made in the
    same pass.  ``values=False`` leaves ``y`` out (None) for a consumer of the 8 bits alone."""
    gpu = _gpu(x)
    if gpu < 0 or _gpu(weight) != gpu or (residual is not None and _gpu(residual) != gpu):
        _check_tensors(x=x, weight=weight, residual=residual)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return rms_norm(x, weight, residual, eps, relu, values, eight_bit)
    n, dim, ld = _rows(x, "x")
    _vector(weight, "weight", dim, x.dtype)
    if not eps >= 0:
        raise RuntimeError("eps must not be negative")
    if not values and not eight_bit:
        raise RuntimeError("nothing is asked for: neither values nor the 8-bit form")
    h, ld_r, r_ptr, h_ptr = x, 0, None, None
    if residual is not None:
        ld_r = _rows(residual, "residual", x.dtype, x.shape)[2]
        h = _empty_like(x)
        r_ptr, h_ptr = residual.data_ptr(), h.data_ptr()
    y = _empty_like(x) if values else None
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    kept, q_ptr, s_ptr = None, None, None
    if eight_bit:
        kept = _empty_rows8(x, n, dim)
        q_ptr, s_ptr = kept.q.data_ptr(), kept.scales.data_ptr()
    rc = lib().pspmm_rms_norm(x.data_ptr(), ld, r_ptr, ld_r, weight.data_ptr(), _DTYPES[x.dtype], n, dim, eps, 1 if relu else 0,
                              h_ptr, dim, y.data_ptr() if values else None, dim, rstd.data_ptr(), q_ptr, dim + -dim % 16, s_ptr,
                              _stream())
    if rc:
        check(rc)
    return y, h, rstd, kept


def rms_norm_backward(dy, h, rstd, weight, dh=None, relu=False):
    """Gradients ``(dx, dweight)`` of :func:`rms_norm` from ``dy`` and, where the residual stream goes on, the gradient ``dh`` that
    reaches ``h`` itself; ``dx`` is the gradient of ``x`` and of ``residual`` alike."""
    gpu = _gpu(dy)
    if gpu < 0 or _gpu(h) != gpu or _gpu(rstd) != gpu or _gpu(weight) != gpu or (dh is not None and _gpu(dh) != gpu):
        _check_tensors(dy=dy, h=h, rstd=rstd, weight=weight, dh=dh)
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return rms_norm_backward(dy, h, rstd, weight, dh, relu)
    n, dim, ld_h = _rows(h, "h")
    ld_dy = _rows(dy, "dy", h.dtype, h.shape)[2]
    ld_dh = _rows(dh, "dh", h.dtype, h.shape)[2] if dh is not None else 0
    _vector(weight, "weight", dim, h.dtype)
    if rstd.dtype is not torch.float32 or rstd.shape != h.shape[:-1] or not rstd.is_contiguous():
        raise RuntimeError("rstd must be contiguous float32, one per row")
    dx = _empty_like(h)
    dw = _empty_like(weight)
    scratch, need = _scratch("pspmm_rms_norm_backward_scratch_bytes", (n, dim), h.device)
    rc = lib().pspmm_rms_norm_backward(dy.data_ptr(), ld_dy, h.data_ptr(), ld_h, rstd.data_ptr(), weight.data_ptr(), _ptr(dh), ld_dh,
                                       _DTYPES[h.dtype], n, dim, 1 if relu else 0, dx.data_ptr(), dim, dw.data_ptr(), _ptr(scratch),
                                       need, _stream())
    if rc:
        check(rc)
    return dx, dw
