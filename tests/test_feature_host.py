"""What the operators around the layers refuse, without a GPU: raw pointers leave Python here, so operands of a wrong kind have to
stop before, and the C entry points answer with codes."""
import ctypes

import pytest
import torch

NULL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(4096)  # never dereferenced: the checks come first


def _arg(rc):
    from paramspmm_ae_b200 import _lib
    assert rc == _lib.PSPMM_E_ARG


def test_rows8_entry_points_refuse(pspmm_lib):
    from paramspmm_ae_b200 import _lib
    quant = lambda x=ONE, t=0, ld=64, n=4, dim=64, q=ONE, pitch=64, s=ONE: pspmm_lib.pspmm_quantize_rows(
        x, t, ld, n, dim, q, pitch, s, NULL)
    back = lambda x=ONE, t=0, ld=64, n=4, dim=64, q=ONE, pitch=64, s=ONE: pspmm_lib.pspmm_dequantize_rows(
        q, pitch, s, t, x, ld, n, dim, NULL)
    for call in (quant, back):
        for bad in (dict(x=NULL), dict(q=NULL), dict(s=NULL), dict(t=3), dict(t=-1), dict(n=-1), dict(dim=0), dict(ld=63),
                    dict(pitch=48), dict(pitch=72), dict(q=ctypes.c_void_p(4097)), dict(x=ctypes.c_void_p(4098)),
                    dict(t=1, x=ctypes.c_void_p(4097)), dict(s=ctypes.c_void_p(4098))):
            _arg(call(**bad))
        assert call(n=1 << 40) == _lib.PSPMM_E_RANGE
        assert call(n=0, x=NULL, q=NULL, s=NULL) == _lib.PSPMM_OK


def test_rms_norm_entry_points_refuse(pspmm_lib):
    from paramspmm_ae_b200 import _lib

    def forward(x=ONE, ldx=64, r=NULL, ldr=64, w=ONE, t=0, n=4, dim=64, eps=1e-6, h=NULL, ldh=64, y=ONE, ldy=64, rstd=ONE, q=NULL,
                pitch=64, s=NULL):
        return pspmm_lib.pspmm_rms_norm(x, ldx, r, ldr, w, t, n, dim, eps, 0, h, ldh, y, ldy, rstd, q, pitch, s, NULL)

    for bad in (dict(x=NULL), dict(w=NULL), dict(rstd=NULL), dict(t=7), dict(n=-1), dict(dim=0), dict(eps=-1.0),
                dict(eps=float("nan")), dict(ldx=63), dict(r=ONE, ldr=3), dict(h=ONE, ldh=3), dict(ldy=3), dict(q=ONE),
                dict(s=ONE), dict(q=ONE, s=ONE, pitch=65), dict(q=ONE, s=ONE, pitch=48), dict(x=ctypes.c_void_p(4097)),
                dict(rstd=ctypes.c_void_p(4098))):
        _arg(forward(**bad))
    assert forward(n=0, x=NULL, w=NULL, y=NULL, rstd=NULL) == _lib.PSPMM_OK

    need = ctypes.c_size_t(0)
    assert pspmm_lib.pspmm_rms_norm_backward_scratch_bytes(4, 64, ctypes.byref(need)) == 0 and need.value == 4 * 64 * 4
    _arg(pspmm_lib.pspmm_rms_norm_backward_scratch_bytes(4, 0, ctypes.byref(need)))
    _arg(pspmm_lib.pspmm_rms_norm_backward_scratch_bytes(4, 64, None))

    def backward(dy=ONE, ldy=64, h=ONE, ldh=64, rstd=ONE, w=ONE, dh=NULL, lddh=64, t=0, n=4, dim=64, dx=ONE, lddx=64, dw=ONE,
                 scratch=ONE, size=4 * 64 * 4):
        return pspmm_lib.pspmm_rms_norm_backward(dy, ldy, h, ldh, rstd, w, dh, lddh, t, n, dim, 0, dx, lddx, dw, scratch, size, NULL)

    for bad in (dict(dy=NULL), dict(h=NULL), dict(rstd=NULL), dict(w=NULL), dict(dx=NULL), dict(dw=NULL), dict(scratch=NULL),
                dict(size=4 * 64 * 4 - 1), dict(t=3), dict(n=-1), dict(dim=0), dict(ldy=1), dict(ldh=1), dict(dh=ONE, lddh=1),
                dict(lddx=1), dict(dx=ctypes.c_void_p(4098))):
        _arg(backward(**bad))


def test_embedding_entry_points_refuse(pspmm_lib):
    from paramspmm_ae_b200 import _lib

    def look(ids=ONE, n=4, table=ONE, t=0, rows=9, dim=16, ld=16, out=ONE, ldo=16, wide=1):
        return pspmm_lib.pspmm_embedding(ids, wide, n, table, t, rows, dim, ld, 1.0, out, ldo, NULL)

    for bad in (dict(ids=NULL), dict(table=NULL), dict(out=NULL), dict(t=3), dict(n=-1), dict(rows=-1), dict(dim=0), dict(ld=15),
                dict(ldo=15), dict(ids=ctypes.c_void_p(4100)), dict(wide=0, ids=ctypes.c_void_p(4098)),
                dict(out=ctypes.c_void_p(4098))):
        _arg(look(**bad))
    assert look(n=0, ids=NULL, table=NULL, out=NULL) == _lib.PSPMM_OK

    need = ctypes.c_size_t(0)
    assert pspmm_lib.pspmm_embedding_grad_scratch_bytes(100, 16, ctypes.byref(need)) == 0 and need.value > 0
    size = need.value
    assert pspmm_lib.pspmm_embedding_grad_scratch_bytes(0, 16, ctypes.byref(need)) == 0 and need.value == 0
    _arg(pspmm_lib.pspmm_embedding_grad_scratch_bytes(-1, 16, ctypes.byref(need)))

    def grad(ids=ONE, n=100, g=ONE, t=0, ld=16, rows=9, dim=16, out=ONE, ldo=16, scratch=ONE, size=size):
        return pspmm_lib.pspmm_embedding_grad(ids, 1, n, g, t, ld, rows, dim, 1.0, -1, out, ldo, scratch, size, NULL)

    for bad in (dict(ids=NULL), dict(g=NULL), dict(out=NULL), dict(scratch=NULL), dict(size=size - 1), dict(t=3), dict(n=-1),
                dict(rows=-1), dict(dim=0), dict(ld=15), dict(ldo=15), dict(scratch=ctypes.c_void_p(4104))):
        _arg(grad(**bad))
    assert grad(n=2 ** 31) == _lib.PSPMM_E_RANGE
    assert grad(rows=2 ** 32) == _lib.PSPMM_E_RANGE
    assert grad(rows=0, out=NULL, ids=NULL, g=NULL) == _lib.PSPMM_OK


def test_cpu_tensors_and_non_tensors_are_refused():
    from paramspmm_ae_b200 import feature_ops as fo
    x, w, ids = torch.randn(4, 8), torch.ones(8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: fo.quantize_rows(x), lambda: fo.rms_norm(x, w), lambda: fo.embedding(ids, x),
                 lambda: fo.embedding_grad(ids, x, 5), lambda: fo.rms_norm_backward(x, x, torch.ones(4), w)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="must be a tensor"):
        fo.quantize_rows([1.0])


def test_rows_takes_rows_and_refuses_the_rest():
    from paramspmm_ae_b200 import feature_ops as fo
    x = torch.zeros(6, 10)
    assert fo._rows(x, "x") == (6, 10, 10)
    assert fo._rows(x[:, 2:7], "x") == (6, 5, 10)
    assert fo._rows(torch.zeros(2, 3, 4), "x") == (6, 4, 4)
    assert fo._rows(torch.zeros(4), "x") == (1, 4, 4)
    assert fo._rows(torch.zeros(0, 4), "x") == (0, 4, 4)
    for bad in (x.t(), x[:, ::2], torch.zeros(1, 5).expand(6, 5), torch.zeros(2, 3, 4)[:, :, 1:], torch.zeros(6, 0), torch.tensor(1.0),
                torch.zeros(6, 10, dtype=torch.float64), torch.zeros(6, 10, dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            fo._rows(bad, "x")
    with pytest.raises(RuntimeError, match="dtype"):
        fo._rows(x, "x", torch.bfloat16)
    with pytest.raises(RuntimeError, match="shape"):
        fo._rows(x, "x", torch.float32, torch.Size((6, 9)))


def test_rows8_refuses_other_layouts():
    from paramspmm_ae_b200 import feature_ops as fo
    q, s = torch.zeros(5, 208, dtype=torch.int8), torch.zeros(5, 2)
    assert fo.Rows8(q, s, 200).shape == (5, 200)
    assert fo.Rows8(q, s, 200, (1, 5, 200)).shape == (1, 5, 200)
    for bad in ((q[:, :192], s, 190), (q.float(), s, 200), (q[:, :200].contiguous(), s, 200), (q, s, 209), (q, s, 0),
                (q, s[:, :1].contiguous(), 200), (q, s.double(), 200), (q, s.t(), 200), (q[0], s, 200),
                (q.view(-1)[1:], s, 200), (q, s, 200, (5, 2, 200))):
        with pytest.raises(RuntimeError):
            fo.Rows8(*bad)


class _Cuda:
    """A tensor that says it lies on a GPU."""

    is_cuda = True

    def __new__(cls, t, gpu):
        class On(torch.Tensor):
            is_cuda = True

            def get_device(self):
                return gpu

        return t.as_subclass(On)


def test_operands_on_two_gpus_are_refused():
    from paramspmm_ae_b200 import feature_ops as fo
    a, b = _Cuda(torch.zeros(4, 8), 0), _Cuda(torch.zeros(4, 8), 1)
    w, ids = _Cuda(torch.ones(8), 1), _Cuda(torch.zeros(4, dtype=torch.int64), 1)
    for call in (lambda: fo.rms_norm(a, w), lambda: fo.rms_norm(a, _Cuda(torch.ones(8), 0), b), lambda: fo.embedding(ids, a),
                 lambda: fo.embedding_grad(ids, a, 5), lambda: fo.rms_norm_backward(a, b, w, w)):
        with pytest.raises(RuntimeError, match="another device"):
            call()


def test_rows8_product_entry_point_refuses(pspmm_lib):
    from paramspmm_ae_b200 import _lib
    need = ctypes.c_size_t(0)
    assert pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(100000, 64, 16, 0, 1, ctypes.byref(need)) == 0 and need.value > 0
    size = need.value
    assert pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(0, 64, 16, 0, 1, ctypes.byref(need)) == 0 and need.value == 0
    _arg(pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(-1, 64, 16, 0, 1, ctypes.byref(need)))
    _arg(pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(1, 64, 16, 0, 1, None))
    _arg(pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(1, 64, 16, 3, 1, ctypes.byref(need)))
    assert pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(100000, 64, 17, 1, 1, ctypes.byref(need)) == 0
    without = need.value
    assert pspmm_lib.pspmm_rows8_mm_t_scratch_bytes(100000, 64, 17, 1, 0, ctypes.byref(need)) == 0
    assert need.value == without + 100000 * 24 * 2

    def mm(q=ONE, pitch=64, s=ONE, n=100000, dim=64, G=ONE, t=0, ld=16, cols=16, C=ONE, ldc=16, scratch=ONE, size=size):
        return pspmm_lib.pspmm_rows8_mm_t(q, pitch, s, n, dim, G, t, ld, cols, C, ldc, scratch, size, NULL)

    for bad in (dict(q=NULL), dict(s=NULL), dict(G=NULL), dict(C=NULL), dict(scratch=NULL), dict(size=size - 1), dict(pitch=63),
                dict(pitch=72), dict(pitch=48), dict(n=-1), dict(dim=0), dict(t=3), dict(ld=15), dict(ldc=15), dict(cols=-1),
                dict(q=ctypes.c_void_p(4104)), dict(G=ctypes.c_void_p(4098)), dict(scratch=ctypes.c_void_p(4104))):
        _arg(mm(**bad))
    assert mm(n=1 << 50) == _lib.PSPMM_E_RANGE
    assert mm(cols=1 << 21, ld=1 << 21, ldc=1 << 21) == _lib.PSPMM_E_RANGE
    assert mm(cols=0, C=NULL, G=NULL) == _lib.PSPMM_OK
