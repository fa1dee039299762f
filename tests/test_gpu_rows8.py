"""Rows held in 8 bits, against the definition in 64 bits.  Whole numbers and scales have to be equal: a / 127 and 127 / a are
single 32-bit divisions, and x * (127 / a) is exact in 64 bits before it is rounded."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
BLOCK, TINY = 128, 2.0 ** -119


def eight(y):
    """(whole numbers [n, dim], scales) of a CPU matrix, from 32-bit largest magnitudes."""
    n, dim = y.shape
    q, scales = torch.zeros(n, dim, dtype=torch.float64), torch.zeros(n, (dim + BLOCK - 1) // BLOCK)
    for b in range(scales.shape[1]):
        v = y[:, b * BLOCK:(b + 1) * BLOCK].double()
        a = v.abs().amax(1).float()
        held, top = a >= TINY, torch.full_like(a, 127)  # (`127 / a` would be the rounded 1 / a, times 127)
        scales[:, b] = torch.where(held, a / top, 0.0)
        up = torch.where(held, top / a, 0.0).double()
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.round(v * up[:, None])
    return q, scales


def check(kept, y):
    n, dim = y.shape
    q, scales = eight(y)
    assert torch.equal(kept.scales.cpu(), scales)
    got = kept.q.cpu()
    assert torch.equal(got[:, :dim].double(), q)
    assert not got[:, dim:].any()
    return q, scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 16, 31, 47, 100, 127, 128, 129, 136, 250, 252, 256, 500, 1000, 1025, 4096])
def test_whole_numbers_and_scales(dtype, dim):
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator().manual_seed(dim)
    x = (torch.randn(37, dim, generator=g) * torch.exp(3 * torch.randn(37, 1, generator=g))).to(dtype)
    x[3] = 0
    x[5, : dim // 2] = 0
    kept = fo.quantize_rows(x.cuda())
    q, scales = check(kept, x.float())
    for out in TYPES:
        want = (q.float() * scales.repeat_interleave(BLOCK, 1)[:, :dim]).to(out)
        assert torch.equal(kept.dequantize(out).cpu(), want)
    # half a step of the block's scale, and the roundings of 127 / a and a / 127
    off = (kept.dequantize().cpu().double() - x.double()).abs()
    assert (off <= scales.double().repeat_interleave(BLOCK, 1)[:, :dim] * (0.5 + 2 ** -15)).all()


@pytest.mark.parametrize("n", [0, 1, 2, 31, 1000, 20011])
def test_row_counts_shapes_and_views(n):
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, 72, generator=g)
    check(fo.quantize_rows(x.cuda()), x)
    wide = torch.randn(n, 200, generator=g)
    for a, b in ((3, 103), (4, 104), (64, 200)):  # misaligned and aligned column slices
        check(fo.quantize_rows(wide.cuda()[:, a:b]), wide[:, a:b])
    three = torch.randn(n, 3, 24, generator=g)
    kept = fo.quantize_rows(three.cuda())
    check(kept, three.reshape(-1, 24))
    assert kept.dequantize().shape == three.shape


def test_values_at_the_ends():
    from paramspmm_ae_b200 import feature_ops as fo
    x = torch.zeros(9, 256)
    x[0, 0], x[0, 200] = 3.4e38, -3.4e38
    x[1, :] = 2.0 ** -126
    x[2, :] = torch.full((), 2.0 ** -119)
    x[3, :] = 1.4e-45
    x[4, 3], x[4, 4] = float("inf"), 1.0
    x[5, 3], x[5, 4] = float("nan"), 1.0
    x[6, 130], x[6, 4] = float("-inf"), 1.0
    x[7, :] = -0.0
    x[8, :128] = torch.arange(128) - 64.0  # 127 / a = 1.98: halves round to even
    kept = fo.quantize_rows(x.cuda())
    got = kept.dequantize().cpu()
    q, scales = eight(x)
    for r in (0, 1, 2, 3, 7, 8):
        assert torch.equal(kept.q[r].cpu().double(), q[r]) and torch.equal(kept.scales[r].cpu(), scales[r])
        assert torch.isfinite(got[r]).all()
    assert not got[1].any() and not got[3].any() and (got[2] == 2.0 ** -119).all()
    for r, b in ((4, 0), (5, 0), (6, 1)):  # the block that holds it, and no other
        other = slice(128, 256) if b == 0 else slice(0, 128)
        assert torch.isnan(got[r, b * 128:(b + 1) * 128]).all() and torch.isfinite(got[r, other]).all()
    assert got[6, 4] == 1.0


def test_captured_and_replayed_on_another_stream():
    from paramspmm_ae_b200 import feature_ops as fo
    x = torch.randn(300, 130, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fo.quantize_rows(x).dequantize()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = fo.quantize_rows(x)
        out = kept.dequantize()
    for seed in (1, 2):
        x.copy_(torch.randn(300, 130, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        check(kept, x.cpu())
        assert torch.equal(out, fo.quantize_rows(x).dequantize())


def test_more_than_two_to_the_31_values():
    from paramspmm_ae_b200 import feature_ops as fo
    n, dim = 530000, 4096  # 2.17 G values, 4.3 GB of bf16
    x = torch.empty(n, dim, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, 262143, 524287, 524288, 524289, n - 1])
    x[rows.cuda()] = torch.randn(len(rows), dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    kept = fo.quantize_rows(x)
    part = fo.Rows8(kept.q[rows.cuda()].contiguous(), kept.scales[rows.cuda()].contiguous(), dim)
    check(part, x[rows.cuda()].float().cpu())
    out = kept.dequantize(torch.bfloat16)
    assert torch.equal(out[rows.cuda()], part.dequantize(torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [5, 40, 47, 144, 300, 1030, 9000])
def test_a_longer_pitch_is_left_alone(pspmm_lib, dtype, dim):
    """Through the C ABI: columns up to the next multiple of 16 become zeros, those behind them keep what they held."""
    n, used = 9, dim + -dim % 16
    pitch, t = used + 160, TYPES.index(dtype)
    x = torch.randn(n, dim, generator=torch.Generator().manual_seed(dim)).to(dtype).cuda()
    w = torch.ones(dim, dtype=dtype, device="cuda")
    scales = torch.empty(n, (dim + BLOCK - 1) // BLOCK, device="cuda")
    rstd = torch.empty(n, device="cuda")
    ptr = lambda a: ctypes.c_void_p(a.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for norm in (False, True):
        q = torch.full((n, pitch), 77, dtype=torch.int8, device="cuda")
        if norm:
            rc = pspmm_lib.pspmm_rms_norm(ptr(x), dim, None, 0, ptr(w), t, n, dim, 1e-6, 0, None, dim, None, dim, ptr(rstd), ptr(q),
                                          pitch, ptr(scales), stream)
        else:
            rc = pspmm_lib.pspmm_quantize_rows(ptr(x), t, dim, n, dim, ptr(q), pitch, ptr(scales), stream)
        assert rc == 0
        assert not q[:, dim:used].any() and (q[:, used:] == 77).all()
        assert (q[:, :dim].abs().amax(1) == 127).all()
        out = torch.empty(n, dim, device="cuda")
        assert pspmm_lib.pspmm_dequantize_rows(ptr(q), pitch, ptr(scales), 0, ptr(out), dim, n, dim, stream) == 0
        assert torch.equal(out, q[:, :dim].float() * scales.repeat_interleave(BLOCK, 1)[:, :dim])
