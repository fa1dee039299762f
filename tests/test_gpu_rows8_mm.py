"""Weight gradients from rows held in 8 bits, against fp64.

Tolerance, with u = 2^-24 and S = sum |q scale G| of an element: scale * G is rounded once (u S); a chain of 32 rows takes six
additions in the tensor core, which truncates (2 u each: 12 u S); then one addition per chain and one per range of rows, in sequence
at worst: (n / 32 + 40) u S.  Together less than (n / 32 + 64) u S.  Whole numbers are exact while sums stay below 2^24."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def held(n, dim, seed, exact=False):
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch, blocks = (dim + 15) // 16 * 16, (dim + 127) // 128
    q = torch.randint(-127, 128, (n, pitch), generator=g, device="cuda").to(torch.int8)  # (what lies beyond dim is not used)
    if exact:
        q = q.clamp(-3, 3)
        scales = 2.0 ** torch.randint(0, 3, (n, blocks), generator=g, device="cuda").float()
    else:
        scales = torch.exp(torch.randn(n, blocks, generator=g, device="cuda")) * 0.01
    return fo.Rows8(q, scales, dim)


def values(rows):
    return rows.q[:, :rows.dim].double() * rows.scales.double().repeat_interleave(128, 1)[:, :rows.dim]


def check(rows, G, **kw):
    from paramspmm_ae_b200 import feature_ops as fo
    got = fo.rows8_mm_t(rows, G, **kw)
    X, n = values(rows), G.shape[0]
    want, size = X.t() @ G.double(), X.abs().t() @ G.double().abs()
    off = (got.double() - want).abs()
    assert got.dtype is torch.float32 and got.shape == want.shape
    assert (off <= (n / 32 + 64) * U * size).all(), (off / (U * size).clamp(min=1e-300)).max()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,cols", [(1, 1), (16, 16), (47, 8), (128, 128), (100, 47), (129, 33), (256, 256), (500, 16), (16, 500),
                                      (130, 130), (384, 272), (1000, 7), (2048, 24)])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 95, 97, 1000, 10007])
def test_whole_numbers(dtype, dim, cols, n):
    from paramspmm_ae_b200 import feature_ops as fo
    rows = held(n, dim, n + dim, exact=True)
    G = torch.randint(-4, 5, (n, cols), generator=torch.Generator().manual_seed(n)).to(dtype).cuda()
    assert torch.equal(fo.rows8_mm_t(rows, G).double(), values(rows).t() @ G.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols,ld", [(47, 47), (1, 1), (2, 2), (7, 9), (33, 50), (130, 131), (64, 65)])
@pytest.mark.parametrize("n", [1, 33, 1000, 10007])
@pytest.mark.parametrize("at", [0, 1, 3])
def test_unaligned_rows_without_room_for_a_copy(dtype, cols, ld, n, at):
    """The C call with the scratch that it requires and no more; ``at``: where the first row begins."""
    from paramspmm_ae_b200 import _lib
    rows = held(n, 150, n + cols, exact=True)
    store = torch.full((n * ld + 8,), float("nan"), dtype=dtype, device="cuda")
    G = store[at:at + n * ld].view(n, ld)[:, :cols]
    G.copy_(torch.randint(-4, 5, (n, cols), generator=torch.Generator().manual_seed(n)))
    need = ctypes.c_size_t(0)
    code = TYPES.index(dtype)
    _lib.check(_lib.lib().pspmm_rows8_mm_t_scratch_bytes(n, 150, cols, code, 1, ctypes.byref(need)))
    scratch = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda")
    C = torch.full((150, cols), float("nan"), device="cuda")
    _lib.check(_lib.lib().pspmm_rows8_mm_t(rows.q.data_ptr(), rows.q.shape[1], rows.scales.data_ptr(), n, 150, G.data_ptr(), code, ld,
                                           cols, C.data_ptr(), cols, scratch.data_ptr(), need.value,
                                           torch.cuda.current_stream().cuda_stream))
    want = values(rows).t() @ G.double()
    assert torch.equal(C.double(), want)
    from paramspmm_ae_b200 import feature_ops as fo
    if cols > 1:
        assert torch.equal(fo.rows8_mm_t(rows, G).double(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,cols,n", [(1, 1, 5), (47, 8, 300), (100, 47, 2001), (256, 256, 9000), (500, 16, 19717), (1024, 1024, 3000),
                                        (64, 300, 100003), (1760, 103, 1501)])
def test_real_values(dtype, dim, cols, n):
    rows = held(n, dim, n)
    G = (torch.randn(n, cols, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda") * 1e-3).to(dtype)
    got = check(rows, G)
    assert torch.equal(got, check(rows, G))


def test_no_bias_over_a_long_sum():
    """300,000 rows of one sign: truncation in long chains would lose a part in a thousand."""
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 300000
    rows = fo.Rows8(torch.randint(1, 128, (n, 64), generator=g, device="cuda").to(torch.int8), torch.rand(n, 1, generator=g, device="cuda"), 64)
    G = torch.rand(n, 40, generator=g, device="cuda")
    got, want = fo.rows8_mm_t(rows, G).double(), values(rows).t() @ G.double()
    # chains of 32 lose at most 12 u each, then 300,000 / 32 additions rounded to nearest over the ranges of rows; measured against
    # 64 u, as if a third of all errors agreed
    assert ((got - want).abs() / want).max() <= 64 * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,cols", [(47, 8), (130, 130)])
@pytest.mark.parametrize("n", [1, 32, 63, 64, 65, 128, 129, 1000, 10007, 100003])
def test_chains_as_they_are(dtype, dim, cols, n):
    """The bound from the chains that the kernel runs, on values of one sign, where truncations agree: two stages of 32 rows, of each
    three parts in two instructions, so 12 truncating additions (24 u S) per 64 rows; scale * G is rounded once (u S); then one addition
    per chain, and over at most 592 ranges of rows 19 + 3 + 2 + 7 in sequence.  Together less than (n / 64 + 60) u S."""
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    rows = fo.Rows8(torch.randint(1, 128, (n, (dim + 15) // 16 * 16), generator=g, device="cuda").to(torch.int8),
                    torch.rand(n, (dim + 127) // 128, generator=g, device="cuda") + 0.01, dim)
    G = (torch.rand(n, cols, generator=g, device="cuda") + 1e-3).to(dtype)
    got, want = fo.rows8_mm_t(rows, G).double(), values(rows).t() @ G.double()
    assert ((got - want).abs() <= (n / 64 + 60) * U * want).all(), ((got - want).abs() / want).max().item() / U


def test_rows_quantised_here_and_views():
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator(device="cuda").manual_seed(2)
    H = torch.relu(torch.randn(3001, 200, generator=g, device="cuda"))
    rows = fo.quantize_rows(H)
    wide = torch.randn(3001, 100, generator=g, device="cuda")
    for a, b in ((0, 64), (1, 48), (4, 100), (0, 47)):
        check(rows, wide[:, a:b])
    out = torch.full((200, 90), 7.0, device="cuda")
    check(rows, wide[:, :47], out=out[:, 20:67])
    assert (out[:, :20] == 7).all() and (out[:, 67:] == 7).all()


def test_gradient_of_the_values_held_against_autograd():
    """d/dW of <(q scale) W, G> is what the product gives; and within the 8 bits' error it is the gradient from the fp32 input."""
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator(device="cuda").manual_seed(3)
    H, G = torch.randn(500, 140, generator=g, device="cuda"), torch.randn(500, 20, generator=g, device="cuda")
    rows = fo.quantize_rows(H)
    W = torch.zeros(140, 20, dtype=torch.float64, device="cuda", requires_grad=True)
    ((rows.dequantize().double() @ W) * G.double()).sum().backward()
    got = check(rows, G).double()
    # dequantize rounds q * scale once more, u of every term
    assert ((got - W.grad).abs() <= (500 / 32 + 66) * U * (values(rows).abs().t() @ G.double().abs())).all()
    full = H.double().t() @ G.double()
    step = rows.scales.double().repeat_interleave(128, 1)[:, :140] * (0.5 + 2 ** -15)
    assert ((got - full).abs() <= step.t() @ G.double().abs() + 80 * U * (H.double().abs().t() @ G.double().abs())).all()


def test_infinities_and_nans():
    from paramspmm_ae_b200 import feature_ops as fo
    rows = held(100, 300, 4, exact=True)
    rows.q[7, 0], rows.q[7, 1], rows.q[7, 2] = 2, -2, 0
    G = torch.ones(100, 30, device="cuda")
    G[7, 3], G[7, 4], G[7, 5] = float("inf"), float("-inf"), float("nan")
    G[8, 6] = 3.3e38  # finite, rounds up in 8 bits
    rows.q[8, :], rows.scales[8, :] = 1, 1.0
    rows.scales[9, 1] = float("nan")
    got = fo.rows8_mm_t(rows, G).cpu()
    inf = float("inf")
    assert got[0, 3] == inf and got[1, 3] == -inf and torch.isnan(got[2, 3])
    assert got[0, 4] == -inf and got[1, 4] == inf and torch.isnan(got[2, 4])
    assert torch.isnan(got[:, 5]).all()
    assert torch.isnan(got[128:256]).all()  # the block whose scale is NaN
    some = [c for c in range(30) if c not in (3, 4, 5)]
    assert torch.isfinite(got[:128][:, some]).all() and torch.isfinite(got[256:][:, some]).all()
    assert abs(got[0, 6] / 3.3e38 - 1) < 1e-5
    G[8, 6] = 1.0
    rows.scales[9, 1] = 1.0
    G[7, 3:6] = 1.0
    check(rows, G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [130, 128, 47])  # rows of G on 16 bytes and off them (16 bits: 130 columns, 260 bytes)
def test_an_infinity_in_every_stage(dtype, cols):
    """Stages whose values have no split are stored a second time, value by value: the second store is the one that counts.  Whole
    numbers beside one infinity per column of G, at a row of another stage each: equality, signs and NaN included."""
    from paramspmm_ae_b200 import feature_ops as fo
    n = 32 * cols - 5
    rows = held(n, 300, cols, exact=True)
    G = torch.randint(-4, 5, (n, cols), generator=torch.Generator().manual_seed(cols)).to(dtype).cuda()
    at = (torch.arange(cols) * 32 + torch.arange(cols) * 7 % 27).cuda()
    G[at, torch.arange(cols).cuda()] = torch.where(torch.arange(cols) % 2 == 0, float("inf"), float("-inf")).to(dtype).cuda()
    X, inf = values(rows), float("inf")
    want = torch.where(X[at].t() == 0, float("nan"), torch.where(X[at].t() > 0, inf, -inf)) * torch.where(torch.arange(cols).cuda() % 2 == 0, 1.0, -1.0)
    for _ in range(4):
        torch.testing.assert_close(fo.rows8_mm_t(rows, G), want.float(), rtol=0, atol=0, equal_nan=True)


def test_no_rows_captured_other_streams():
    from paramspmm_ae_b200 import feature_ops as fo
    e = held(0, 40, 1)
    assert not fo.rows8_mm_t(e, torch.empty(0, 9, device="cuda")).any()
    rows, G = held(5000, 256, 5), torch.randn(5000, 64, device="cuda")
    alone = fo.rows8_mm_t(rows, G)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(fo.rows8_mm_t(rows, G))
    torch.cuda.synchronize()
    assert all(torch.equal(a, alone) for a in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fo.rows8_mm_t(rows, G)
    G.mul_(-2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alone * -2)


def test_refusals():
    from paramspmm_ae_b200 import feature_ops as fo
    rows, G = held(60, 40, 6), torch.zeros(60, 8, device="cuda")
    for bad in (lambda: fo.rows8_mm_t(rows.q, G), lambda: fo.rows8_mm_t(rows, G[:59]), lambda: fo.rows8_mm_t(rows, G.double()),
                lambda: fo.rows8_mm_t(rows, G.cpu()), lambda: fo.rows8_mm_t(rows, G.t()),
                lambda: fo.rows8_mm_t(rows, G, out=torch.zeros(40, 9, device="cuda")),
                lambda: fo.rows8_mm_t(rows, G, out=torch.zeros(40, 8, device="cuda", dtype=torch.float16))):
        with pytest.raises(RuntimeError):
            bad()


def test_a_wait_that_runs_out_is_told():
    """The status stays set for the process: in a process of its own."""
    import subprocess
    import sys
    code = """
import ctypes, torch
from paramspmm_ae_b200 import _lib, feature_ops as fo
lib = _lib.lib()
q, s, G = torch.ones(400, 64, dtype=torch.int8, device="cuda"), torch.ones(400, 1, device="cuda"), torch.ones(400, 32, device="cuda")
rows = fo.Rows8(q, s, 64)
assert (fo.rows8_mm_t(rows, G) == 400).all() and fo.rows8_mm_status() == 0
need = ctypes.c_size_t(0)
_lib.check(lib.pspmm_rows8_mm_t_scratch_bytes(400, 64, 32, 0, 1, ctypes.byref(need)))
scratch = torch.zeros(max(need.value, 16), dtype=torch.uint8, device="cuda")
C = torch.zeros(64, 32, device="cuda")
_lib.check(lib.pspmm_rows8_mm_t_stalled(q.data_ptr(), 64, s.data_ptr(), 400, 64, G.data_ptr(), 0, 32, 32, C.data_ptr(), 32,
                                        scratch.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream))
torch.cuda.synchronize()
assert torch.isnan(C).all() and fo.rows8_mm_status() == 1
assert (fo.rows8_mm_t(rows, G) == 400).all()
print("told")
"""
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "told" in p.stdout, p.stderr
