"""Root-mean-square norm with the residual's addition against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of the 32 bits the kernel computes in) and half = eps / 2 of the type, the rounding of what
is stored.  fp16 also has subnormals, 2^-25 off at most.
h     one 32-bit rounding of x + r, one of the store:                            (u + half) |h|
y     h, rstd, and two products, one rounding each, and what h's roundings do to rstd (u at most):  (5 u + half) |y|
dx    rstd (g - m s) + dh with m = h rstd, g = dy w, s = mean(g m).  m and g carry 2 u each; a product g m then 4 u and its
      addition; s is a sum of at most 16 terms per thread, five steps of shuffles, 32 warps and a division: (16 + 5 + 32 + 5) u of
      the mean magnitude A = mean |g m|.  So rstd (4 u |g| + |m| (64 + 4) u A) + 4 u of the result's parts + half |dx|
      (rows wider than 8,192 columns: a thread adds dim / 1024 terms, in the place of 16)
dw    sum over rows of dy m: 4 u per term, rows in sequence and then tree: at most n + 60 additions, u each, of the sum of magnitudes
"""
import pytest
import torch

from test_gpu_rows8 import check

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return 2.0 ** -25 if t is torch.float16 else 0.0


def inputs(n, dim, dtype, seed, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, dim, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype)
    r = torch.randn(n, dim, generator=g).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype)
    return x, r, w


def formula(x, r, w, eps, relu):
    h = x.double() + (r.double() if r is not None else 0)
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = h * rstd * w.double()
    return h, rstd, y.clamp(min=0) if relu else y


def close(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), "off by %.3g where %.3g is allowed" % (
        (off - bound).max().item(), bound.reshape(-1)[(off - bound).reshape(-1).argmax()].item())


def check_forward(x, r, w, eps=1e-6, relu=False, eight=False, values=True, move=lambda t: t):
    from paramspmm_ae_b200 import feature_ops as fo
    t = x.dtype
    y, h, rstd, kept = fo.rms_norm(move(x.cuda()), w.cuda(), None if r is None else move(r.cuda()), eps=eps, relu=relu,
                                   eight_bit=eight, values=values)
    h64, rstd64, y64 = formula(x, r, w, eps, relu)
    if values:
        assert y.dtype is t and y.shape == x.shape
        close(y, y64, (5 * U + half(t)) * y64.abs() + tiny(t))
    else:
        assert y is None
    close(h, h64, (U + half(t)) * h64.abs() + tiny(t))
    close(rstd, rstd64.squeeze(-1), 2 * U * rstd64.squeeze(-1))
    if eight:
        check(kept, y64.reshape(-1, x.shape[-1]))
    else:
        assert kept is None
    return h, rstd


WIDTHS = [1, 2, 8, 16, 24, 31, 32, 33, 47, 63, 64, 72, 100, 128, 130, 144, 192, 200, 250, 256, 260, 384, 500, 512, 520, 1000, 1024, 1030, 2047, 2048, 2056, 4096,
          4100, 8191, 8192, 8200, 10001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_forward(dtype, dim):
    n = 67 if dim < 2000 else 9
    x, r, w = inputs(n, dim, dtype, dim)
    check_forward(x, r, w)
    check_forward(x, r, w, relu=True, eight=True)
    check_forward(x, None, w, eight=True, values=False)


@pytest.mark.parametrize("n", [0, 1, 2, 33, 1000, 40013])
@pytest.mark.parametrize("dim", [16, 47, 96, 1100])
def test_row_counts(n, dim):
    if n * dim > 5000000:
        n = 3001
    x, r, w = inputs(n, dim, torch.float32, n + dim)
    check_forward(x, r, w, relu=True, eight=True)
    check_forward(x, r, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_and_shapes(dtype):
    """Rows of a wider array, at aligned and at odd places, and arrays of more dimensions."""
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = inputs(50, 300, dtype, 5)
    for a, b in ((0, 64), (8, 136), (4, 104), (1, 102), (3, 300)):
        wide_x, wide_r = x.cuda(), r.cuda()
        y, h, _, kept = fo.rms_norm(wide_x[:, a:b], w[a:b].cuda(), wide_r[:, a:b], eight_bit=True)
        h64, _, y64 = formula(x[:, a:b], r[:, a:b], w[a:b], 1e-6, False)
        close(y, y64, (5 * U + half(dtype)) * y64.abs() + tiny(dtype))
        close(h, h64, (U + half(dtype)) * h64.abs() + tiny(dtype))
        check(kept, y64)
    x, r, w = inputs(24, 40, dtype, 6)
    check_forward(x.reshape(2, 3, 4, 40), r.reshape(2, 3, 4, 40), w, eight=True)
    check_forward(x[0], r[0], w)


def test_a_misaligned_weight():
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = inputs(20, 64, torch.float32, 7)
    store = torch.zeros(65, device="cuda")
    store[1:] = w.cuda()
    y = fo.rms_norm(x.cuda(), store[1:], r.cuda())[0]
    _, _, y64 = formula(x, r, w, 1e-6, False)
    close(y, y64, 5 * U * y64.abs() + U * y64.abs())


def test_rows_of_zeros_and_values_at_the_ends():
    from paramspmm_ae_b200 import feature_ops as fo
    x, _, w = inputs(7, 256, torch.float32, 8)
    x[0] = 0
    x[1] *= 1e30       # squares beyond 32 bits
    x[2] *= 1e-30
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    y, _, rstd, kept = fo.rms_norm(x.cuda(), w.cuda(), eight_bit=True)
    y, got = y.cpu(), kept.dequantize().cpu()
    _, _, y64 = formula(x, None, w, 1e-6, False)
    for r in (0, 1, 2, 5, 6):
        close(y[r], y64[r], 6 * U * y64[r].abs() + 1e-44)
        assert torch.isfinite(got[r]).all()
    assert torch.isnan(y[3]).all() and torch.isnan(got[3]).all()
    # h = inf: rstd = 0, so 0 * inf = NaN there and 0 elsewhere; the 8-bit block that holds the NaN comes back as NaN
    assert torch.isnan(y[4, 9]) and (y[4, 10:] == 0).all() and torch.isnan(got[4, :128]).all() and not got[4, 128:].any()
    y = fo.rms_norm(x.cuda(), w.cuda(), eps=0.0)[0].cpu()
    assert torch.isnan(y[0]).all() and torch.isfinite(y[[1, 2, 5, 6]]).all()  # 0 * (1 / 0)
    relu = fo.rms_norm(x.cuda(), w.cuda(), relu=True)[0].cpu()
    assert torch.isnan(relu[3]).all() and (relu[5] >= 0).all()


@pytest.mark.parametrize("dim", [64, 300, 1100, 4101])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_residuals_at_the_ends(dtype, dim):
    """Sums whose squares and remainders leave 32 bits, infinities and NaN on either side of the addition."""
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = inputs(8, dim, dtype, 21)
    x[0] *= 1e25
    r[1] *= 1e30
    x[2], r[2] = x[2] * 1e28, r[2] * 1e21  # the remainders of a row, added up, leave 32 bits
    x[3, 5] = r[4, 6] = float("inf")
    r[5, 7] = float("nan")
    x[6, 8], r[6, 8] = float("inf"), float("-inf")
    y, h, rstd, kept = fo.rms_norm(x.cuda(), w.cuda(), r.cuda(), eight_bit=True)
    h64, rstd64, y64 = formula(x, r, w, 1e-6, False)
    rows = [0, 1, 2, 7]
    close(y[rows], y64[rows], (5 * U + half(dtype)) * y64[rows].abs() + 1e-44)
    close(rstd[rows], rstd64[rows].squeeze(-1), 2 * U * rstd64[rows].squeeze(-1))
    check(fo.Rows8(kept.q[rows].contiguous(), kept.scales[rows].contiguous(), dim), y64[rows])
    y, h = y.cpu(), h.cpu()
    for row, c in ((3, 5), (4, 6)):
        assert torch.isinf(h[row, c]) and rstd[row] == 0
        assert torch.isnan(y[row, c]) and not y[row, c + 1:].any()
    assert torch.isnan(y[5:7]).all() and torch.isnan(rstd[5:7]).all()


def backward_formula(dy, h, rstd, w, dh, relu):
    h, w, rstd = h.double(), w.double(), rstd.double().unsqueeze(-1)
    m = h * rstd
    dy = dy.double()
    if relu:
        dy = dy * (m * w > 0)
    g = dy * w
    s = (g * m).mean(-1, keepdim=True)
    size = (g * m).abs().mean(-1, keepdim=True)
    dx = rstd * (g - m * s)
    parts = rstd * (4 * U * g.abs() + 4 * U * (m * s).abs() + 68 * U * m.abs() * size)
    if dh is not None:
        dx = dx + dh.double()
    flat = (dy * m).reshape(-1, h.shape[-1])
    dw, dw_size = flat.sum(0), flat.abs().sum(0)
    return dx, parts, dw, dw_size, flat.shape[0]


def check_backward(x, r, w, relu, stream, seed, move=lambda t: t):
    from paramspmm_ae_b200 import feature_ops as fo
    t = x.dtype
    g = torch.Generator().manual_seed(seed)
    dy = torch.randn(x.shape, generator=g).to(t)
    dh = torch.randn(x.shape, generator=g).to(t) if stream else None
    _, h, rstd, _ = fo.rms_norm(x.cuda(), w.cuda(), None if r is None else r.cuda(), relu=relu)
    dx, dw = fo.rms_norm_backward(move(dy.cuda()), h, rstd, w.cuda(), None if dh is None else move(dh.cuda()), relu=relu)
    dx64, parts, dw64, dw_size, n = backward_formula(dy, h.cpu(), rstd.cpu(), w, dh, relu)
    wide = max(1.0, x.shape[-1] / 1024 / 16)
    close(dx, dx64, wide * parts + (4 * U + half(t)) * dx64.abs() + tiny(t))
    close(dw, dw64, (n + 64) * U * dw_size + half(t) * dw64.abs() + tiny(t))
    assert dx.dtype is t and dw.dtype is t
    again = fo.rms_norm_backward(move(dy.cuda()), h, rstd, w.cuda(), None if dh is None else move(dh.cuda()), relu=relu)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_backward(dtype, dim):
    n = 67 if dim < 2000 else 9
    x, r, w = inputs(n, dim, dtype, dim)
    check_backward(x, r, w, False, True, 1)
    check_backward(x, None, w, True, False, 2)


@pytest.mark.parametrize("n", [1, 2, 31, 1000, 40013])
@pytest.mark.parametrize("dim", [16, 47, 96, 1100])
def test_backward_row_counts(n, dim):
    if n * dim > 5000000:
        n = 3001
    x, r, w = inputs(n, dim, torch.float32, n + dim)
    check_backward(x, r, w, True, True, n)


def test_backward_of_no_rows_and_of_views():
    from paramspmm_ae_b200 import feature_ops as fo
    w = torch.ones(24, device="cuda")
    e = torch.empty(0, 24, device="cuda")
    dx, dw = fo.rms_norm_backward(e, e, torch.empty(0, device="cuda"), w)
    assert dx.shape == (0, 24) and dw.shape == (24,) and not dw.any()
    x, r, w = inputs(40, 60, torch.float32, 9)

    def at_an_odd_place(t):
        wide = torch.empty(t.shape[0], 75, device="cuda")
        wide[:, 3:63] = t
        return wide[:, 3:63]

    check_backward(x, r, w, False, True, 3, move=at_an_odd_place)


def test_gradients_against_differences():
    """fp64 differences of the formula the kernel computes, at a few places."""
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = inputs(5, 40, torch.float32, 10)
    dy = torch.randn(5, 40, generator=torch.Generator().manual_seed(1))
    _, h, rstd, _ = fo.rms_norm(x.cuda(), w.cuda(), r.cuda(), relu=True)
    dx, dw = fo.rms_norm_backward(dy.cuda(), h, rstd, w.cuda(), relu=True)
    loss = lambda x, w: (formula(x, r, w, 1e-6, True)[2] * dy.double()).sum()
    d = 1e-6  # (the difference's own error: d^2 times a third derivative of order 10)
    for i, j in ((0, 0), (2, 17), (4, 39)):
        e = torch.zeros(5, 40, dtype=torch.float64)
        e[i, j] = d
        want = (loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * d)
        assert abs(dx[i, j].item() - want) <= 1e-5 * max(1, abs(want))
        want = (loss(x.double(), w.double() + e[i]) - loss(x.double(), w.double() - e[i])) / (2 * d)
        assert abs(dw[j].item() - want) <= 1e-5 * max(1, abs(want))


def test_two_streams_and_a_captured_step():
    """Calls on two streams at once give what they give alone; a captured step is replayed on new inputs."""
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = (t.cuda() for t in inputs(5000, 192, torch.float32, 11))
    dy = torch.randn_like(x)

    def step():
        y, h, rstd, kept = fo.rms_norm(x, w, r, relu=True, eight_bit=True)
        dx, dw = fo.rms_norm_backward(dy, h, rstd, w, dh=y, relu=True)
        return y, h, kept.q, kept.scales, dx, dw

    alone = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, alone))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.mul_(0.5).add_(0.1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals():
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = (t.cuda() for t in inputs(6, 32, torch.float32, 12))
    for bad in (lambda: fo.rms_norm(x.double(), w), lambda: fo.rms_norm(x, w.half()), lambda: fo.rms_norm(x, w[:31]),
                lambda: fo.rms_norm(x, w, r[:5]), lambda: fo.rms_norm(x, w, r.half()), lambda: fo.rms_norm(x.t(), w),
                lambda: fo.rms_norm(x, w, eps=-1.0), lambda: fo.rms_norm(x, w, values=False), lambda: fo.rms_norm(x, w[::1].expand(2, 32)),
                lambda: fo.rms_norm_backward(x[:5], x, torch.ones(6, device="cuda"), w),
                lambda: fo.rms_norm_backward(x, x, torch.ones(5, device="cuda"), w),
                lambda: fo.rms_norm_backward(x, x, torch.ones(6, device="cuda").double(), w)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 36), (torch.float32, 47), (torch.float32, 100), (torch.float32, 4100), (torch.float32, 8200),
                                       (torch.bfloat16, 24), (torch.bfloat16, 100), (torch.bfloat16, 250), (torch.bfloat16, 2056), (torch.float16, 4101)])
def test_columns_behind_rows_of_nan_are_zeros_in_8_bits(dtype, dim):
    """The columns from dim to the next multiple of 16, whatever the row holds."""
    from paramspmm_ae_b200 import feature_ops as fo
    x, r, w = inputs(9, dim, dtype, 31)
    x[0, 0], x[1, dim - 1], x[2, dim // 2] = float("nan"), float("nan"), float("inf")
    x[3], r[3] = 0, 0
    x[4] = float("nan")
    for eps in (1e-6, 0.0):
        for relu in (False, True):
            kept = fo.rms_norm(x.cuda(), w.cuda(), r.cuda(), eps=eps, relu=relu, eight_bit=True)[3]
            assert kept.q.shape[1] == (dim + 15) // 16 * 16 and not kept.q[:, dim:].any()


def rows_between_two_roundings(n, dim, dtype, seed):
    """Rows whose (mean h^2)^-1/2 lies, as far as 64 bits tell, half way between two 32-bit numbers: the order in which the squares are
    added decides which of the two it becomes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, dim, generator=g).to(dtype).double()
    x[:, -8:] = 0
    near = x.square().mean(-1).mul(1.0001).rsqrt().float()
    half_way = (near.double() + torch.nextafter(near, torch.zeros_like(near)).double()) / 2
    want = half_way.pow(-2) * dim
    for c in range(dim - 8, dim):  # what is missing, as far as one more value can give it
        x[:, c] = (want - x.square().sum(-1)).clamp(min=0).sqrt().mul(1 - 2.0 ** -12 if c < dim - 1 else 1).to(dtype).double()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [24, 68, 96, 132, 144, 192, 260, 300, 384, 1000, 2056])
def test_the_8_bit_form_leaves_the_other_outputs_alone(dtype, dim):
    from paramspmm_ae_b200 import feature_ops as fo
    x = rows_between_two_roundings(30000, dim, dtype, dim).cuda()
    w, r = torch.ones(dim, dtype=dtype, device="cuda"), torch.zeros_like(x)
    for residual in (None, r):
        y, h, rstd, _ = fo.rms_norm(x, w, residual, eps=0.0)
        y8, h8, rstd8, _ = fo.rms_norm(x, w, residual, eps=0.0, eight_bit=True)
        assert torch.equal(h, h8) and torch.equal(rstd, rstd8) and torch.equal(y, y8), (rstd != rstd8).sum().item()
