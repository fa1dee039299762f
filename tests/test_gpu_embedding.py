"""Embedding lookup and its gradient.

The lookup is one 32-bit product and one rounding: equal to torch's.  The gradient of row t is a sum of the c rows of G whose id is
t, then a product: with u = 2^-24 and half = eps / 2 of the type, (c + 2) u |scale| sum |G| + half |result| at most.  Gradients of
whole numbers are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def sums(ids, G, V, padding=None):
    """(sum, sum of magnitudes, count) per row in 64 bits."""
    ids, G = ids.reshape(-1).long(), G.reshape(-1, G.shape[-1]).double()
    some = (ids >= 0) & (ids < V) & (ids != (-1 if padding is None else padding))
    ids, G = ids[some], G[some]
    total, size = (torch.zeros(V, G.shape[1], dtype=torch.float64, device=G.device) for _ in range(2))
    total.index_add_(0, ids, G)
    size.index_add_(0, ids, G.abs())
    return total, size, torch.bincount(ids, minlength=V).double()


def check_grad(ids, G, V, scale=1.0, padding=None):
    from paramspmm_ae_b200 import feature_ops as fo
    got = fo.embedding_grad(ids, G, V, scale, padding_idx=padding)
    assert got.shape == (V, G.shape[-1]) and got.dtype is G.dtype
    total, size, count = sums(ids, G, V, padding)
    want = total * scale
    bound = (count[:, None] + 2) * U * abs(scale) * size + torch.finfo(G.dtype).eps / 2 * want.abs()
    if G.dtype is torch.float16:
        bound = bound + 2.0 ** -25
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off - bound).max()
    assert not got[count == 0].any()
    assert torch.equal(got, fo.embedding_grad(ids, G, V, scale, padding_idx=padding))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 3, 4, 16, 47, 64, 100, 250, 256, 516, 1024, 1500])
@pytest.mark.parametrize("wide", [True, False])
def test_lookup(dtype, dim, wide):
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator().manual_seed(dim)
    table = torch.randn(301, dim, generator=g).to(dtype).cuda()
    for shape in ((0,), (1,), (777,), (5, 3, 7)):
        ids = torch.randint(0, 301, shape, generator=g, dtype=torch.int64 if wide else torch.int32).cuda()
        got = fo.embedding(ids, table, 3.7)
        assert torch.equal(got, (table[ids.long()].float() * torch.tensor(3.7, device="cuda")).to(dtype))
    assert torch.equal(fo.embedding(ids, table), table[ids.long()])


def test_lookup_from_a_view_and_out_of_range():
    from paramspmm_ae_b200 import feature_ops as fo
    wide = torch.randn(50, 90, device="cuda")
    ids = torch.tensor([0, 49, 7, 7], device="cuda")
    for a, b in ((0, 32), (1, 48), (4, 90)):
        assert torch.equal(fo.embedding(ids, wide[:, a:b]), wide[:, a:b][ids])
    for bad in (torch.tensor([0, 50, -1, 2 ** 40, 3], device="cuda"), torch.tensor([0, 50, -1, 2 ** 31 - 1, 3], device="cuda").int()):
        got = fo.embedding(bad, wide)
        assert torch.isnan(got[1:4]).all() and torch.equal(got[[0, 4]], wide[[0, 3]])
        G = torch.ones(5, 8, device="cuda")
        grad = fo.embedding_grad(bad, G, 50)
        assert (grad[[0, 3]] == 1).all() and grad.sum() == 16
    assert fo.embedding_status() == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 3, 16, 47, 64, 100, 250, 256, 516, 1024])
@pytest.mark.parametrize("n,V", [(1, 1), (7, 3), (33, 40), (600, 100), (2048, 5000), (2049, 300), (5000, 70000), (30000, 255),
                                 (30000, 256)])
def test_gradient(dtype, dim, n, V):
    g = torch.Generator().manual_seed(n + dim)
    ids = (torch.rand(n, generator=g) ** 3 * V).long().clamp_(max=V - 1).cuda()
    check_grad(ids, torch.randn(n, dim, generator=g).to(dtype).cuda(), V, scale=1.7)


@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 2047, 2048, 2049, 4096, 65536, 65537, 262145, 1048577])
def test_one_id_takes_everything(n):
    """All ids equal, all but one, runs that end and begin at the ends of chunks."""
    g = torch.Generator().manual_seed(n)
    G = torch.randint(-4, 5, (n, 20), generator=g).float().cuda()
    ids = torch.full((n,), 5, dtype=torch.int32, device="cuda")
    got = check_grad(ids, G, 9)
    assert torch.equal(got[5], G.sum(0, dtype=torch.float64).float())
    ids[n // 2] = 3
    check_grad(ids, G, 9)
    run = 32 if n <= 1 << 16 else 64 if n <= 1 << 18 else 128 if n <= 1 << 20 else 256
    for length in (run - 1, run, run + 1, 2 * run, 2 * run + 1, 3 * run - 1):
        ids = (torch.arange(n, device="cuda") // length)
        V = int(ids.max()) + 2
        got = check_grad(ids, G, V)
        assert torch.equal(got.sum(0), G.sum(0, dtype=torch.float64).float()) or n > 1 << 20
        check_grad(ids.flip(0).contiguous(), G, V)


def chunk_length(n):
    """Positions of a chunk of the gradient, from the pieces that its scratch has room for: two rows per chunk."""
    import ctypes
    from paramspmm_ae_b200 import _lib
    need = [ctypes.c_size_t(0) for _ in range(2)]
    for dim, c in zip((64, 128), need):  # (multiples of the 256 bytes that parts of the scratch are rounded to)
        _lib.check(_lib.lib().pspmm_embedding_grad_scratch_bytes(n, dim, ctypes.byref(c)))
    chunks = (need[1].value - need[0].value) // (2 * 64 * 4)
    return next(run for run in (2 ** i for i in range(12)) if (n + run - 1) // run == chunks)


@pytest.mark.parametrize("n,dim", [(2048, 20), (4096, 130), (4097, 47), (65536, 20), (65537, 130), (262145, 20), (1048576, 8), (1048577, 3)])
def test_runs_around_the_length_of_chunks(n, dim):
    """Runs one shorter and longer than a chunk, than a few, and than the 64 from which on a CTA of its own adds the pieces, that
    begin with a chunk and inside one.  Whole numbers: equality."""
    from paramspmm_ae_b200 import feature_ops as fo
    run = chunk_length(n)
    G = torch.randint(-4, 5, (n, dim), generator=torch.Generator().manual_seed(n)).float().cuda()
    for chunks in (1, 2, 3, 63, 64, 65, 66):
        for length in (chunks * run - 1, chunks * run, chunks * run + 1):
            for before in (0, 1, run // 2, run - 1, run + 3):
                ids = torch.div(torch.arange(n, device="cuda") + length - before % length, length, rounding_mode="floor")
                V = int(ids[-1]) + 2
                want = torch.zeros(V, dim, device="cuda").index_add_(0, ids, G)  # (whole numbers below 2^24 in any order)
                assert torch.equal(fo.embedding_grad(ids, G, V), want), (length, before)


@pytest.mark.parametrize("V", [1, 2, 255, 256, 257, 511, 512, 65535, 65536, 65537, 131072, 262143, 262144, 16777217])
@pytest.mark.parametrize("n", [3001, 70001])
def test_table_sizes(V, n):
    """Keys of one to three passes of every width, the last id among them, with few tiles of keys and with many."""
    g = torch.Generator().manual_seed(V)
    ids = (torch.rand(n, generator=g, dtype=torch.float64) * V).long().clamp_(max=V - 1)
    ids[:4] = V - 1
    G = torch.randint(-4, 5, (n, 4), generator=g).float()
    from paramspmm_ae_b200 import feature_ops as fo
    got = fo.embedding_grad(ids.cuda(), G.cuda(), V)
    want = torch.zeros(V, 4).index_add_(0, ids, G)
    assert torch.equal(got.cpu(), want)
    ids = ids[:1000]
    assert torch.equal(fo.embedding_grad(ids.cuda(), G[:1000].cuda(), V).cpu(), torch.zeros(V, 4).index_add_(0, ids, G[:1000]))


@pytest.mark.parametrize("n", [3001, 70001])
def test_a_table_of_four_passes(n):
    from paramspmm_ae_b200 import feature_ops as fo
    V = 2 ** 27 + 1
    g = torch.Generator().manual_seed(n)
    ids = (torch.rand(n, generator=g, dtype=torch.float64) * V).long().clamp_(max=V - 1).cuda()
    ids[:4] = V - 1
    G = torch.randint(1, 5, (n, 1), generator=g).float().cuda()
    got = fo.embedding_grad(ids, G, V)
    want = torch.zeros(V, 1, device="cuda").index_add_(0, ids, G)  # whole numbers: any order is exact
    assert torch.equal(got, want)


def test_padding_no_ids_no_rows():
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator().manual_seed(1)
    for n in (500, 9000):
        ids = torch.randint(0, 11, (n,), generator=g).cuda()
        ids[::3] = 4
        G = torch.randn(n, 33, generator=g).cuda()
        for pad in (0, 4, 10):
            assert not check_grad(ids, G, 11, 2.0, padding=pad)[pad].any()
    e = torch.empty(0, dtype=torch.int64, device="cuda")
    assert not fo.embedding_grad(e, torch.empty(0, 5, device="cuda"), 7).any()
    assert fo.embedding_grad(e, torch.empty(0, 5, device="cuda"), 0).shape == (0, 5)
    assert torch.isnan(fo.embedding(torch.zeros(2, dtype=torch.int64, device="cuda"), torch.empty(0, 5, device="cuda"))).all()


def test_gradient_of_views_and_shapes():
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 60, (40, 50), generator=g).cuda()
    check_grad(ids, torch.randn(40, 50, 24, generator=g).cuda(), 60)
    wide = torch.randn(2000, 80, generator=g).cuda()
    for a, b in ((0, 32), (1, 48), (4, 80)):
        check_grad(ids.reshape(-1), wide[:, a:b], 60)


def test_captured_and_on_two_streams():
    from paramspmm_ae_b200 import feature_ops as fo
    g = torch.Generator().manual_seed(3)
    for n in (1500, 20000):
        ids = torch.randint(0, 300, (n,), generator=g).cuda()
        table, G = torch.randn(300, 64, generator=g).cuda(), torch.randn(n, 64, generator=g).cuda()
        step = lambda: (fo.embedding(ids, table, 0.5), fo.embedding_grad(ids, G, 300, 0.5))
        alone = step()
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for _ in range(4):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for r in got for a, b in zip(r, alone))
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        outs = []
        for gr in graphs:
            with torch.cuda.graph(gr):
                outs.append(step())
        for seed in (4, 5):
            ids.copy_(torch.randint(0, 300, (n,), generator=torch.Generator().manual_seed(seed)))
            for gr in graphs:
                gr.replay()
            torch.cuda.synchronize()
            want = step()
            assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_refusals():
    from paramspmm_ae_b200 import feature_ops as fo
    ids, table = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(6, 8, device="cuda")
    for bad in (lambda: fo.embedding(ids.float(), table), lambda: fo.embedding(ids[::2], table), lambda: fo.embedding(ids, table.double()),
                lambda: fo.embedding(ids, table[0]), lambda: fo.embedding(ids, table.t()), lambda: fo.embedding_grad(ids, table, 6),
                lambda: fo.embedding_grad(ids, table[:4], 6, padding_idx=6), lambda: fo.embedding_grad(ids, table[:4], -1)):
        with pytest.raises(RuntimeError):
            bad()
