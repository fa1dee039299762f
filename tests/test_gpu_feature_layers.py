"""The layers around the graph layers, and graph layers that keep their input in 8 bits: gradients through autograd, alone and in a
deep network that uses all of them."""
import pytest
import torch

from test_gpu_layers import _close, _graph, _operator

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _step(rows):
    """Largest error of each value held: half a step of its block's scale."""
    return rows.scales.double().repeat_interleave(128, 1)[:, :rows.dim] * (0.5 + 2 ** -15)


def test_node_embedding_trains():
    from paramspmm_ae_b200 import gnn_conv
    torch.manual_seed(1)
    layer = gnn_conv.NodeEmbedding(50, 24, scale=2.5, padding_idx=7).cuda()
    assert not layer.weights[7].any()
    ids = torch.randint(0, 50, (4, 100), device="cuda")
    ids[0, :9] = 7
    G = torch.randn(4, 100, 24, device="cuda")
    out = layer(ids)
    out.backward(G)
    W = layer.weights.detach().double().requires_grad_(True)
    ref = 2.5 * W[ids]
    (ref * G.double() * (ids != 7).unsqueeze(-1)).sum().backward()
    _close(out.detach(), ref.detach())
    _close(layer.weights.grad, W.grad)
    assert not layer.weights.grad[7].any()
    (layer(ids).sum()).backward()  # an expanded gradient


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("uses", ["y", "h", "both"])
def test_rms_norm_layer(relu, residual, uses):
    from paramspmm_ae_b200 import gnn_conv
    torch.manual_seed(2)
    layer = gnn_conv.RMSNorm(70, relu=relu).cuda()
    layer.weights.data.uniform_(0.5, 1.5)
    x = torch.randn(33, 70, device="cuda", requires_grad=True)
    r = torch.randn(33, 70, device="cuda", requires_grad=True) if residual else None
    a, b = torch.randn(33, 70, device="cuda"), torch.randn(33, 70, device="cuda")
    loss = lambda y, h, a, b: ((y * a).sum() if uses != "h" else 0) + ((h * b).sum() if uses != "y" else 0)
    loss(*layer(x, r), a, b).backward()
    X, W = x.detach().double().requires_grad_(True), layer.weights.detach().double().requires_grad_(True)
    R = r.detach().double().requires_grad_(True) if residual else None
    H = X + R if residual else X
    Y = H * (H.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * W
    loss(torch.relu(Y) if relu else Y, H, a.double(), b.double()).backward()
    _close(x.grad, X.grad)
    if residual:
        _close(r.grad, R.grad)
    if uses == "h":
        assert layer.weights.grad is None
    else:
        _close(layer.weights.grad, W.grad)


def test_rms_norm_layer_refuses_a_second_derivative():
    from paramspmm_ae_b200 import gnn_conv
    layer = gnn_conv.RMSNorm(8).cuda()
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(layer(x)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("split", [False, "plan"])
@pytest.mark.parametrize("fin,fout", [(12, 32), (140, 16), (32, 47)])
@pytest.mark.parametrize("reorder", [False, True])
def test_gcn_layer_with_its_input_in_8_bits(split, fin, fout, reorder):
    from paramspmm_ae_b200 import feature_ops, gnn_conv
    dev = torch.device("cuda:0")
    g, A = _graph(dev)
    P = _operator(g, dev, split)
    torch.manual_seed(3)
    layer = gnn_conv.GCNConv(fin, fout).to(dev)
    H = torch.randn(g.n_rows, fin, device=dev, requires_grad=True)
    G = torch.randn(g.n_rows, fout, device=dev)
    old, gnn_conv.REORDER_NARROW_FIRST = gnn_conv.REORDER_NARROW_FIRST, reorder
    try:
        got = []
        for eight, kept in ((False, None), (True, None), (False, feature_ops.quantize_rows(H.detach()))):
            layer.keep_input_8bit = eight
            H.grad = layer.weights.grad = None
            out = layer(H, {fout: P, fin: P}, kept) if kept is not None else layer(H, {fout: P, fin: P})
            out.backward(G)
            got.append((out.detach(), H.grad.clone(), layer.weights.grad.clone()))
    finally:
        gnn_conv.REORDER_NARROW_FIRST = old
    for other in got[1:]:
        assert torch.equal(other[0], got[0][0]) and torch.equal(other[1], got[0][1])
        assert torch.equal(other[2], got[1][2])
    narrow = reorder and fin < fout
    held = (A @ H.detach().double()).float() if narrow else H.detach()
    other = G.double() if narrow else A @ G.double()
    bound = _step(feature_ops.quantize_rows(held)).t() @ other.abs()
    off = (got[1][2].double() - held.double().t() @ other).abs()
    assert (off <= 1.01 * bound + 1e-4).all() and off.max() > 1e-5  # (1.01: fp32 sums in A G and A H)
    saved = []
    layer.keep_input_8bit = True
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.dtype) or t, lambda t: t):
        layer(H, {fout: P, fin: P})
    assert torch.int8 in saved


def test_gin_and_agnn_layers_with_their_inputs_in_8_bits():
    from paramspmm_ae_b200 import feature_ops, gnn_conv
    dev = torch.device("cuda:0")
    g, A = _graph(dev)
    P = _operator(g, dev, False)
    torch.manual_seed(4)
    X = torch.randn(g.n_rows, 150, device=dev)
    X = (X / X.norm(dim=1, keepdim=True)).requires_grad_(True)
    col = P.colIdx.unsqueeze(-1)
    for kind in ("gin", "agnn fused", "agnn recomputed", "agnn composed"):
        layer = (gnn_conv.GINConv if kind == "gin" else gnn_conv.AGNNConv)(150, 32).to(dev)
        layer.keep_scores = kind != "agnn recomputed"
        G = torch.randn(g.n_rows, 32, device=dev)
        fused, gnn_conv.FUSE_AGNN_TRAINING = gnn_conv.FUSE_AGNN_TRAINING, kind != "agnn composed"
        try:
            got = []
            for eight in (False, True, "kept"):
                if eight == "kept" and kind == "gin":
                    continue
                layer.keep_input_8bit = eight is True
                layer.zero_grad()
                X.grad = None
                args = () if kind == "gin" else (col,)
                if eight == "kept":
                    args += (feature_ops.quantize_rows(X.detach()),)
                out = layer(X, {32: P}, *args)
                out.backward(G)
                got.append([out.detach(), X.grad.clone(), layer.weights.grad.clone()])
        finally:
            gnn_conv.FUSE_AGNN_TRAINING = fused
        for other in got[1:]:
            assert torch.equal(other[0], got[0][0]) and torch.equal(other[1], got[0][1]) and torch.equal(other[2], got[1][2])
        # the weight gradient is linear in what is held: off by its error times the other factor, whose size is at most
        held = (A @ X.detach().double()).float() if kind == "gin" else X.detach()
        if kind == "gin":
            other = G.double()
        else:
            W, beta = layer.weights.detach().double(), layer.attention_w.detach().double()
            Xp = X.detach().double() @ W
            other = ((A != 0) * (Xp @ Xp.t()) * beta) @ G.double()
        bound = _step(feature_ops.quantize_rows(held)).t() @ other.abs()
        off = (got[1][2].double() - held.double().t() @ other).abs()
        assert (off <= 1.01 * bound + 1e-4).all() and off.max() > 1e-5


def test_what_a_layer_refuses_to_keep():
    from paramspmm_ae_b200 import feature_ops, gnn_conv
    dev = torch.device("cuda:0")
    g, _ = _graph(dev)
    P = _operator(g, dev, False)
    layer = gnn_conv.GCNConv(20, 16).to(dev)
    H = torch.randn(g.n_rows, 20, device=dev)
    for kept in (H, feature_ops.quantize_rows(H[:, :19].contiguous()), feature_ops.quantize_rows(H[:-1])):
        with pytest.raises(RuntimeError, match="8 bits"):
            layer(H, {16: P}, kept)
    layer.keep_input_8bit = True
    with torch.no_grad():
        layer(H, {16: P})


class _Deep(torch.nn.Module):
    """Learned features, then blocks of norm, relu and a graph layer on a residual stream."""

    def __init__(self, n, dim, classes, blocks, eight):
        super().__init__()
        from paramspmm_ae_b200 import gnn_conv
        self.eight, self.trace = eight, None
        self.features = gnn_conv.NodeEmbedding(n, dim, scale=dim ** 0.5)
        self.norms = torch.nn.ModuleList(gnn_conv.RMSNorm(dim, relu=True) for _ in range(blocks))
        self.convs = torch.nn.ModuleList(gnn_conv.GCNConv(dim, dim if b < blocks - 1 else classes) for b in range(blocks))

    def forward(self, ids, operators):
        x, h = self.features(ids), None
        for norm, conv in zip(self.norms, self.convs):
            y, h, *kept = norm(x, h, eight_bit=self.eight)
            x = conv(y, operators, *kept)
            if self.trace is not None:
                x.retain_grad()
                self.trace.append((kept, x))
        return x

    def formula(self, ids, A):
        """The same in fp64 from parameters ``p``."""
        p = {k: v.detach().double().requires_grad_(True) for k, v in self.named_parameters()}
        x, h = p["features.weights"][ids] * self.features.scale, 0
        for b, norm in enumerate(self.norms):
            h = x + h
            y = torch.relu(h * (h.square().mean(-1, keepdim=True) + norm.eps).rsqrt() * p["norms.%d.weights" % b])
            x = A @ (y @ p["convs.%d.weights" % b])
        return x, p


def test_a_deep_network_of_all_of_them():
    dev = torch.device("cuda:0")
    g, A = _graph(dev)
    operators = {d: _operator(g, dev, False) for d in (48, 7)}
    torch.manual_seed(5)
    net = _Deep(300, 48, 7, 4, False).to(dev)
    ids = torch.randint(0, 300, (g.n_rows,), device=dev)
    label = torch.randint(0, 7, (g.n_rows,), device=dev)
    grads = []
    for eight in (False, True):
        net.eight, net.trace = eight, []
        net.zero_grad()
        out = net(ids, operators)
        torch.nn.functional.cross_entropy(out, label).backward()
        grads.append({k: v.grad.clone() for k, v in net.named_parameters()})
        if not eight:
            first = out.detach()
    assert torch.equal(first, out.detach())
    ref, p = net.formula(ids, A)
    torch.nn.functional.cross_entropy(ref, label).backward()
    _close(first, ref.detach())
    for k in grads[0]:
        _close(grads[0][k], p[k].grad)
        if k.startswith("convs"):
            (kept,), x = net.trace[int(k.split(".")[1])]
            bound = _step(kept).t() @ (A @ x.grad.double()).abs()
            off = (grads[1][k].double() - p[k].grad).abs()
            # (a hundredth for the roundings in the factor A G, and what 32 bits leave where all errors are tiny)
            assert (off <= 1.01 * bound + 1e-5 * p[k].grad.abs().max()).all()
            assert not torch.equal(grads[1][k], grads[0][k])
        else:
            assert torch.equal(grads[1][k], grads[0][k])


def test_the_deep_network_keeps_less():
    """What lives between forward and backward: per block h in 32 bits and y in 8, against both in 32."""
    dev = torch.device("cuda:0")
    from paramspmm_ae_b200 import synth
    g = synth.powerlaw_graph(40000, 100000, seed=3).to(dev)
    operators = {128: _operator(g, dev, False)}
    torch.manual_seed(6)
    net = _Deep(40000, 128, 128, 6, False).to(dev)
    ids = torch.arange(40000, device=dev)
    took = []
    for eight in (False, True):
        net.eight = eight
        net.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = net(ids, operators)
        took.append(torch.cuda.memory_allocated() - before)
        out.sum().backward()
        del out
    dense = 40000 * 128 * 4
    # 6 y's: 32 bits against 8 and a 32nd for the scales
    assert took[0] - took[1] >= 6 * dense * (3 / 4 - 1 / 32) * 0.95


def test_a_training_step_of_the_deep_network_is_captured():
    dev = torch.device("cuda:0")
    g, _ = _graph(dev)
    operators = {d: _operator(g, dev, False) for d in (32, 8)}
    torch.manual_seed(7)
    net = _Deep(g.n_rows, 32, 8, 3, True).to(dev)
    ids = torch.arange(g.n_rows, device=dev)
    label = torch.randint(0, 8, (g.n_rows,), device=dev)

    def step():
        net.zero_grad(set_to_none=True)
        loss = torch.nn.functional.cross_entropy(net(ids, operators), label)
        loss.backward()
        return loss

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step().detach_()
    torch.cuda.current_stream().wait_stream(s)
    net.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step().detach()
    grads = {k: v.grad for k, v in net.named_parameters()}
    with torch.no_grad():
        for p in net.parameters():
            p.mul_(1.1)
    graph.replay()
    torch.cuda.synchronize()
    got = {k: v.clone() for k, v in grads.items()}
    value = loss.clone()
    del graph
    want = step()
    assert torch.equal(value, want.detach())
    for k, v in net.named_parameters():
        assert torch.equal(got[k], v.grad), k


def _layouts(t):
    """The same values stored by rows, by columns and as rows of a wider array."""
    wide = torch.zeros(t.shape[0], t.shape[1] + 5, device=t.device)
    wide[:, 3:3 + t.shape[1]] = t
    return [t, t.t().contiguous().t(), wide[:, 3:3 + t.shape[1]]]


@pytest.mark.parametrize("kind", ["gcn", "gcn narrow first", "gin", "agnn fused", "agnn recomputed", "agnn composed"])
def test_gradients_and_inputs_of_any_strides_with_8_bits(kind):
    """A layer that keeps its input in 8 bits takes what it takes without: the gradient of a sum (strides of 0), of a transposed view,
    and inputs that are stored by columns, with equal results."""
    from paramspmm_ae_b200 import gnn_conv
    dev = torch.device("cuda:0")
    g, _ = _graph(dev)
    P = _operator(g, dev, False)
    torch.manual_seed(6)
    fin, fout = (12, 32) if kind == "gcn narrow first" else (36, 32)
    layer = (gnn_conv.GINConv if kind == "gin" else gnn_conv.AGNNConv if "agnn" in kind else gnn_conv.GCNConv)(fin, fout).to(dev)
    layer.keep_scores, layer.keep_input_8bit = kind != "agnn recomputed", True
    args = (P.colIdx.unsqueeze(-1),) if "agnn" in kind else ()
    X, G = torch.randn(g.n_rows, fin, device=dev), torch.randn(g.n_rows, fout, device=dev)
    fused, gnn_conv.FUSE_AGNN_TRAINING = gnn_conv.FUSE_AGNN_TRAINING, kind != "agnn composed"
    old, gnn_conv.REORDER_NARROW_FIRST = gnn_conv.REORDER_NARROW_FIRST, kind == "gcn narrow first"

    def step(x, back):
        layer.zero_grad()
        x = x.detach().requires_grad_(True)
        out = layer(x, {fin: P, fout: P}, *args)
        back(out)
        return out.detach(), x.grad, layer.weights.grad

    try:
        want = step(X, lambda out: out.backward(G))
        for x in _layouts(X)[1:] if kind != "gin" else ():  # (the aggregation of GIN itself takes contiguous rows alone)
            for a, b in zip(step(x, lambda out: out.backward(G)), want):
                _close(a, b)
        for grad in _layouts(G)[1:]:
            for a, b in zip(step(X, lambda out: out.backward(grad)), want):
                _close(a, b)
        ones = step(X, lambda out: out.backward(torch.ones_like(G)))
        for a, b in zip(step(X, lambda out: out.sum().backward()), ones):
            _close(a, b)
    finally:
        gnn_conv.FUSE_AGNN_TRAINING, gnn_conv.REORDER_NARROW_FIRST = fused, old


@pytest.mark.parametrize("which", ["embedding", "rows8_mm", "dense"])
def test_status_words_wait_for_every_stream(which):
    """A status read while the call that sets it waits its turn on a side stream, in a process of its own (the words stay set)."""
    import subprocess
    import sys
    code = """
import ctypes, sys, torch
from paramspmm_ae_b200 import _lib, feature_ops as fo, ops
which = sys.argv[1]
lib, side = _lib.lib(), torch.cuda.Stream()
status = {"embedding": fo.embedding_status, "rows8_mm": fo.rows8_mm_status, "dense": ops.dense_status}[which]
table, ids = torch.ones(4, 8, device="cuda"), torch.tensor([0, 4], device="cuda")
q, s, G = torch.ones(400, 64, dtype=torch.int8, device="cuda"), torch.ones(400, 1, device="cuda"), torch.ones(400, 32, device="cuda")
A, C, scratch = torch.ones(400, 64, device="cuda"), torch.zeros(64, 32, device="cuda"), torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
def stalled(of):
    at = torch.cuda.current_stream().cuda_stream
    if of == "rows8_mm":
        _lib.check(lib.pspmm_rows8_mm_t_stalled(q.data_ptr(), 64, s.data_ptr(), 400, 64, G.data_ptr(), 0, 32, 32, C.data_ptr(), 32,
                                                scratch.data_ptr(), 1 << 22, at))
    else:
        _lib.check(lib.pspmm_dense_mm_stalled(1, 0, 64, 32, 400, A.data_ptr(), 64, G.data_ptr(), 32, C.data_ptr(), 32,
                                              scratch.data_ptr(), 1 << 22, at))
fo.embedding(ids[:1], table)
fo.rows8_mm_t(fo.Rows8(q, s, 64), G)
ops.dense_mm(A, G, transA=True)
torch.cuda.synchronize()
assert status() == 0
with torch.cuda.stream(side):
    torch.cuda._sleep(100000000)  # some 50 ms
    fo.embedding(ids, table) if which == "embedding" else stalled(which)
assert status() == 1
print("told")
"""
    p = subprocess.run([sys.executable, "-c", code, which], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "told" in p.stdout, p.stderr


def test_node_embedding_and_norm_take_any_strides():
    """Ids that are a column of a batch, activations that are stored by columns or that repeat one row: equal to their copies."""
    from paramspmm_ae_b200 import gnn_conv
    torch.manual_seed(7)
    layer = gnn_conv.NodeEmbedding(50, 24).cuda()
    batch = torch.randint(0, 50, (40, 6), device="cuda")
    for ids in (batch[:, 2], batch.t(), batch[::3, 1::2], batch[0, 0], batch[:1].expand(5, 6)):
        got = []
        for i in (ids, ids.clone(memory_format=torch.contiguous_format)):
            layer.zero_grad()
            out = layer(i)
            out.square().sum().backward()
            got.append((out.detach(), layer.weights.grad))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][0], layer.weights[ids])
    norm = gnn_conv.RMSNorm(70).cuda()
    norm.weights.data.uniform_(0.5, 1.5)
    base, res = torch.randn(70, 33, device="cuda"), torch.randn(1, 70, device="cuda")
    wide = torch.randn(4, 33, 75, device="cuda")
    for x, r in ((base.t(), None), (base.t(), res.expand(33, 70)), (res.expand(33, 70), base.t()), (wide[:, :, 2:72], None),
                 (wide[1, :, 2:72], base.t())):
        got = []
        for copy in (False, True):
            norm.zero_grad()
            a, b = ((t if t is None else (t.clone(memory_format=torch.contiguous_format) if copy else t.detach()).requires_grad_(True)) for t in (x, r))
            y, h, kept = norm(a, b, eight_bit=True)
            (y * h).square().sum().backward()
            got.append([y.detach(), h.detach(), kept.q, a.grad, norm.weights.grad] + ([] if b is None else [b.grad]))
        _close(got[0][0], got[1][0])
        assert torch.equal(got[0][1], got[1][1]) and (got[0][2] != got[1][2]).sum() == 0
        for p, q in zip(got[0][3:], got[1][3:]):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-4 * float(q.abs().max()))


def test_offsets_beyond_32_bits():
    """Arrays of more than 2^31 values (4.4 GB each): the rows at their ends are what they are in arrays of their own."""
    from paramspmm_ae_b200 import feature_ops as fo
    n, dim, m = 16600000, 130, 999
    assert n * dim > 2 ** 31 and (n - m) * dim > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(8)
    end = torch.randint(-4, 5, (m, dim), generator=g, device="cuda").bfloat16()
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda")
    x[-m:] = end
    w = torch.rand(dim, generator=g, device="cuda").bfloat16()
    alone, whole = fo.rms_norm(end, w, end, eight_bit=True), fo.rms_norm(x, w, x, eight_bit=True)
    for a, b in zip(alone[:3] + (alone[3].q, alone[3].scales), whole[:3] + (whole[3].q, whole[3].scales)):
        assert torch.equal(a, b[-m:]) and b.shape[0] == n
    assert torch.equal(alone[3].dequantize(torch.bfloat16), whole[3].dequantize(torch.bfloat16)[-m:])
    a, b = (fo.rms_norm_backward(t, s[1], s[2], w, dh=t) for t, s in ((end, alone), (x, whole)))
    assert torch.equal(a[0], b[0][-m:])
    torch.testing.assert_close(b[1].float(), a[1].float(), rtol=2 ** -7, atol=1e-2)  # (rows of zeros add none; other partial sums)
    del whole, b
    held, kept = fo.quantize_rows(end), fo.quantize_rows(x)
    assert torch.equal(held.q, kept.q[-m:]) and torch.equal(held.scales, kept.scales[-m:])
    kept = fo.Rows8(kept.q, kept.scales.fill_(0.5), dim)  # (products of whole numbers and halves: exact)
    held = fo.Rows8(held.q, held.scales.fill_(0.5), dim)
    want = (held.q[:, :dim].double() * 0.5).t() @ end.double()
    assert torch.equal(fo.rows8_mm_t(held, end).double(), want) and torch.equal(fo.rows8_mm_t(kept, x).double(), want)
    wide = torch.zeros(n, 132, dtype=torch.bfloat16, device="cuda")  # rows that begin off 16 bytes, and no room needed for a copy of them
    wide[-m:, 1:131] = end
    assert torch.equal(fo.rows8_mm_t(kept, wide[:, 1:131]).double(), want)
    del kept, wide
    ids = torch.randperm(m, generator=g, device="cuda")
    assert torch.equal(fo.embedding(ids + (n - m), x), end[ids])
    grad = fo.embedding_grad(ids + (n - m), end, n)
    assert torch.equal(grad[-m:][ids], end) and not grad[:-m].any()
    del grad
    ids = torch.cat([torch.full((n - m,), 3, device="cuda"), ids + 10])
    table = torch.randn(m + 10, dim, generator=g, device="cuda").bfloat16()
    assert torch.equal(fo.embedding(ids, table)[-m:], table[ids[-m:]])
    grad = fo.embedding_grad(ids, x, m + 10)
    assert torch.equal(grad[ids[-m:]], end) and not grad[:10].any()
