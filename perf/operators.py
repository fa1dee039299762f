"""The operators around the graph layers, as cases that can be timed and compared.

``kind`` names the operator:

* ``embedding``  rows of a table looked up by id and scaled, and the table's gradient
* ``norm``       root-mean-square norm of ``x + residual`` (and relu): the forward, with an output in 8 bits where ``eight``
                 says so, or the forward and the backward of a training step
* ``keep``       an activation held in 8 bits (a scale per row and block of 128 columns) and brought back
* ``gradient``   the weight gradient of a layer from its input as held in 8 bits

With ``own`` the package's kernels run, without it the same formulas in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128           # columns that share a scale
TINY = 2.0 ** -119    # a block whose largest magnitude is below this has no normal scale: it is held as zeros
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # A sampled batch of nodes of a citation-size graph: launches are what counts.
        dict(name="embedding small batch", kind="embedding", type="fp32", ids="int64", V=19717, n=512, dim=16, skew=1, pad=False),
        # Learned features of a product-graph's nodes, looked up for the neighbourhood of a batch, hubs more often.
        dict(name="embedding neighbourhood", kind="embedding", type="fp32", ids="int32", V=2449029, n=1000003, dim=64, skew=2,
             pad=False),
        # Tokens of a batch of sequences, padding among them: few rows of the table take most of the gradient.
        dict(name="embedding tokens", kind="embedding", type="bf16", ids="int64", V=50021, n=32768, dim=1024, skew=4, pad=True),
        # A class-count width, which leaves rows that admit narrow loads only.
        dict(name="embedding odd width", kind="embedding", type="fp32", ids="int64", V=100003, n=200003, dim=47, skew=1, pad=False),
        # One row of a server's step, for a consumer that reads 8 bits.
        dict(name="norm one row", kind="norm", type="bf16", n=1, dim=4096, step=False, relu=False, eight=True),
        # A hidden layer of a training step over a citation graph of 169 K nodes.
        dict(name="norm step fp32", kind="norm", type="fp32", n=169343, dim=128, step=True, relu=True, eight=False),
        # The same on wide rows in 16 bits.
        dict(name="norm step bf16", kind="norm", type="bf16", n=16384, dim=4096, step=True, relu=False, eight=False),
        # A feature width that is no multiple of the 8-bit form's blocks; the next layer keeps the 8 bits.
        dict(name="norm eight bits", kind="norm", type="fp32", n=89251, dim=100, step=False, relu=True, eight=True),
        # Class scores at an odd width, held until the backward.
        dict(name="keep odd width", kind="keep", type="fp32", n=89251, dim=47),
        # Wide activations in 16 bits.
        dict(name="keep wide", kind="keep", type="bf16", n=32768, dim=4096),
        # First layer of a small citation graph: 500 features, 16 hidden columns.
        dict(name="gradient small", kind="gradient", type="fp32", n=19717, dim=500, cols=16),
        # Hidden layer of the full-size training step.
        dict(name="gradient large", kind="gradient", type="fp32", n=2449029, dim=256, cols=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 8, some of 4, some odd."""
    w, r = _log(rng, lo, hi), rng.random()
    if r < 0.6:
        return max(8, w // 8 * 8)
    return max(4, w // 4 * 4) if r < 0.75 else w | 1


def draw(rng):
    kind = rng.choice(["embedding", "norm", "keep", "gradient"])
    case = dict(kind=kind, type=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    if kind == "embedding":
        case.update(ids=rng.choice(["int32", "int64"]), dim=_width(rng, 16, 1024), skew=rng.choice([1, 2, 4]),
                    pad=rng.random() < 0.3)
        most = 400000000 // case["dim"]  # values of the table, and of the rows looked up
        case.update(V=_log(rng, 1000, min(2500000, most)), n=_log(rng, 64, min(2000000, most)))
    elif kind == "norm":
        case.update(dim=_width(rng, 16, 8192), step=rng.random() < 0.5, relu=rng.random() < 0.5)
        case.update(n=_log(rng, 1, min(1000000, 200000000 // case["dim"])), eight=not case["step"] and rng.random() < 0.7)
    elif kind == "keep":
        case.update(dim=_width(rng, 16, 8192))
        case.update(n=_log(rng, 1, min(2400000, 400000000 // case["dim"])))
    else:
        case.update(dim=_width(rng, 16, 2048), cols=_width(rng, 8, 1024))
        most = min(400000000 // max(case["dim"], case["cols"]), 150000000000 // (case["dim"] * case["cols"]))
        case.update(n=_log(rng, 256, min(2400000, most)))
    return case


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, n, dim = TYPES[case["type"]], case["n"], case["dim"]
    s = dict(kind=case["kind"], type=t)
    if case["kind"] == "embedding":
        V = case["V"]
        # ids of a power law (skew 1: uniform), scattered over the table
        ids = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** case["skew"] * V).long().clamp_(max=V - 1)
        ids = torch.randperm(V, generator=g, device="cuda")[ids]
        if case["pad"]:
            ids[torch.rand(n, generator=g, device="cuda") < 0.1] = 0
        s.update(ids=ids.to(torch.int32) if case["ids"] == "int32" else ids, table=(_normal(g, V, dim) * 0.02).to(t),
                 G=_normal(g, n, dim).mul_(1e-2).to(t), scale=math.sqrt(dim), pad=0 if case["pad"] else None)
    elif case["kind"] == "norm":
        spread = torch.exp(_normal(g, n, 1))  # rows of nodes with many neighbours are larger
        s.update(x=_normal(g, n, dim).mul_(spread).to(t), r=_normal(g, n, dim).to(t), w=(1 + 0.1 * _normal(g, dim)).to(t),
                 step=case["step"], relu=case["relu"], eight=case["eight"], eps=1e-6)
        if case["step"]:
            s.update(dy=_normal(g, n, dim).mul_(1e-2).to(t), dh=_normal(g, n, dim).mul_(1e-2).to(t))
    elif case["kind"] == "keep":
        s.update(x=torch.relu(_normal(g, n, dim).mul_(torch.exp(_normal(g, n, 1)))).to(t))
    else:
        # what the layer's forward left: whole numbers in rows padded to 16 bytes, and the scales
        cols, pitch, blocks = case["cols"], (dim + 15) // 16 * 16, (dim + BLOCK - 1) // BLOCK
        q = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")
        q[:, :dim] = (_normal(g, n, dim) * 40).clamp_(0, 127).to(torch.int8)
        s.update(q=q, dim=dim, scales=torch.exp(_normal(g, n, blocks)).mul_(0.01), G=_normal(g, n, cols).mul_(1e-3).to(t))
    return s


def _to_eight(y):
    """(whole numbers, scales) of rows in 32 or 64 bits.  The products with the reciprocal scale are formed in 64 bits: what they
    are rounded to turns on values next to a half."""
    n, dim = y.shape
    blocks = (dim + BLOCK - 1) // BLOCK
    b = torch.nn.functional.pad(y, (0, blocks * BLOCK - dim)).view(n, blocks, BLOCK)
    a = b.abs().amax(2).float()
    held, top = a >= TINY, torch.full_like(a, 127)  # (by a number, a quotient would be a product with the rounded reciprocal)
    scales = torch.where(held, a / top, 0.0)
    up = torch.where(held, top / a, 0.0)
    return torch.round(b.double() * up.double().unsqueeze(2)), scales


def _from_eight(q, scales, dim):
    return (q.float() * scales.unsqueeze(2)).flatten(1)[:, :dim]


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from paramspmm_ae_b200 import feature_ops as fo
    if s["kind"] == "embedding":
        out = fo.embedding(s["ids"], s["table"], s["scale"])
        return dict(out=out, grad=fo.embedding_grad(s["ids"], s["G"], s["table"].shape[0], s["scale"], padding_idx=s["pad"]))
    if s["kind"] == "norm":
        y, h, rstd, kept = fo.rms_norm(s["x"], s["w"], s["r"], eps=s["eps"], relu=s["relu"], eight_bit=s["eight"])
        if s["step"]:
            dx, dw = fo.rms_norm_backward(s["dy"], h, rstd, s["w"], dh=s["dh"], relu=s["relu"])
            return dict(y=y, h=h, dx=dx, dw=dw)
        return dict(y=y, h=h, kept=kept.dequantize()) if s["eight"] else dict(y=y, h=h)
    if s["kind"] == "keep":
        return fo.quantize_rows(s["x"]).dequantize(s["type"])
    return fo.rows8_mm_t(fo.Rows8(s["q"], s["scales"], s["dim"]), s["G"])


def _run_plain(s):
    t = s["type"]
    if s["kind"] == "embedding":
        ids, table, G = s["ids"].long(), s["table"], s["G"].float()
        out = (table[ids].float() * s["scale"]).to(t)
        if s["pad"] is not None:
            G = G * (ids != s["pad"]).unsqueeze(1)
        grad = torch.zeros(table.shape, dtype=torch.float32, device=ids.device).index_add_(0, ids, G)
        return dict(out=out, grad=(grad * s["scale"]).to(t))
    if s["kind"] == "norm":
        wide = torch.float64 if s["eight"] else torch.float32  # the 8-bit form's values lie next to halves
        h, w = s["x"].to(wide) + s["r"].to(wide), s["w"].to(wide)
        rstd = (1 / torch.sqrt(h.double().square().mean(1, keepdim=True) + s["eps"])).to(wide)
        y = h * rstd * w
        if s["relu"]:
            y = torch.relu(y)
        out = dict(y=y.to(t), h=h.to(t))
        if s["eight"]:
            out["kept"] = _from_eight(*_to_eight(y), y.shape[1])
        if s["step"]:
            h, dy = out["h"].float(), s["dy"].float()  # the sum as it was kept
            n = h * rstd
            if s["relu"]:
                dy = torch.where(n * w > 0, dy, 0.0)
            g = dy * w
            out["dx"] = ((g - n * (g * n).mean(1, keepdim=True)) * rstd + s["dh"].float()).to(t)
            out["dw"] = (dy * n).sum(0).to(t)
        return out
    if s["kind"] == "keep":
        x = s["x"].float()
        return _from_eight(*_to_eight(x), x.shape[1]).to(t)
    n, dim = s["q"].shape[0], s["dim"]
    h = s["q"][:, :dim].float() * s["scales"].repeat_interleave(BLOCK, 1)[:, :dim]
    return torch.mm(h.t(), s["G"].float())


def _distinct(V, n, skew):
    """Rows of the table that n ids of the case's distribution are expected to touch."""
    edges = (np.arange(V + 1) / V) ** (1 / skew)
    return float((-np.expm1(n * np.log1p(-np.minimum(np.diff(edges), 1 - 1e-12)))).sum())


def work(case):
    n, dim, b = case["n"], case["dim"], BYTES[case["type"]]
    blocks = (dim + BLOCK - 1) // BLOCK
    held = n * (dim + 4 * blocks)  # a byte per value and the scales
    if case["kind"] == "embedding":
        rows = _distinct(case["V"], n, case["skew"])
        ids = n * (4 if case["ids"] == "int32" else 8)
        return {"bytes": int(ids + (rows + 2 * n + case["V"]) * dim * b), "flops": 2 * n * dim}
    if case["kind"] == "norm":
        # x, residual, h and y; the step reads what comes back and writes what goes on
        size = n * dim * b
        more = held + 4 * n * dim if case["eight"] else 0
        return {"bytes": (7 if case["step"] else 4) * size + more, "flops": (16 if case["step"] else 5) * n * dim}
    if case["kind"] == "keep":
        return {"bytes": 2 * n * dim * b + 2 * held, "flops": 4 * n * dim}
    return {"bytes": held + n * case["cols"] * b + 4 * dim * case["cols"], "flops": 2 * n * dim * case["cols"]}


def _exact_eight(y):
    """What the 8-bit form of 64-bit rows stands for: block after block, largest magnitude and both factors held in 32 bits."""
    out = torch.empty_like(y)
    for c in range(0, y.shape[1], BLOCK):
        b = y[:, c:c + BLOCK]
        a = b.abs().max(1, keepdim=True).values.float().double()
        up, scale = (127 / a).float().double(), (a / 127).float().double()
        out[:, c:c + BLOCK] = torch.where(a >= TINY, torch.round(b * up) * scale, 0.0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embedding":
        ids, V = s["ids"].long(), case["V"]
        if V * case["dim"] + 2 * case["n"] * case["dim"] > 2000000000:
            return None
        grad = torch.zeros(V, case["dim"], dtype=torch.float64, device="cuda")
        some = ids != s["pad"] if s["pad"] is not None else torch.ones_like(ids, dtype=torch.bool)
        grad.index_put_((ids[some],), s["G"].double()[some], accumulate=True)
        return dict(out=s["table"].double().mul_(s["scale"])[ids], grad=grad * s["scale"])
    if case["kind"] == "norm":
        h = s["x"].double() + s["r"].double()
        w, d = s["w"].double(), case["dim"]
        rstd = torch.rsqrt((h * h).sum(1, keepdim=True) / d + s["eps"])
        y = h * rstd * w
        if s["relu"]:
            y = y.clamp(min=0)
        out = dict(y=y, h=h)
        if s["eight"]:
            out["kept"] = _exact_eight(y)
        if s["step"]:
            # by the chain rule over rstd, at the sum as it is kept
            hk, dy = h.to(s["type"]).double(), s["dy"].double()
            if s["relu"]:
                dy = dy * (hk * w > 0)
            through = (dy * w * hk).sum(1, keepdim=True)
            out["dx"] = s["dh"].double() + dy * w * rstd - hk * rstd ** 3 * through / d
            out["dw"] = torch.einsum("nd,nd->d", dy, hk * rstd)
        return out
    if case["kind"] == "keep":
        return _exact_eight(s["x"].double())
    out = torch.zeros(case["dim"], case["cols"], dtype=torch.float64, device="cuda")
    for c in range(0, case["dim"], BLOCK):
        e = min(c + BLOCK, case["dim"])
        for i in range(0, case["n"], 1 << 19):
            G = s["G"][i:i + (1 << 19)].double() * s["scales"][i:i + (1 << 19), c // BLOCK, None].double()
            out[c:e] += s["q"][i:i + (1 << 19), c:e].double().t() @ G
    return out
