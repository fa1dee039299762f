"""GCN / GIN / AGNN layers over the PCSR operators: mirror of the reference's ``gnn_conv.py``.

Same module and autograd-function names, constructor arguments and forward signatures
(gnn_conv.py:13-238 of the reference).  The layer semantics are the reference's:

* GCN   forward  A (H W); backward AG = A G (A itself: the normalised adjacency is symmetric),
        dH = AG W^T, dW = H^T AG.  With REORDER_NARROW_FIRST (off by default) layers that widen
        their input aggregate first instead, (A H) W.
* GIN   forward  (A X) W; backward dW = (A X)^T G, dX = A (G W^T).
* AGNN  forward  X' = X W, e = SDDMM(X', X') * beta, out = SpMM(e, X'); no edge softmax and no
        row normalisation (the reference has none); the gradient w.r.t. beta follows the
        reference's expression (gnn_conv.py:164-172).

Beside them stand two layers that the reference does not have, ``NodeEmbedding`` (learned features of graphs that come without)
and ``RMSNorm`` (the residual stream of deep networks), and a layer can keep its input for the backward in 8 bits
(``keep_input_8bit``, or the 8-bit form that an ``RMSNorm`` left, as ``kept``).
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import feature_ops, ops

n_heads = 1


# When a GCN layer widens its input (fan-in < fan-out) the aggregation is cheaper before the
# projection: A (H W) = (A H) W, and the SpMM then runs at the narrower width.  The reference always
# aggregates after the projection (SpCONV/SpCONV.h:43-72), and so does this module by default, so
# that layer outputs and gradients are the reference's up to the summation order inside the SpMM.
# Setting this to True is an opt-in: results then differ from the reference's by fp32
# re-association of the two products (both orders are tested against fp64 algebra), the backward
# keeps A H instead of H, and the operator is looked up under the input width when the caller's
# dictionary has one for it.
REORDER_NARROW_FIRST = False


def _aggregate(P, X):
    out = P.GIN_spmm(X.contiguous())
    return out[: X.shape[0]] if out.shape[0] != X.shape[0] else out  # block layouts pad the row count


def _save(ctx, kept, *others):
    """What the backward needs: the factor of the weight gradient, as a tensor or in 8 bits, and ``others``."""
    ctx.kept_dim = None if isinstance(kept, torch.Tensor) else kept.dim
    ctx.save_for_backward(*((kept,) if ctx.kept_dim is None else (kept.q, kept.scales)), *others)


def _saved(ctx):
    t = ctx.saved_tensors
    return t if ctx.kept_dim is None else (feature_ops.Rows8(t[0], t[1], ctx.kept_dim), *t[2:])


def _held(X, eight):
    """``X`` as the backward is to have it: itself, or in 8 bits (``eight``: True, or those bits).  ``X`` has any strides."""
    return X if eight is None else feature_ops.quantize_rows(ops._as_rows(X)) if eight is True else eight


class GCNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, H, weight, ParamSpMM, eight=None):
        ctx.ParamSpMM = ParamSpMM
        ctx.narrow_first = bool(REORDER_NARROW_FIRST and weight.shape[0] < weight.shape[1])
        if ctx.narrow_first:
            AH = _aggregate(ParamSpMM, H)
            _save(ctx, _held(AH, None if eight is None else True), weight)
            return torch.mm(AH, weight)
        _save(ctx, _held(H, eight), weight)
        return ParamSpMM.forward(H, weight)

    @staticmethod
    def backward(ctx, d_output):
        P = ctx.ParamSpMM
        d_output = d_output.contiguous()
        if ctx.narrow_first:
            # dW = (A H)^T G with A H kept from the forward; dH = A (G W^T) (A is symmetric),
            # skipped when the layer input needs no gradient (the first layer).
            AH, weight = _saved(ctx)
            d_weight = ops._weight_grad(AH, d_output)
            d_input = _aggregate(P, ops.dense_mm(d_output, weight, transB=True)) if ctx.needs_input_grad[0] else None
            return d_input, d_weight, None, None
        H, weight = _saved(ctx)
        if ctx.needs_input_grad[0]:
            d_input, d_weight = P.backward(d_output, H, weight)
        else:  # the first layer: dH = AG W^T is not formed (the reference forms and drops it)
            d_input, d_weight = P.backward(d_output, H, weight, input_grad=False)
        return d_input, d_weight, None, None


class GINFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, weight, ParamSpMM, eight=None):
        X_agg = ParamSpMM.GIN_spmm(X)
        _save(ctx, _held(X_agg, eight), weight)
        ctx.ParamSpMM = ParamSpMM
        return torch.mm(X_agg, weight)

    @staticmethod
    def backward(ctx, d_output):
        X_agg, weight = _saved(ctx)
        d_weight = ops._weight_grad(X_agg, d_output)
        d_input = ctx.ParamSpMM.GIN_spmm(ops.dense_mm(d_output, weight, transB=True).contiguous())
        return d_input, d_weight, None, None


# Under torch.no_grad() an AGNN layer on a plain or split CSR operator runs as the fused kernel
# (SDDMM -> scale -> SpMM in one pass).  Set to False to always use the three-kernel composition.
FUSE_AGNN_INFERENCE = True

# With gradients enabled the same layers run AGNNFusedFunction: the forward is the fused kernel, which leaves
# the edge scores for the backward (4 bytes per edge; the reference's composition writes the attention values in
# the forward and the score gradient in the backward, gnn_conv.py:130-180).  Outputs and gradients are the
# reference's up to fp32 summation order.
# Set to False to train through the three-kernel composition (AGNNFunction).  ``AGNNConv.keep_scores`` chooses per layer
# whether the scores are kept.
FUSE_AGNN_TRAINING = True
_SCORES_UNASKED = 16 << 20  # bytes up to which scores are kept without a look at the free memory (12 us of host time)


def _room(device):
    """Bytes of a device that torch has not handed out, within the limit of the process.  (The driver's own figure for free memory
    takes 0.2 ms, at times several.)"""
    try:
        limit = torch.cuda.get_per_process_memory_fraction(device) * torch.cuda.get_device_properties(device).total_memory
        return limit - torch.cuda.memory_stats_as_nested_dict(device)["allocated_bytes"]["all"]["current"]
    except (RuntimeError, KeyError):  # an allocator of the host's, which keeps no figures: its allocation tells
        return float("inf")


def _keeps_scores(nnz, Xp):
    """Whether the scores of ``nnz`` edges may take memory until the backward.  They stand in for the projected features, up to
    whose size a step takes no more than without; beyond it up to a 32nd of what is free, so that the layers behind this one find
    the room they found without (a second gather per edge instead: 115 M edges, 64 columns, a step of 4.1 ms becomes 6.1)."""
    nbytes = 4 * nnz
    return nbytes <= _SCORES_UNASKED or nbytes <= Xp.numel() * Xp.element_size() or 32 * nbytes <= _room(Xp.device)


def _beta(attention_w):
    """The attention weight as the one float on the device that the fused passes read."""
    return attention_w.detach().reshape(1).to(torch.float32)


def _can_fuse(P, dim):
    return getattr(P, "vec_size", 1) == 1 and dim % 4 == 0 and dim <= 256


def _is_operator_colidx(P, colIdx):
    """The fused backward weights edges by the operator's own column ids; callers pass them as an
    [nnz, 1] column (GNN.py:224-225).  Compared once per content of a tensor, not per step: the operator holds
    the last one it compared, so that its memory is not another tensor's meanwhile, and its version."""
    own = P.colIdx
    if colIdx.is_inference() or own.is_inference():  # (these keep no version)
        return _same_entries(colIdx, own)
    seen = P.__dict__.get("_colidx_checked")
    if seen is None or own is not seen[1] or (colIdx._version, own._version) != seen[2] or (
            colIdx is not seen[0] and (colIdx.data_ptr() != seen[0].data_ptr() or colIdx.shape != seen[0].shape
                                       or colIdx.stride() != seen[0].stride() or colIdx.dtype != seen[0].dtype)):
        seen = P._colidx_checked = (colIdx, own, (colIdx._version, own._version), _same_entries(colIdx, own))
    return seen[3]


def _same_entries(colIdx, own):
    flat = colIdx.reshape(-1)
    return bool(flat.shape == own.shape and flat.dtype == own.dtype and torch.equal(flat, own))


class AGNNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, weights, attention_w, ParamSpMM, colIdx, eight=None):
        X_prime = ops.dense_mm(X, weights)
        edge = ParamSpMM.AGNN_sddmm(X_prime)
        # [n_edges] for CSR, [n_blocks, V] for block layouts; one attention head
        edge_attentions = (edge * attention_w.reshape(())).contiguous()
        out = ParamSpMM.AGNN_spmm(edge_attentions, X_prime)
        _save(ctx, _held(X, eight), weights, edge_attentions)
        ctx.colIdx, ctx.ParamSpMM = colIdx, ParamSpMM
        return out

    @staticmethod
    def backward(ctx, d_output):
        P = ctx.ParamSpMM
        X, weights, edge_attentions = _saved(ctx)
        d_output = d_output.contiguous()
        d_prime = P.AGNN_spmm(edge_attentions, d_output)
        d_input = ops.dense_mm(d_prime, weights, transB=True)
        d_weights = ops._weight_grad(X, d_prime)
        d_att = P.AGNN_sddmm(d_output)
        if d_att.dim() != 1:
            d_att = d_att.reshape(-1)[P.mask]  # back to CSR entry order
        d_attention_w = torch.mm(d_att[None, :].expand(n_heads, -1), ctx.colIdx.float()).transpose(0, 1)
        return d_input, d_weights, d_attention_w, None, None, None


class AGNNFusedFunction(torch.autograd.Function):
    """AGNN layer on a CSR / split-CSR operator in one pass over the pattern per direction.

    forward   X' = X W,  out_i = sum_j beta <X'_i, X'_j> X'_j     (one fused pass, which leaves the scores)
    backward  D_i = sum_j beta <X'_i, X'_j> G_j           (gradient rows gathered, scores read; with ``keep_scores=False``, or
              little room for them, the rows of X' are kept and gathered again and the scores recomputed)
              dX = D W^T,  dW = X^T D                                      (gnn_conv.py:157-160)
              d_beta = sum over edges of <G_i, G_j> * colIdx[e]              (gnn_conv.py:163-172: the
              reference multiplies the score gradient by the column-index column it is handed), summed
              in the same pass while the gradient row is in registers.
    The attention weight stays on the device (reading it back made every forward wait for the GPU).
    Like the reference's backward, the edge values are treated as constants with respect to X'."""

    @staticmethod
    def forward(ctx, X, weights, attention_w, P, colIdx, keep_scores=True, eight=None):
        Xp = ops.dense_mm(X, weights)
        beta, scores = _beta(attention_w), None
        if keep_scores and _keeps_scores(P.colIdx.shape[0], Xp):
            try:
                scores = torch.empty(P.colIdx.shape[0], dtype=torch.float32, device=Xp.device)
            except torch.cuda.OutOfMemoryError:
                pass
        if scores is None:
            beta = beta.clone()  # (the backward uses the value of this forward)
        out = ops.agnn_layer_forward(Xp, P.rowPtr, P.colIdx, beta, P.target_row, scores)
        _save(ctx, _held(X, eight), weights, *((Xp, beta) if scores is None else (scores,)))
        ctx.P = P
        return out

    @staticmethod
    def backward(ctx, d_output):
        X, weights, *rest = _saved(ctx)
        Xp, beta, scores = (*rest, None) if len(rest) == 2 else (None, None, *rest)
        P = ctx.P
        D, d_att = ops.agnn_layer_backward(Xp, d_output.contiguous(), P.rowPtr, P.colIdx, beta, P.target_row,
                                           beta_grad=ctx.needs_input_grad[2], scores=scores)
        d_input = ops.dense_mm(D, weights, transB=True) if ctx.needs_input_grad[0] else None
        d_weights = ops._weight_grad(X, D) if ctx.needs_input_grad[1] else None
        return d_input, d_weights, d_att, None, None, None, None


class EmbeddingFunction(torch.autograd.Function):
    """scale * table[ids]; the table's gradient is dense, sums over equal ids in the order of their positions."""

    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, padding_idx)
        return feature_ops.embedding(ids, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, feature_ops.embedding_grad(ids, grad.contiguous(), *ctx.args), None, None


class RMSNormFunction(torch.autograd.Function):
    """(y, h, q, scales) of ``feature_ops.rms_norm``; h is None without a residual, q and scales without ``eight_bit``.  Kept for the
    backward: h and one float per row."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, relu, eight_bit):
        y, h, rstd, kept = feature_ops.rms_norm(x, weight, residual, eps, relu, eight_bit=eight_bit)
        ctx.save_for_backward(h, rstd, weight)
        ctx.relu, ctx.stream = relu, residual is not None
        ctx.set_materialize_grads(False)
        q, scales = (kept.q, kept.scales) if eight_bit else (None, None)
        if eight_bit:
            ctx.mark_non_differentiable(q, scales)
        return y, h if ctx.stream else None, q, scales

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh, _q, _scales):
        h, rstd, weight = ctx.saved_tensors
        if dy is None:  # only the residual stream went on
            return dh, dh if ctx.stream else None, None, None, None, None
        dx, dw = feature_ops.rms_norm_backward(dy.contiguous(), h, rstd, weight, None if dh is None else dh.contiguous(), ctx.relu)
        return dx, dx if ctx.stream else None, dw, None, None, None


class NodeEmbedding(torch.nn.Module):
    """Learned features: ``scale * weights[ids]`` for graphs whose nodes have none.  ``padding_idx`` names a row that takes no
    gradient (ids that fill up a batch).  ``ids``: int32 or int64 on the weights' GPU, of any shape and strides."""

    def __init__(self, n_rows, dim, scale=1.0, padding_idx=None):
        super().__init__()
        if padding_idx is not None and not 0 <= padding_idx < n_rows:
            raise ValueError("padding_idx must be a row of the table")
        self.scale, self.padding_idx = scale, padding_idx
        self.weights = torch.nn.Parameter(torch.empty(n_rows, dim))
        self.reset_parameters()

    def reset_parameters(self):
        stdv = 1.0 / math.sqrt(self.weights.size(1))
        self.weights.data.uniform_(-stdv, stdv)
        if self.padding_idx is not None:
            self.weights.data[self.padding_idx] = 0

    def forward(self, ids):
        return EmbeddingFunction.apply(ids.contiguous() if isinstance(ids, torch.Tensor) else ids, self.weights, self.scale, self.padding_idx)


class RMSNorm(torch.nn.Module):
    """Root-mean-square norm of ``x + residual``, then relu where asked for: the step between the layers of a deep network,

        y, h = norm(conv_out, h)              # h: the residual stream
        y, h, kept = norm(conv_out, h, eight_bit=True)
        conv_out = conv(y, spmm_dict, kept)   # the layer keeps those 8 bits for its backward instead of y

    The backward keeps h, so that with relu in here and the next layer's input in 8 bits nothing else of this step lives on.
    ``x`` and ``residual`` have one shape, any strides (other than rows are copied), and the weights' type: float32, or what
    ``.to`` has made of it."""

    def __init__(self, dim, eps=1e-6, relu=False):
        super().__init__()
        self.eps, self.relu = eps, relu
        self.weights = torch.nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None, eight_bit=False):
        x, residual = (ops._as_rows(t) if isinstance(t, torch.Tensor) else t for t in (x, residual))
        y, h, q, scales = RMSNormFunction.apply(x, residual, self.weights, self.eps, self.relu, eight_bit)
        h = x if residual is None else h
        return (y, h, feature_ops.Rows8(q, scales, x.shape[-1], x.shape)) if eight_bit else (y, h)


class _Conv(torch.nn.Module):
    # True: what a layer keeps for its weight gradient (its input; GIN: the aggregated one) is kept in 8 bits, a scale per row and 128
    # columns, and the gradient is formed from those: a quarter of the memory, off by at most 1/254 of the largest value that
    # shares the scale
    keep_input_8bit = False

    def __init__(self, input_dim, output_dim):
        super().__init__()
        self.weights = torch.nn.Parameter(torch.randn(input_dim, output_dim))
        self.reset_parameters()

    def reset_parameters(self):
        stdv = 1.0 / math.sqrt(self.weights.size(1))
        self.weights.data.uniform_(-stdv, stdv)

    def _operator(self, spmm_dict):
        dim = self.weights.size(1)
        if dim not in spmm_dict:
            raise ValueError("SpMMDecider not support dim: " + str(dim))
        return spmm_dict[dim]

    def _eight(self, X, kept):
        """``kept`` where the caller has the input in 8 bits, True where it is to be made, None where it is kept as it is."""
        if kept is None:
            return True if self.keep_input_8bit and torch.is_grad_enabled() else None
        if not isinstance(kept, feature_ops.Rows8) or kept.shape != X.shape or kept.q.device != X.device:
            raise RuntimeError("kept must be the layer's input in 8 bits")
        return kept


class GCNConv(_Conv):
    def forward(self, H, spmm_dict, kept=None):
        P = self._operator(spmm_dict)
        if REORDER_NARROW_FIRST and self.weights.size(0) < self.weights.size(1):
            P = spmm_dict.get(self.weights.size(0), P)  # the aggregation runs at the input width
        return GCNFunction.apply(H, self.weights, P, self._eight(H, kept))


class GINConv(_Conv):
    def forward(self, X, spmm_dict):
        return GINFunction.apply(X, self.weights, self._operator(spmm_dict), self._eight(X, None))


class AGNNConv(_Conv):
    # False: a fused training step keeps the projected features and recomputes the edge scores in the backward, for a
    # network that has no room for 4 bytes per edge and layer
    keep_scores = True

    def __init__(self, input_dim, output_dim):
        super().__init__(input_dim, output_dim)
        self.attention_w = torch.nn.Parameter(torch.randn(1, n_heads))

    def forward(self, X, spmm_dict, colIdx, kept=None):
        P = self._operator(spmm_dict)
        if FUSE_AGNN_INFERENCE and not torch.is_grad_enabled() and _can_fuse(P, self.weights.size(1)):
            # No gradient will be asked for: scores, scaling and aggregation in one kernel, without
            # the per-edge array the backward would need.
            Xp = ops.dense_mm(X, self.weights)
            out = ops.agnn_layer_forward(Xp, P.rowPtr, P.colIdx, _beta(self.attention_w), P.target_row)
            return out[: P.mtx_nodes if P.target_row is not None else P.rowPtr.shape[0] - 1]
        eight = self._eight(X, kept)
        if (FUSE_AGNN_TRAINING and torch.is_grad_enabled() and _can_fuse(P, self.weights.size(1))
                and _is_operator_colidx(P, colIdx)):
            return AGNNFusedFunction.apply(X, self.weights, self.attention_w, P, colIdx, self.keep_scores, eight)
        return AGNNFunction.apply(X, self.weights, self.attention_w, P, colIdx, eight)
