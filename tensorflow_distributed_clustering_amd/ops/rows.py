"""Row operators: norm, routing to clusters, grouping by cluster and the weighted way back.

What a model does to its rows (tokens, embeddings) around their assignment to clusters:

``rms_norm``, ``rms_norm_fp8``   root-mean-square norm with the residual's addition, to the
                                 rows' type or to the fp8 operand of the wide assignment
                                 (:class:`Fp8Rows`, read by ``ClusterPredictor(dtype="fp8")``)
``topk_gate``                    the k best clusters of each row and their softmax weights
``group_plan``, ``group_rows``   rows sorted by cluster
``combine_rows``                 back to the rows' order, summed with weights

On the GPU every one runs its HIP kernel (csrc/rows_*.hip), on the current stream of its
tensors' device; CPU tensors run the same formulas in PyTorch (ops/reference.py).  Rows are
fp32, fp16 or bf16 [N, D] with contiguous columns and any row stride.  All but the fp8 norm
are differentiable (once, and backward: a GPU tensor with a forward-mode tangent raises
NotImplementedError).  Nothing synchronises with the host and every buffer is a new tensor,
so the calls can be captured into a HIP graph, the gradients too: capture forward and
backward together, with no other live autograd graph of the same leaves (a captured gradient
that would go into one raises RuntimeError).  The operators can be traced and compiled:
they have shape functions and dispatch as PyTorch's own do.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import _native
from . import fp8_dim, reference as ref

ROW_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_WIDTH = 16384            # columns of a normalised row
MAX_CHOSEN = 16              # clusters per row that topk_gate chooses
MAX_GROUPS = (1 << 22) - 1
MAX_SLOTS = (1 << 31) - 2    # labels of one plan

_tdc = None


def _ops():
    global _tdc
    if _tdc is None:
        _tdc = _native.require()
    return _tdc


def _on_gpu(x, a=None, b=None) -> bool:
    """Whether the kernels take the call.  Their bindings check its arguments themselves, with
    the errors of the checks below, which are the CPU path's: a request pays for one set."""
    if (isinstance(x, torch.Tensor) and (a is None or isinstance(a, torch.Tensor))
            and (b is None or isinstance(b, torch.Tensor))):
        return x.is_cuda
    raise TypeError(f"expected tensors, got {', '.join(type(t).__name__ for t in (x, a, b) if t is not None)}")


def _check_rows(x, name: str):
    if x.dim() != 2 or x.dtype not in ROW_DTYPES:
        raise ValueError(f"{name} must be fp32, fp16 or bf16 rows [N, D], got {x.dtype} {tuple(x.shape)}")
    if x.shape[1] < 1:
        raise ValueError(f"{name} has no columns")
    if x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError(f"{name} must have contiguous columns, got strides {x.stride()}")


def _check_weight(w, x, shape, name: str):
    if tuple(w.shape) != tuple(shape) or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous {tuple(shape)}, got {tuple(w.shape)}")
    if w.dtype not in (torch.float32, x.dtype):
        raise ValueError(f"{name} must be fp32 or {x.dtype}, got {w.dtype}")
    if w.device != x.device:
        raise ValueError(f"{name} is on {w.device}, the rows on {x.device}")


# ----------------------------------------------------------------- norm
def _check_norm(x, weight, residual, eps):
    _check_rows(x, "x")
    if x.shape[1] > MAX_WIDTH:
        raise ValueError(f"rms_norm takes up to {MAX_WIDTH} columns, got {x.shape[1]}")
    if weight is not None:
        _check_weight(weight, x, (x.shape[1],), "weight")
    if residual is not None:
        _check_rows(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError("residual must have the shape, type and device of x")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
             residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``h / sqrt(mean(h^2) + eps) * weight`` of each row of ``h = x + residual``.

    Returns ``y``, or ``(y, h)`` with a residual.  ``h`` is rounded to the rows' type and
    ``y`` is the norm of that rounded row, so ``h`` is all the gradient keeps (on the
    GPU the gradient raises where it was edited in place).  ``weight`` [D] is fp32 or of the rows' type (None: ones).
    The squares are summed in fp32: a row whose sum of squares passes 3.4e38 becomes zeros.
    With ``eps`` = 0 a row of zeros becomes NaN, and one of values so small that their squares
    are zeros in fp32 (below 1e-23) becomes infinite."""
    if not _on_gpu(x, weight, residual):
        _check_norm(x, weight, residual, eps)
        return ref.rms_norm(x, weight, residual, eps)
    out = _ops().rms_norm(x, weight, residual, eps)
    return out[0] if residual is None else (out[0], out[1])


class Fp8Rows:
    """Rows in fp8: ``q`` e4m3 [N, width], ``scales`` uint8 [N, width / 32] (a value is
    ``q * 2^(scale - 127)``), ``d`` columns of them in use, zeros behind.  The operand
    layout of the fp8 assignment."""

    __slots__ = ("q", "scales", "d")

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, d: int):
        self.q, self.scales, self.d = q, scales, int(d)

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.q.shape[0], self.d)

    @property
    def device(self) -> torch.device:
        return self.q.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [N, d].  Exact in fp32 and bf16 while they are normal numbers."""
        if dtype not in ROW_DTYPES:
            raise ValueError(f"dequantize to fp32, fp16 or bf16, got {dtype}")
        if self.q.device.type != "cuda":
            return ref.dequant_fp8(self.q, self.scales, self.d).to(dtype)
        return _ops().dequant_fp8(self.q, self.scales, self.d, dtype)


def fp8_width(d: int) -> int:
    """Columns that ``d`` take as an fp8 operand: the widths of the fp8 assignment up to
    1024, then whole blocks of 32."""
    return fp8_dim(d) or (d + 31) // 32 * 32


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """:func:`rms_norm` whose ``y`` is computed in fp64 and rounded to :class:`Fp8Rows`, one
    exponent per 32 columns.  Returns the rows, or ``(rows, h)`` with a residual.  For serving:
    it has no gradient, and refuses inputs that ask for one or have a forward-mode tangent."""
    gpu = _on_gpu(x, weight, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    if not gpu and any(t is not None and unpack_dual(t).tangent is not None for t in (x, weight, residual)):
        raise NotImplementedError("rms_norm_fp8 has no forward-mode gradient")
    if not gpu or x.dim() != 2:
        _check_norm(x, weight, residual, eps)
    d = x.shape[1]
    if not gpu:
        out = ref.rms_norm_fp8(x, weight, residual, eps, fp8_width(d))
    else:
        out = _ops().rms_norm_fp8(x, weight, residual, eps, fp8_width(d))
    rows = Fp8Rows(out[0], out[1], d)
    return rows if residual is None else (rows, out[2])


# ----------------------------------------------------------------- gate
def topk_gate(scores: torch.Tensor, k: int, mask: Optional[torch.Tensor] = None,
              normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` clusters of the largest ``scores`` [N, K] of each row, 1 <= k <= min(16, K).

    Returns ``(weights fp32 [N, k], labels int32 [N, k])`` in falling order of score, equal
    scores in the order of the cluster.  ``weights``: the softmax over the chosen
    (``normalize``) or over all allowed clusters.  ``mask`` (bool [N, K], or broadcast to
    it): True where a cluster is allowed; one that is not, and one whose score is -inf, is
    never chosen, its score is not looked at and its gradient is zero.  Where fewer than k
    are left the last labels are -1 with weight 0, which :func:`group_plan` leaves out.  Both
    may be edited in place (labels over a capacity set to -1): the gradient keeps its own.  A
    NaN or +inf among the allowed scores makes the row's weights NaN."""
    gpu = _on_gpu(scores, mask)
    k, normalize = int(k), bool(normalize)
    if mask is not None and mask.shape != scores.shape:
        try:
            mask = mask.expand(scores.shape)
        except RuntimeError:
            raise ValueError(f"mask {tuple(mask.shape)} does not broadcast to "
                             f"{tuple(scores.shape)}") from None
    if gpu:
        return _ops().topk_gate(scores, mask, k, normalize)
    _check_rows(scores, "scores")
    if not 1 <= k <= min(MAX_CHOSEN, scores.shape[1]):
        raise ValueError(f"k must be 1 to {min(MAX_CHOSEN, scores.shape[1])}, got {k}")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise ValueError("mask must be a bool tensor")
        if mask.device != scores.device:
            raise ValueError(f"mask is on {mask.device}, the scores on {scores.device}")
    return ref.topk_gate(scores, k, mask, normalize)


# ----------------------------------------------------------------- groups
class RowGroups:
    """Where the rows of a batch go when they are sorted by cluster (:func:`group_plan`).

    Slot ``n * k + j`` is row n's j-th label.  ``order`` [N * k]: the slot at each place;
    ``pos`` (the labels' shape): the place of each slot; ``offsets`` [n_clusters + 1]: cluster
    c has the places ``offsets[c]`` to ``offsets[c + 1]``, in the rows' order.  Slots
    without a cluster have the places from ``offsets[n_clusters]`` on.  All int32."""

    __slots__ = ("offsets", "order", "pos", "n_clusters")

    def __init__(self, offsets: torch.Tensor, order: torch.Tensor, pos: torch.Tensor, n_clusters: int):
        self.offsets, self.order, self.pos, self.n_clusters = offsets, order, pos, n_clusters

    @property
    def n_rows(self) -> int:
        return self.pos.shape[0]

    @property
    def n_slots(self) -> int:
        return self.order.shape[0]

    @property
    def counts(self) -> torch.Tensor:
        """Rows of each cluster, int32 [n_clusters]."""
        return self.offsets[1:] - self.offsets[:-1]


def group_plan(labels: torch.Tensor, n_clusters: int) -> RowGroups:
    """Plan of the rows with ``labels`` (int32 or int64, [N] or [N, k]: k clusters per row)
    sorted by cluster; rows of one cluster keep their order.  Labels outside
    [0, n_clusters) drop their slot.  The same labels give the same plan."""
    n_clusters = int(n_clusters)
    if _on_gpu(labels):
        return RowGroups(*_ops().group_plan(labels, n_clusters), n_clusters)
    if labels.dim() not in (1, 2) or labels.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"labels must be int32 or int64 [N] or [N, k], got {labels.dtype} "
                         f"{tuple(labels.shape)}")
    if labels.dim() == 2 and labels.shape[1] < 1:
        raise ValueError("labels have no columns")
    if not 1 <= n_clusters <= MAX_GROUPS:
        raise ValueError(f"n_clusters must be 1 to {MAX_GROUPS}, got {n_clusters}")
    if labels.numel() > MAX_SLOTS:
        raise ValueError(f"at most {MAX_SLOTS} labels, got {labels.numel()}")
    return RowGroups(*ref.group_plan(labels, n_clusters), n_clusters)


def _check_groups(groups):
    if not isinstance(groups, RowGroups):
        raise TypeError(f"groups must be the RowGroups of group_plan, got {type(groups).__name__}")


def group_rows(x: torch.Tensor, groups: RowGroups) -> torch.Tensor:
    """The rows of ``x`` [N, D] sorted by cluster, [N * k, D]: a row once for each of its
    labels, zeros at the places from ``groups.offsets[-1]`` on.  The gradient sums a row's
    copies in fp32."""
    _check_groups(groups)
    if _on_gpu(x):
        return _ops().group_rows(x, groups.offsets, groups.pos)
    _check_rows(x, "x")
    if x.shape[0] != groups.n_rows or x.device != groups.pos.device:
        raise ValueError(f"the plan is of {groups.n_rows} rows on {groups.pos.device}, "
                         f"x has {x.shape[0]} on {x.device}")
    return ref.group_rows(x, groups.offsets, groups.order, groups.pos)


def combine_rows(y: torch.Tensor, groups: RowGroups, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Sorted rows ``y`` [N * k, D] back in the rows' order, [N, D]: ``sum_j weights[n, j] *
    y[place of slot (n, j)]``, in fp32 in the order of j and rounded once.  ``weights`` have
    the shape of the plan's labels, fp32 or of the rows' type (None: ones).  Slots without a
    cluster add nothing, whatever ``y`` holds there; a row that has none left is zeros."""
    _check_groups(groups)
    if _on_gpu(y, weights):
        return _ops().combine_rows(y, groups.offsets, groups.pos, weights)
    _check_rows(y, "y")
    if y.shape[0] != groups.n_slots or y.device != groups.pos.device:
        raise ValueError(f"the plan is of {groups.n_slots} places on {groups.pos.device}, "
                         f"y has {y.shape[0]} rows on {y.device}")
    if weights is not None:
        _check_weight(weights, y, groups.pos.shape, "weights")
    return ref.combine_rows(y, groups.offsets, groups.pos, weights)
