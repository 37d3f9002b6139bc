"""Oracles of the row operators in 64 bits, and the tolerances that follow from their types.

half(t) is the largest relative error of one rounding to t.  The kernels' fp32 sums of n
terms are off by at most about n * half(fp32) of the sum of magnitudes, in practice far
less; SUM covers widths to 16384 with tree sums (log2 n + a few roundings, taken as 32).
"""
import torch

import tensorflow_distributed_clustering_amd as tdc
from tensorflow_distributed_clustering_amd.ops import rows as R

DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def half(t):
    return torch.finfo(t).eps / 2


SUM = 32 * half(torch.float32)


def close(got, want, dtype, scale=None, factor=1.0):
    """got (of dtype) against want (fp64): one rounding to dtype and fp32 arithmetic of
    `factor` sums, relative to `scale` (default: the value itself); the smallest normal of
    fp16 bounds what its subnormals lose."""
    want = want.double().to(got.device)
    scale = want.abs() if scale is None else scale.double().to(got.device)
    tol = half(dtype) * want.abs() * 1.01 + factor * SUM * scale + torch.finfo(dtype).tiny * half(dtype) * 2
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} off, worst "
        f"{float(((got.double() - want).abs() / tol).nan_to_num(nan=1e9).max()):.3g} of the tolerance")


def sum_kept(x, residual):
    """h: the sum in fp32, rounded to the rows' type (exact sum, one rounding, for 16 bits
    unless the fp32 sum is itself rounded, in the kernel alike)."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def norm(h, weight, eps):
    h = h.double()
    t = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return t, (t if weight is None else t * weight.double())


def norm_grads(h, weight, eps, dy, dh):
    """(dx, scale of dx's terms, dw, scale of dw's terms) from the formula."""
    h64, dy = h.double(), dy.double()
    rstd = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps)
    t = h64 * rstd
    g = dy if weight is None else dy * weight.double()
    c, ca = (g * t).mean(1, keepdim=True), (g * t).abs().mean(1, keepdim=True)
    dx, scale = rstd * (g - t * c), rstd * (g.abs() + t.abs() * ca)
    if dh is not None:
        dx, scale = dx + dh.double(), scale + dh.double().abs()
    return dx, scale, (dy * t).sum(0), (dy * t).abs().sum(0)


def fp8(y64, width):
    """(values, exponents) of rows in 64 bits as e4m3 with one exponent per 32 columns."""
    # on the CPU, where powers of two come out exact
    b = torch.nn.functional.pad(y64.cpu(), (0, width - y64.shape[1])).view(y64.shape[0], width // 32, 32)
    top = b.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 8, -127).clamp(-127, 126)
    v = torch.ldexp(b, -e)
    x = torch.where(v == 0, -6, torch.frexp(v)[1] - 1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(v), x - 3)
    q = torch.round(v / step) * step
    return torch.ldexp(q, e).view(y64.shape[0], width).to(y64.device), e.squeeze(2).to(y64.device)


def gate(scores, k, mask, normalize, dw=None):
    """(weights, labels[, ds]) row by row: NaN above +inf, equal scores by their index."""
    v = scores.double()
    n, clusters = v.shape
    ok = (v != -torch.inf) if mask is None else (mask.expand(v.shape) & (v != -torch.inf))
    weights = torch.zeros(n, k, dtype=torch.float64)
    labels = torch.full((n, k), -1, dtype=torch.int32)
    ds = torch.zeros(n, clusters, dtype=torch.float64)
    for r in range(n):
        idx = ok[r].nonzero().flatten()
        nan = v[r, idx].isnan()
        idx = torch.cat([idx[nan], idx[~nan][torch.sort(v[r, idx[~nan]], descending=True, stable=True)[1]]])
        pick = idx[:k]
        if not len(pick):
            continue
        of = pick if normalize else idx
        p = torch.zeros(clusters, dtype=torch.float64)
        p[of] = torch.softmax(v[r, of], 0)
        labels[r, :len(pick)] = pick.int()
        weights[r, :len(pick)] = p[pick]
        if dw is not None:
            up = torch.zeros(clusters, dtype=torch.float64)
            up[pick] = dw[r, :len(pick)].double()
            ds[r] = p * (up - (p * up).sum())
    return (weights, labels) if dw is None else (weights, labels, ds)


def plan(labels, clusters):
    flat = labels.reshape(-1).tolist()
    key = [v if 0 <= v < clusters else clusters for v in flat]
    order = sorted(range(len(key)), key=lambda i: key[i])
    pos = [0] * len(key)
    for p, i in enumerate(order):
        pos[i] = p
    offsets = [sum(1 for v in key if v < c) for c in range(clusters + 1)] if len(key) * clusters < 1 << 22 else \
        torch.searchsorted(torch.tensor(sorted(key)), torch.arange(clusters + 1)).tolist()
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return t(offsets), t(order), t(pos).view(labels.shape)


def check_dropped_weights(device, bad):
    """Slots without a cluster add nothing to a row and get no gradient, whatever weight and
    row they hold.  Every value is a small whole number: exact in any order."""
    lab = torch.tensor([[0, -1], [5, 1], [-1, 7], [1, 0]], dtype=torch.int32, device=device)
    drop = (lab < 0) | (lab >= 2)
    w = torch.tensor([[2.0, 0.0], [0.0, 3.0], [0.0, 0.0], [1.0, -4.0]], device=device)
    w = torch.where(drop, bad, w).requires_grad_()
    groups = tdc.group_plan(lab, 2)
    y = torch.arange(8.0, device=device)[:, None] + torch.tensor([0.0, 10.0, 20.0], device=device)
    y[int(groups.offsets[-1]):] = bad
    y.requires_grad_()
    out = tdc.combine_rows(y, groups, w)
    at = torch.where(drop, 0, groups.pos.long())
    rows = y.detach()[at]                            # [4, 2, 3]; place 0 is kept
    keep = torch.where(drop, 0.0, w.detach())[..., None]
    assert torch.equal(out.detach(), (keep * rows).sum(1))
    dout = torch.arange(12.0, device=device).view(4, 3)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    assert torch.equal(dw, torch.where(drop, 0.0, (rows * dout[:, None]).sum(2)))
    want = torch.zeros(8, 3, device=device)
    for r, j in (~drop).nonzero().tolist():
        want[groups.pos[r, j].long()] = keep[r, j] * dout[r]
    assert torch.equal(dy, want)


def check_gate_edited(device, normalize):
    """What a router does with its choice: drop labels over a capacity, put the weights right,
    in place."""
    g = torch.Generator().manual_seed(1)
    s, dw = torch.randn(50, 12, generator=g).to(device), torch.randn(50, 3, generator=g).to(device)
    over = (torch.rand(50, 3, generator=g) < 0.3).to(device)
    res = []
    for edit in (True, False):
        leaf = s.clone().requires_grad_()
        w, lab = tdc.topk_gate(leaf, 3, normalize=normalize)
        if edit:
            lab[over] = -1
            w.masked_fill_(over, 0.0).mul_(2.0)
        else:
            lab, w = torch.where(over, -1, lab), torch.where(over, 0.0, w) * 2.0
        res.append((w.detach(), lab, torch.autograd.grad(w, leaf, dw)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*res))


# calls that are refused, on rows x [4, 8] and labels l [4] of either device
REFUSALS = {
    "norm list": (lambda x, l: tdc.rms_norm([1.0]), TypeError),
    "norm 1-D": (lambda x, l: tdc.rms_norm(x[0]), ValueError),
    "norm fp64": (lambda x, l: tdc.rms_norm(x.double()), ValueError),
    "norm columns": (lambda x, l: tdc.rms_norm(x.t()), ValueError),
    "norm no columns": (lambda x, l: tdc.rms_norm(x[:, :0]), ValueError),
    "norm too wide": (lambda x, l: tdc.rms_norm(x.new_zeros(1, R.MAX_WIDTH + 1)), ValueError),
    "norm weight list": (lambda x, l: tdc.rms_norm(x, [1.0] * 8), TypeError),
    "norm weight short": (lambda x, l: tdc.rms_norm(x, x.new_ones(7)), ValueError),
    "norm weight type": (lambda x, l: tdc.rms_norm(x, x.new_ones(8).half()), ValueError),
    "norm weight strided": (lambda x, l: tdc.rms_norm(x, x.new_ones(16)[::2]), ValueError),
    "norm weight 2-D": (lambda x, l: tdc.rms_norm(x, x.new_ones(1, 8)), ValueError),
    "norm residual type": (lambda x, l: tdc.rms_norm(x, residual=x.half()), ValueError),
    "norm residual rows": (lambda x, l: tdc.rms_norm(x, residual=x[:3]), ValueError),
    "norm residual columns": (lambda x, l: tdc.rms_norm(x[:, :4], residual=x.t()[:4]), ValueError),
    "norm eps negative": (lambda x, l: tdc.rms_norm(x, eps=-1.0), ValueError),
    "norm eps nan": (lambda x, l: tdc.rms_norm(x, eps=float("nan")), ValueError),
    "fp8 gradient": (lambda x, l: tdc.rms_norm_fp8(x.clone().requires_grad_()), RuntimeError),
    "fp8 1-D": (lambda x, l: tdc.rms_norm_fp8(x[0]), ValueError),
    "fp8 too wide": (lambda x, l: tdc.rms_norm_fp8(x.new_zeros(1, R.MAX_WIDTH + 1)), ValueError),
    "fp8 to fp64": (lambda x, l: tdc.rms_norm_fp8(x).dequantize(torch.float64), ValueError),
    "gate k 0": (lambda x, l: tdc.topk_gate(x, 0), ValueError),
    "gate k above clusters": (lambda x, l: tdc.topk_gate(x, 9), ValueError),
    "gate k 17": (lambda x, l: tdc.topk_gate(x.new_zeros(2, 40), 17), ValueError),
    "gate scores": (lambda x, l: tdc.topk_gate(l, 2), ValueError),
    "gate mask type": (lambda x, l: tdc.topk_gate(x, 2, mask=x), ValueError),
    "gate mask shape": (lambda x, l: tdc.topk_gate(x, 2, mask=x[:3] == 0), ValueError),
    "gate mask list": (lambda x, l: tdc.topk_gate(x, 2, mask=[True] * 8), TypeError),
    "plan list": (lambda x, l: tdc.group_plan([1], 2), TypeError),
    "plan floats": (lambda x, l: tdc.group_plan(x, 2), ValueError),
    "plan 3-D": (lambda x, l: tdc.group_plan(l[:, None, None], 2), ValueError),
    "plan no columns": (lambda x, l: tdc.group_plan(l[:, None][:, :0], 2), ValueError),
    "plan no clusters": (lambda x, l: tdc.group_plan(l, 0), ValueError),
    "plan too many clusters": (lambda x, l: tdc.group_plan(l, R.MAX_GROUPS + 1), ValueError),
    "group no plan": (lambda x, l: tdc.group_rows(x, None), TypeError),
    "group rows": (lambda x, l: tdc.group_rows(x, tdc.group_plan(l[:3], 2)), ValueError),
    "group type": (lambda x, l: tdc.group_rows(x.double(), tdc.group_plan(l, 2)), ValueError),
    "combine rows": (lambda x, l: tdc.combine_rows(x, tdc.group_plan(l[:3], 2)), ValueError),
    "combine weights shape": (lambda x, l: tdc.combine_rows(x, tdc.group_plan(l, 2), x.new_ones(4, 1)), ValueError),
    "combine weights type": (lambda x, l: tdc.combine_rows(x, tdc.group_plan(l, 2), x.new_ones(4).double()), ValueError),
    "combine weights list": (lambda x, l: tdc.combine_rows(x, tdc.group_plan(l, 2), [1.0] * 4), TypeError),
}
