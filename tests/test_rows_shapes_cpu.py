"""Shapes of the row operators' results for tensors without data, as tracing and compilation
ask for them: the GPU operators on fake tensors, which need no GPU, against the CPU path."""
import pytest
import sympy
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

import tensorflow_distributed_clustering_amd as tdc
from tensorflow_distributed_clustering_amd import _native
from tests import rows_cases as rc

pytestmark = pytest.mark.skipif(not _native.available(), reason="native extension not built")


def on(device, dtype=torch.float32, n=6):
    x, r = torch.zeros(n, 40, dtype=dtype, device=device), torch.zeros(n, 40, dtype=dtype, device=device)
    w = torch.ones(40, device=device)
    y, wt = torch.zeros(2 * n, 40, dtype=dtype, device=device), torch.ones(n, 2, device=device)
    lab = torch.zeros(n, 2, dtype=torch.int64, device=device)
    mask = torch.ones(n, 40, dtype=torch.bool, device=device)
    return x, r, w, y, wt, lab, mask


def results(x, r, w, y, wt, lab, mask):
    groups, flat = tdc.group_plan(lab, 5), tdc.group_plan(lab[:, 0], 3000)
    rows, h = tdc.rms_norm_fp8(x, w, residual=r)
    out = [tdc.rms_norm(x), *tdc.rms_norm(x, w, residual=r), rows.q, rows.scales, h,
           rows.dequantize(torch.float16), *tdc.topk_gate(x, 3), *tdc.topk_gate(x, 1, mask=mask, normalize=False),
           *(t for g in (groups, flat) for t in (g.offsets, g.order, g.pos)),
           tdc.group_rows(x, groups), tdc.group_rows(x, flat), tdc.combine_rows(y, groups, wt),
           tdc.combine_rows(y, groups), tdc.combine_rows(y[: x.shape[0]], flat)]
    return out


def gradients(x, r, w, y, wt, lab, mask):
    """What the backward operators return, and the shapes they should have."""
    ops = _native.require()
    groups = tdc.group_plan(lab, 5)
    n, k = wt.shape
    stat = torch.zeros(n, 2, device=x.device)
    best, labels = tdc.topk_gate(x, 3)
    chosen = torch.zeros(n, 3, 2, dtype=torch.int32, device=x.device)
    return [
        (ops.rms_norm_train(x, w, None, 1e-6), [x, torch.zeros(n, device=x.device)]),
        (ops.rms_norm_train(x, w, r, 1e-6), [x, x, torch.zeros(n, device=x.device)]),
        (ops.rms_norm_bwd(x, w, stat[:, 0].contiguous(), r, None, True, True), [x, w]),
        (ops.rms_norm_bwd(x, w, stat[:, 0].contiguous(), r, None, False, True), [w]),
        (ops.rms_norm_bwd(x, None, stat[:, 0].contiguous(), r, r, True, False), [x]),
        (ops.topk_gate_train(x, None, 3, True), [best, labels, chosen]),
        (ops.topk_gate_train(x, mask, 3, False), [best, labels, chosen, stat]),
        ([ops.topk_gate_bwd(None, None, chosen, None, best, 40, x.dtype)], [x]),
        ([ops.topk_gate_bwd(x, mask, chosen, stat, best, 40, x.dtype)], [x]),
        (ops.combine_rows_bwd(x, y, groups.offsets, groups.pos, wt, True), [y, wt]),
        (ops.combine_rows_bwd(x, None, groups.offsets, groups.pos, wt, True), [y]),
        (ops.combine_rows_bwd(x, y, groups.offsets, groups.pos, wt, False), [wt]),
    ]


def same(got, want, device="cuda"):
    assert got.dtype == want.dtype and got.device.type == device
    assert [int(s) for s in got.shape] == list(want.shape)
    assert [int(s) for s in got.stride()] == list(torch.empty(want.shape).stride())


@pytest.mark.parametrize("dtype", rc.DTYPES)
@pytest.mark.parametrize("n", [0, 6])
def test_shapes(dtype, n):
    want = results(*on("cpu", dtype, n))
    with FakeTensorMode():
        got = results(*on("cuda", dtype, n))
        assert len(got) == len(want)
        for a, b in zip(got, want):
            same(a, b)
        for outs, like in gradients(*on("cuda", dtype, n)):
            assert len(outs) == len(like)
            for a, b in zip(outs, like):
                same(a, b)


def test_shapes_with_a_graph():
    """The autograd nodes, whose forward half is an operator of its own."""
    args, want = on("cpu"), results(*on("cpu"))
    with FakeTensorMode():
        x, r, w, y, wt, lab, mask = on("cuda")
        for t in (x, w, y, wt):
            t.requires_grad_()
        groups = tdc.group_plan(lab, 5)
        for got, shape in ((tdc.rms_norm(x), (6, 40)), (tdc.rms_norm(x, w, residual=r)[1], (6, 40)),
                           (tdc.topk_gate(x, 3)[0], (6, 3)), (tdc.topk_gate(x, 3, mask=mask, normalize=False)[0], (6, 3)),
                           (tdc.group_rows(x, groups), (12, 40)), (tdc.combine_rows(y, groups, wt), (6, 40))):
            assert got.requires_grad and got.shape == shape and got.device.type == "cuda"


def test_shapes_of_any_number_of_rows():
    """The number of rows as a symbol: the operators leave it one."""
    mode = FakeTensorMode(shape_env=ShapeEnv())
    dyn = lambda t: mode.from_tensor(t, symbolic_context=StatelessSymbolicContext(  # noqa: E731
        dynamic_sizes=[DimDynamic.DYNAMIC] + [DimDynamic.STATIC] * (t.dim() - 1)))
    x, lab = dyn(torch.zeros(6, 40, device="meta")), dyn(torch.zeros(6, 2, dtype=torch.int64, device="meta"))
    ops = _native.require()
    with mode:
        outs = [ops.rms_norm(x, None, None, 1e-6)[0], *ops.topk_gate(x, None, 3, True), *ops.group_plan(lab, 5)[1:]]
        assert all(isinstance(t.shape[0], torch.SymInt) for t in outs)
    # what is asked of the symbol are the limits of the calls, not its value
    assert not any(isinstance(g.expr, sympy.Eq) for g in mode.shape_env.guards)


@pytest.mark.parametrize("name", [n for n in rc.REFUSALS if n not in ("fp8 gradient",)])
def test_refusals(name):
    call, error = rc.REFUSALS[name]
    with FakeTensorMode(), pytest.raises(error):
        call(torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"))
