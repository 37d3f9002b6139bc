"""Row operators on the CPU: formulas against 64 bits, gradients against the formulas and
differences, refusals, the predictor's fp8 rows and partition."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import tensorflow_distributed_clustering_amd as tdc
from tensorflow_distributed_clustering_amd.ops import rows as R
from tests import rows_cases as rc

INF = float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ----------------------------------------------------------------- formulas
@pytest.mark.parametrize("dtype", rc.DTYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, residual):
    g = gen(1)
    x = torch.randn(7, 33, generator=g).to(dtype)
    r = torch.randn(7, 33, generator=g).to(dtype) if residual else None
    w = torch.randn(33, generator=g)
    out = tdc.rms_norm(x, w, residual=r, eps=1e-5)
    h = rc.sum_kept(x, r)
    y = out[0] if residual else out
    rc.close(y, rc.norm(h, w, 1e-5)[1], dtype)
    if residual:
        assert torch.equal(out[1], h)


def test_norm_gradient_matches_differences():
    g = gen(2)
    x, r, dy, dh = (torch.randn(3, 9, generator=g) for _ in range(4))
    w = torch.randn(9, generator=g)
    x.requires_grad_(), w.requires_grad_()
    y, h = tdc.rms_norm(x, w, residual=r)
    dx, dw = torch.autograd.grad((y, h), (x, w), (dy, dh))
    fx, _, fw, _ = rc.norm_grads(h.detach(), w.detach(), 1e-6, dy, dh)
    assert torch.allclose(dx.double(), fx, atol=1e-5) and torch.allclose(dw.double(), fw, atol=1e-5)

    def loss(xv, wv):
        hv = xv + r.double()
        return (rc.norm(hv, wv, 1e-6)[1] * dy).sum() + (hv * dh).sum()

    step = 1e-6
    for i, j in ((0, 0), (1, 4), (2, 8)):
        d = torch.zeros(3, 9, dtype=torch.float64)
        d[i, j] = step
        diff = (loss(x.detach().double() + d, w.detach().double())
                - loss(x.detach().double() - d, w.detach().double())) / (2 * step)
        # the oracle's formula against central differences: O(step^2) and cancellation
        assert abs(float(diff - fx[i, j])) < 1e-7 * max(1.0, abs(float(diff)))


@pytest.mark.parametrize("d", [32, 100, 256, 1025])
def test_norm_fp8(d):
    g = gen(3)
    x = torch.randn(5, d, generator=g)
    x[:, ::7] *= 30
    x[2] = 0
    rows = tdc.rms_norm_fp8(x, eps=1e-6)
    assert rows.shape == (5, d) and rows.q.shape[1] == R.fp8_width(d) and rows.q.shape[1] % 32 == 0
    want, e = rc.fp8(rc.norm(x, None, 1e-6)[1], rows.q.shape[1])
    assert torch.equal(rows.scales.int() - 127, e.int())
    assert torch.equal(rows.dequantize(torch.bfloat16).double(), want[:, :d])
    assert bool((rows.q.float()[:, d:] == 0).all())


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_gate(normalize, masked):
    g = gen(4)
    s = torch.randn(12, 10, generator=g).to(torch.bfloat16).float()
    s[1] = s[1, 0]                 # ties: the lowest index first
    s[2] = torch.finfo(torch.float32).min
    s[3, :] = -INF
    s[4, 3:] = -INF
    s[5, 0], s[5, 1] = -0.0, 0.0
    m = torch.rand(12, 10, generator=g) > 0.3 if masked else None
    if masked:
        m[6] = False
        s[7, 2] = float("nan")
        s[7, 4] = INF
        m[7, 2] = m[7, 4] = False  # never looked at
    dw = torch.randn(12, 4, generator=g)
    s.requires_grad_()
    w, lab = tdc.topk_gate(s, 4, mask=m, normalize=normalize)
    ww, wl, wd = rc.gate(s.detach(), 4, m, normalize, dw)
    assert torch.equal(lab, wl)
    rc.close(w.detach(), ww, torch.float32, scale=torch.ones(1))
    ds, = torch.autograd.grad(w, s, dw)
    rc.close(ds, wd, torch.float32, scale=dw.abs().max())


def test_gate_nan_and_inf_that_are_allowed():
    s = torch.tensor([[0.0, float("nan"), 1.0], [0.0, INF, 1.0]])
    for normalize in (True, False):
        w, lab = tdc.topk_gate(s, 2, normalize=normalize)
        assert lab.tolist() == [[1, 2], [1, 2]] and bool(w.isnan()[0].all()) and bool(w.isnan()[1, 0])


@pytest.mark.parametrize("shape,clusters", [((0, 2), 3), ((1,), 1), ((17, 3), 5), ((300,), 4000)])
def test_plan_group_combine(shape, clusters):
    g = gen(5)
    lab = torch.randint(-2, clusters + 2, shape, generator=g)
    groups = tdc.group_plan(lab, clusters)
    for got, want in zip((groups.offsets, groups.order, groups.pos), rc.plan(lab, clusters)):
        assert torch.equal(got, want)
    assert torch.equal(groups.counts, groups.offsets[1:] - groups.offsets[:-1])
    n, k = shape[0], (shape[1] if len(shape) == 2 else 1)
    x = torch.randn(n, 6, generator=g, requires_grad=True)
    xg = tdc.group_rows(x, groups)
    total = int(groups.offsets[-1])
    assert torch.equal(xg[:total], x[groups.order.long()[:total] // k]) and not bool(xg[total:].any())
    w = torch.rand(shape, generator=g, requires_grad=True)
    y = torch.randn(n * k, 6, generator=g)
    y[total:] = float("nan")       # behind the last cluster: never read
    y.requires_grad_()
    out = tdc.combine_rows(y, groups, w)
    dout = torch.randn(n, 6, generator=g)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    want = torch.zeros(n, 6, dtype=torch.float64)
    for p in range(total):
        i = int(groups.order[p])
        want[i // k] += float(w.detach().reshape(-1)[i]) * y[p].detach().double()
        assert torch.allclose(dy[p], w.detach().reshape(-1)[i] * dout[i // k])
        assert torch.allclose(dw.reshape(-1)[i], (y[p].detach() * dout[i // k]).sum(), atol=1e-6)
    assert torch.allclose(out.detach().double(), want, atol=1e-6)
    assert not bool(dy[total:].any())
    dx, = torch.autograd.grad(xg, x, torch.ones_like(xg))
    kept = ((lab >= 0) & (lab < clusters)).view(n, -1).sum(1) if n else torch.zeros(0)
    assert torch.equal(dx, kept[:, None].expand(n, 6).float())


@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_combine_never_looks_at_the_weight_of_a_dropped_slot(bad):
    rc.check_dropped_weights(torch.device("cpu"), bad)


@pytest.mark.parametrize("normalize", [True, False])
def test_gate_outputs_edited_in_place(normalize):
    rc.check_gate_edited(torch.device("cpu"), normalize)


# ----------------------------------------------------------------- refusals
@pytest.mark.parametrize("name", rc.REFUSALS)
def test_refusals(name):
    call, error = rc.REFUSALS[name]
    with pytest.raises(error):
        call(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32))


def test_values_without_rows():
    x = torch.zeros(0, 8, requires_grad=True)
    y, h = tdc.rms_norm(x, residual=torch.zeros(0, 8))
    assert y.shape == (0, 8) and h.shape == (0, 8)
    w, lab = tdc.topk_gate(torch.zeros(0, 8), 3)
    assert w.shape == (0, 3) and lab.shape == (0, 3) and lab.dtype == torch.int32


# ----------------------------------------------------------------- predictor
def test_predictor_fp8_rows_and_partition():
    g = gen(6)
    c = torch.randn(9, 40, generator=g)
    x = torch.randn(50, 40, generator=g)
    p = tdc.ClusterPredictor(c, dtype="fp8", device="cpu")
    rows = tdc.rms_norm_fp8(x)
    lab, d2 = p.predict(rows, return_distance=True)
    assert torch.equal(lab, p.predict(rows.dequantize())) and d2.shape == (50,)
    with pytest.raises(ValueError):
        tdc.ClusterPredictor(c, dtype="fp32", device="cpu").predict(rows)
    with pytest.raises(ValueError):
        p.predict(tdc.rms_norm_fp8(x[:, :39].contiguous()))
    x.requires_grad_()
    parts, groups = p.partition(x)
    assert torch.equal(torch.autograd.grad(parts.sum(), x)[0], torch.ones_like(x))
    x = x.detach()
    lab = p.predict(x)
    for k in range(9):
        at = groups.offsets[k:k + 2].tolist()
        assert torch.equal(parts[at[0]:at[1]], x[lab == k])


def test_models_predict_fp8_rows():
    g = gen(7)
    x = torch.randn(200, 40, generator=g)
    rows = tdc.rms_norm_fp8(x)
    y = rows.dequantize()
    km = tdc.KMeans(tdc.ClusterConfig(n_clusters=5, max_iter=3, dtype="fp8", seed=1)).fit(y)
    assert torch.equal(km.predict(rows), km.predict(y))
    assert km.score(rows) == km.score(y)
    mb = tdc.MiniBatchKMeans(tdc.ClusterConfig(n_clusters=5, max_iter=3, dtype="fp8", batch_size=100, seed=1)).fit(y)
    assert torch.equal(mb.predict(rows), mb.predict(y))
    for model in (tdc.KMeans, tdc.MiniBatchKMeans):
        other = model(tdc.ClusterConfig(n_clusters=5, max_iter=2, dtype="fp32", batch_size=100, seed=1)).fit(y)
        with pytest.raises(ValueError, match="dtype='fp8'"):
            other.predict(rows)


def test_fp8_norm_refuses_forward_mode():
    x, w = torch.randn(4, 40, generator=gen(9)), torch.ones(40)
    with torch.no_grad(), fwd.dual_level():
        for args in ((fwd.make_dual(x, x), w, None), (x, fwd.make_dual(w, w), None), (x, w, fwd.make_dual(x, x))):
            with pytest.raises(RuntimeError, match="gradient"):
                tdc.rms_norm_fp8(*args)
        assert tdc.rms_norm_fp8(x, w).shape == (4, 40)


def test_forward_mode():
    """The CPU path has the tangents that the GPU refuses: against differences of the formula."""
    g = gen(10)
    x, w, t = torch.randn(4, 40, generator=g), torch.randn(40, generator=g), torch.randn(4, 40, generator=g)
    with fwd.dual_level():
        y = fwd.unpack_dual(tdc.rms_norm(fwd.make_dual(x, t), w, eps=1e-5)).tangent
    step = 1e-6
    up, down = (rc.norm(x.double() + s * t.double(), w, 1e-5)[1] for s in (step, -step))
    # values of order 10: fp32 arithmetic of a few roundings, differences of order step^2
    assert torch.allclose(y.double(), (up - down) / (2 * step), rtol=1e-5, atol=1e-5)
