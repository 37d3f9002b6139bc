"""Row operators on the GPU at the sizes that choose another path: plans of one to many chunks
and one or two digits, more labels of a row than one round takes, moved rows past the caches,
masks of any stride, gradients past 2^31 elements."""
import pytest
import torch

import tensorflow_distributed_clustering_amd as tdc
from tests import rows_cases as rc

pytestmark = pytest.mark.gpu


def normal(gpu, seed, *shape, dtype=torch.float32):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=gpu).to(dtype)


def check_plan(groups, labels, clusters):
    flat = labels.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < clusters), flat, clusters)
    skey, order = torch.sort(key, stable=True)
    assert torch.equal(groups.order.long(), order) and groups.pos.shape == labels.shape
    assert torch.equal(groups.pos.reshape(-1)[order].long(), torch.arange(len(flat), device=flat.device))
    assert torch.equal(groups.offsets.long(), torch.searchsorted(skey, torch.arange(clusters + 1, device=flat.device)))


# one chunk of 1024 or 2048 slots, a few chunks, more than the blocks sum themselves, 2048 and
# 4096 slots a chunk; a digit of each
@pytest.mark.parametrize("n", [1024, 1025, 2048, 2049, 40000, 65536, 65537, 200000, 2097152, 2100000])
@pytest.mark.parametrize("clusters", [7, 600, 2047, 4000, 65536, 1 << 20])
def test_plans(gpu, n, clusters):
    g = torch.Generator(device=gpu).manual_seed(n + clusters)
    labels = torch.randint(-1, clusters + 1, (n, 3), generator=g, dtype=torch.int32, device=gpu)
    labels[: n // 3] = clusters // 2                 # one cluster far above the others
    one = labels[:, 1]                               # not contiguous
    check_plan(tdc.group_plan(one, clusters), one, clusters)
    wide = one.long() + torch.where(one < 0, -(1 << 40), 0)
    check_plan(tdc.group_plan(wide, clusters), wide, clusters)


@pytest.mark.parametrize("n,k,clusters", [(700, 9, 5), (300000, 8, 3000)])
def test_plans_of_several_labels_a_row(gpu, n, k, clusters):
    g = torch.Generator(device=gpu).manual_seed(n)
    labels = torch.randint(-1, clusters + 1, (n, k), generator=g, device=gpu)
    check_plan(tdc.group_plan(labels, clusters), labels, clusters)
    back = labels.t().contiguous().t()               # columns far apart
    check_plan(tdc.group_plan(back, clusters), back, clusters)


def check_moved(gpu, n, k, d, dtype):
    """group_rows, combine_rows and their gradients against sums in 64 bits."""
    clusters = 5
    g = torch.Generator(device=gpu).manual_seed(n + k)
    labels = torch.randint(-1, clusters + 1, (n, k), generator=g, device=gpu, dtype=torch.int32)
    labels[: n // 8] = -1                            # rows with nothing left
    groups = tdc.group_plan(labels, clusters)
    total = int(groups.offsets[-1])
    slot = groups.order[:total].long()
    row = slot // k

    def to_rows(v):
        return torch.zeros(n, d, dtype=torch.float64, device=gpu).index_add_(0, row, v)

    x, dxg = normal(gpu, 1, n, d, dtype=dtype).requires_grad_(), normal(gpu, 2, n * k, d, dtype=dtype)
    xg = tdc.group_rows(x, groups)
    assert torch.equal(xg[:total], x[row]) and not bool(xg[total:].any())
    dx, = torch.autograd.grad(xg, x, dxg)
    v = dxg[:total].double()
    rc.close(dx, to_rows(v), dtype, scale=to_rows(v.abs()))
    del x, dxg, xg, dx, v

    y, dout = normal(gpu, 3, n * k, d, dtype=dtype), normal(gpu, 4, n, d, dtype=dtype)
    y[total:] = float("nan")                         # never read
    w = torch.rand(n, k, generator=g, device=gpu)
    y.requires_grad_(), w.requires_grad_()
    out = tdc.combine_rows(y, groups, w)
    ws, ys = w.detach().view(-1, 1).double()[slot], y.detach()[:total].double()
    rc.close(out.detach(), to_rows(ws * ys), dtype, scale=to_rows((ws * ys).abs()))
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    gs = dout[row].double()
    rc.close(dy[:total], ws * gs, dtype)
    assert not bool(dy[total:].any())
    ys *= gs
    want = torch.zeros(2, n * k, dtype=torch.float64, device=gpu)
    want[0, slot], want[1, slot] = ys.sum(1), ys.abs().sum(1)
    rc.close(dw.view(-1), want[0], torch.float32, scale=want[1])
    assert not bool(dw.view(-1)[groups.pos.view(-1) >= total].any())


@pytest.mark.parametrize("k", [9, 11, 16, 17, 33])
@pytest.mark.parametrize("n,d", [(1, 3), (33, 64), (17, 1001), (40, 4096)])
@pytest.mark.parametrize("dtype", rc.DTYPES)
def test_more_labels_a_row_than_one_round_takes(gpu, n, k, d, dtype):
    check_moved(gpu, n, k, d, dtype)


# sorted rows of 256 MiB and more: even and odd widths, rows within a wave's vectors and longer
@pytest.mark.parametrize("n,k,d,dtype", [(16400, 8, 1025, torch.bfloat16), (17000, 4, 1024, torch.float32),
                                         (300000, 1, 451, torch.float16), (7000, 2, 5001, torch.float32),
                                         (9000, 9, 1001, torch.float32), (24000000, 2, 3, torch.bfloat16)])
def test_moved_rows_past_the_caches(gpu, n, k, d, dtype):
    assert n * k * d * dtype.itemsize >= 256 << 20
    check_moved(gpu, n, k, d, dtype)


# ----------------------------------------------------------------- gate
@pytest.mark.parametrize("clusters", [3, 60, 129, 1000, 4099, 9001])
@pytest.mark.parametrize("dtype", rc.DTYPES)
def test_masks_of_any_stride(gpu, clusters, dtype):
    n, k = 9, 3
    s = normal(gpu, clusters, n, clusters, dtype=dtype)
    dw = normal(gpu, 2, n, k)
    flat = torch.rand(clusters, n, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu) > 0.3
    rows = torch.arange(n, device=gpu)[:, None] % 3 > 0
    every = (torch.rand(n, 2 * clusters, generator=torch.Generator(device=gpu).manual_seed(2), device=gpu) > 0.3)[:, ::2]
    back = torch.zeros(n, clusters + 7, dtype=torch.bool, device=gpu)[:, 5:5 + clusters]
    back.copy_(flat.t())
    for mask in (flat.t(), rows, flat.t()[:1], every, back, back[0]):
        for normalize in (True, False):
            leaf = s.detach().requires_grad_()
            w, lab = tdc.topk_gate(leaf, k, mask=mask, normalize=normalize)
            ww, wl, wd = rc.gate(s.cpu(), k, mask.cpu(), normalize, dw.cpu())
            assert torch.equal(lab.cpu(), wl)
            rc.close(w.detach(), ww, torch.float32, scale=torch.ones(1))
            ds, = torch.autograd.grad(w, leaf, dw)
            rc.close(ds, wd, dtype, scale=dw.abs().max())


# ----------------------------------------------------------------- large
def test_norm_gradient_past_32_bits(gpu):
    n, d = 140_000, 16384                            # 2.29e9 elements
    x = torch.ones(n, d, dtype=torch.bfloat16, device=gpu)
    dy = torch.zeros(n, d, dtype=torch.bfloat16, device=gpu)
    at = [0, n // 2, n - 2, n - 1]
    x[at], dy[at] = normal(gpu, 1, 4, d, dtype=torch.bfloat16), normal(gpu, 2, 4, d, dtype=torch.bfloat16)
    w = normal(gpu, 3, d).requires_grad_()
    x.requires_grad_()
    dx, dw = torch.autograd.grad(tdc.rms_norm(x, w), (x, w), dy)
    want, scale, ww, ws = rc.norm_grads(x.detach()[at], w.detach(), 1e-6, dy[at], None)
    rc.close(dx[at], want, torch.bfloat16, scale=scale)
    rc.close(dw, ww, torch.float32, scale=ws, factor=2)
    assert not bool(dx[1:n // 2].any())


def test_moved_rows_past_32_bits(gpu):
    n, k, d = 70_000, 2, 16384                       # 2.29e9 elements of sorted rows
    labels = torch.stack([torch.arange(n, device=gpu) % 7 - 1, torch.arange(n, device=gpu) % 5], 1)
    groups = tdc.group_plan(labels, 5)
    total = int(groups.offsets[-1])
    slot = groups.order.long()
    y = normal(gpu, 1, 1, d, dtype=torch.bfloat16).expand(n * k, d).contiguous()
    y[-40_000:-39_000] *= 2
    dout = normal(gpu, 2, n, d, dtype=torch.bfloat16)
    w = torch.rand(n, k, generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)
    y.requires_grad_(), w.requires_grad_()
    dy, dw = torch.autograd.grad(tdc.combine_rows(y, groups, w), (y, w), dout)
    at = torch.tensor([0, 1, 40_000, total // 2, total - 2, total - 1], device=gpu)
    sl = slot[at]
    gs, ys = dout[sl // k].double(), y.detach()[at].double()
    rc.close(dy[at], w.detach().view(-1)[sl, None].double() * gs, torch.bfloat16)
    rc.close(dw.view(-1)[sl], (gs * ys).sum(1), torch.float32, scale=(gs * ys).abs().sum(1))
    assert not bool(dy[total:].any()) and not bool(dw.view(-1)[slot[total:]].any())
    del y, dy
    x = dout.requires_grad_()
    xg = tdc.group_rows(x, groups)
    assert torch.equal(xg[at], x[sl // k]) and not bool(xg[total:].any())
    dx, = torch.autograd.grad(xg, x, xg.detach())
    r = torch.tensor([0, 1, n - 2, n - 1], device=gpu)
    copies = ((labels[r] >= 0) & (labels[r] < 5)).sum(1, keepdim=True)
    rc.close(dx[r], copies * x.detach()[r].double(), torch.bfloat16, scale=2 * x.detach()[r].double().abs())
