"""Row operators under PyTorch's own machinery on the GPU: forward-mode gradients."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import tensorflow_distributed_clustering_amd as tdc

pytestmark = pytest.mark.gpu


def normal(gpu, seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(gpu)


def plan(gpu):
    return tdc.group_plan((torch.arange(12, device=gpu) * 7 % 5 - 1).view(6, 2), 3)   # -1 .. 3 of 0 .. 2


# name: (call, shapes of its differentiable inputs)
CALLS = {
    "norm": (lambda gpu, x, w, r: tdc.rms_norm(x, w, residual=r), ((6, 40), (40,), (6, 40))),
    "norm alone": (lambda gpu, x: tdc.rms_norm(x), ((6, 40),)),
    "gate": (lambda gpu, s: tdc.topk_gate(s, 3)[0], ((6, 40),)),
    "gate over all": (lambda gpu, s: tdc.topk_gate(s, 3, mask=s.detach() < 1, normalize=False)[0], ((6, 40),)),
    "group": (lambda gpu, x: tdc.group_rows(x, plan(gpu)), ((6, 40),)),
    "combine": (lambda gpu, y, w: tdc.combine_rows(y, plan(gpu), w), ((12, 40), (6, 2))),
    "combine unweighted": (lambda gpu, y: tdc.combine_rows(y, plan(gpu)), ((12, 40),)),
}


def inputs(gpu, name, seed=0):
    return [normal(gpu, seed + i, *s) for i, s in enumerate(CALLS[name][1])]


def tuple_of(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(gpu, name):
    call, shapes = CALLS[name]
    for i in range(len(shapes)):
        for mode in (torch.enable_grad, torch.no_grad):
            args = inputs(gpu, name)
            with mode(), fwd.dual_level():
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward"):
                    call(gpu, *args)
        args = inputs(gpu, name)
        with fwd.dual_level():
            args[i] = fwd.make_dual(args[i].requires_grad_(), torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward"):
                call(gpu, *args)
    # a level without a tangent of ours is fine
    args = inputs(gpu, name)
    with fwd.dual_level():
        fwd.make_dual(torch.ones(2, device=gpu), torch.ones(2, device=gpu))
        assert all(torch.equal(a, b) for a, b in zip(tuple_of(call(gpu, *args)), tuple_of(call(gpu, *args))))


def test_fp8_norm_refuses_forward_mode(gpu):
    x, w = normal(gpu, 1, 4, 40), normal(gpu, 2, 40)
    with torch.no_grad(), fwd.dual_level():
        for args in ((fwd.make_dual(x, x), w, None), (x, fwd.make_dual(w, w), None), (x, w, fwd.make_dual(x, x))):
            with pytest.raises(RuntimeError, match="gradient"):
                tdc.rms_norm_fp8(*args)
