"""Row operators under PyTorch's own machinery on the GPU: forward-mode gradients, dispatch
modes, tracing, compilation, checkpoints, function transforms, gradients that nobody asked for."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

import tensorflow_distributed_clustering_amd as tdc
from tests import rows_cases as rc

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


def with_grads(gpu, call, leaves):
    """Outputs and all gradients, as tensors without a graph."""
    leaves = [t.detach().requires_grad_() for t in leaves]
    outs = tuple_of(call(gpu, *leaves))
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, leaves, [o.detach() * 0.5 for o in outs])


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


class Seen(TorchDispatchMode):
    """The operators of the package that pass, and what they return."""

    def __init__(self):
        super().__init__()
        self.names, self.outs = [], {}

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func.namespace == "tdc":
            name = func.name().split("::")[1]
            self.names.append(name)
            self.outs[name] = out
        return out


@pytest.mark.parametrize("name", CALLS)
def test_dispatch_modes_see_the_calls(gpu, name):
    call, _ = CALLS[name]
    args = inputs(gpu, name)
    want, grads = tuple_of(call(gpu, *args)), with_grads(gpu, call, args)
    for run, result in ((lambda: tuple_of(call(gpu, *args)), want), (lambda: with_grads(gpu, call, args), grads)):
        with Seen() as seen:
            got = run()
        assert all(torch.equal(a, b) for a, b in zip(got, result)) and len(got) == len(result)
        stem = {"norm": "rms_norm", "gate": "topk_gate", "group": "group_rows", "combine": "combine_rows"}[name.split()[0]]
        assert any(n.startswith(stem) for n in seen.names), seen.names
    # the gradient too: one call more than its forward pass, the plan aside
    assert len([n for n in seen.names if n != "group_plan"]) == 2, seen.names


@pytest.mark.parametrize("name", CALLS)
def test_traced_on_one_input_and_run_on_another(gpu, name):
    call, _ = CALLS[name]
    args, other = inputs(gpu, name), inputs(gpu, name, seed=10)
    for f in (lambda *a: tuple_of(call(gpu, *a)), lambda *a: with_grads(gpu, call, a)):
        for mode in ("real", "fake", "symbolic"):
            graph = make_fx(f, tracing_mode=mode)(*args)
            for given in (args, other):
                for a, b in zip(graph(*given), f(*given)):
                    assert torch.equal(a, b)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled(gpu, name, dynamic):
    """Forward and backward graphs of the compiler, run by the operators themselves."""
    call, _ = CALLS[name]
    compiled = torch.compile(lambda *a: tuple_of(call(gpu, *a)), backend="aot_eager", dynamic=dynamic)
    for seed in (0, 10):
        args = inputs(gpu, name, seed)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(compiled(*args), tuple_of(call(gpu, *args))))
        got = with_grads(gpu, lambda gpu, *a: compiled(*a), args)
        assert all(torch.equal(a, b) for a, b in zip(got, with_grads(gpu, call, args)))


def test_registered_as_pytorch_asks(gpu):
    ops = torch.ops.tdc
    x, w, s = normal(gpu, 1, 6, 40), normal(gpu, 2, 40), normal(gpu, 3, 6, 9)
    y, v, groups = normal(gpu, 4, 12, 40), normal(gpu, 5, 6, 2).abs(), plan(gpu)
    lab, rows = groups.pos % 3, tdc.rms_norm_fp8(x)
    for t in (x, w, s, y, v):
        t.requires_grad_()
    # the other checks multiply fp8 tensors, which PyTorch does not
    torch.library.opcheck(ops.rms_norm_fp8.default, (x.detach(), None, None, 1e-6, 256), test_utils="test_faketensor")
    torch.library.opcheck(ops.dequant_fp8.default, (rows.q, rows.scales, 40, torch.float32), test_utils="test_faketensor")
    for op, args in ((ops.rms_norm, (x, w, None, 1e-6)), (ops.rms_norm, (x, w, y[:6].detach(), 1e-6)),
                     (ops.topk_gate, (s, None, 3, True)), (ops.topk_gate, (s, s.detach() < 1, 3, False)),
                     (ops.group_plan, (lab, 3)), (ops.group_rows, (x, groups.offsets, groups.pos)),
                     (ops.combine_rows, (y, groups.offsets, groups.pos, v))):
        torch.library.opcheck(op.default, args, test_utils=(
            "test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.parametrize("d", [7, 300, 5003])          # rows of a few threads, a wave, a block
@pytest.mark.parametrize("with_sum", [False, True])
def test_norm_with_a_gradient_of_the_weight_alone(gpu, d, with_sum):
    x, r, dy = normal(gpu, 1, 70, d), normal(gpu, 2, 70, d), normal(gpu, 3, 70, d)
    residual, w = (r if with_sum else None), normal(gpu, 4, d).requires_grad_()
    out = tuple_of(tdc.rms_norm(x, w, residual=residual))
    assert out[0].requires_grad and not any(h.requires_grad for h in out[1:])
    with Seen() as seen:
        dw, = torch.autograd.grad(out[0], w, dy)
    assert len(seen.outs["rms_norm_bwd"]) == 1           # no gradient of rows is computed
    h = rc.sum_kept(x, residual)
    _, _, want, scale = rc.norm_grads(h, w.detach(), 1e-6, dy, None)
    rc.close(dw, want, torch.float32, scale=scale, factor=2)
    both, = torch.autograd.grad(tuple_of(tdc.rms_norm(x.requires_grad_(), w, residual=residual))[0], w, dy)
    assert torch.equal(both, dw)


@pytest.mark.parametrize("name", CALLS)
def test_checkpointed(gpu, name):
    """Recomputed in the backward pass, whole and with the package's own results kept."""
    call, _ = CALLS[name]
    args = inputs(gpu, name)
    want = with_grads(gpu, call, args)

    def keep(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if op.namespace == "tdc" else CheckpointPolicy.PREFER_RECOMPUTE

    for extra in ({}, {"context_fn": lambda: create_selective_checkpoint_contexts(keep)}):
        again = lambda gpu, *a: checkpoint(lambda *b: tuple_of(call(gpu, *b)), *a, use_reentrant=False, **extra)  # noqa: E731,B023
        assert all(torch.equal(a, b) for a, b in zip(with_grads(gpu, again, args), want))


@pytest.mark.parametrize("name", CALLS)
def test_function_transforms_are_right_or_refused(gpu, name):
    call, _ = CALLS[name]
    args = inputs(gpu, name)
    first = lambda *a: tuple_of(call(gpu, *a))[0]  # noqa: E731
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda *a: first(*a).sum())(*args)
    with pytest.raises(RuntimeError):
        torch.func.jvp(first, tuple(args), tuple(torch.ones_like(a) for a in args))
    many = [torch.stack([a, 2 * a, -a]) for a in args]
    if name.startswith("norm"):        # lists of results have no loop over a batch
        with pytest.raises(RuntimeError):
            torch.vmap(first)(*many)
    else:
        want = torch.stack([first(*(m[i] for m in many)) for i in range(3)])
        assert torch.equal(torch.vmap(first)(*many), want)


def test_gradients_of_leaves_are_their_own(gpu):
    """x and residual have the same gradient, in memory of their own each."""
    x, r = normal(gpu, 1, 6, 40).requires_grad_(), normal(gpu, 2, 6, 40).requires_grad_()
    y, h = tdc.rms_norm(x, residual=r)
    up = torch.ones_like(h)
    torch.autograd.backward((y, h), (y.detach(), up))
    kept = r.grad.clone()
    assert torch.equal(x.grad, kept)
    x.grad.zero_()
    assert torch.equal(r.grad, kept) and bool((up == 1).all())
    x.grad = None
    y, h = tdc.rms_norm(x, residual=r.detach())
    h.backward(up)                     # the incoming gradient goes through
    x.grad.zero_()
    assert bool((up == 1).all())
