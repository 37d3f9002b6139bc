"""Workloads of the row operators: norm (to 16/32 and to 8 bits), top-k gate, grouping and combining.

``listed()`` and ``draw(rng)`` give cases, ``prepare`` a case's inputs, ``run`` one pass in
plain torch operations (or, with ``own``, through the package's operators), ``exact`` the
same outputs in 64 bits from the definitions, ``work`` the bytes and operations of a pass.
"""
import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def norm(n, d, dtype, residual, train):
    return {"op": "norm", "n": n, "d": d, "dtype": dtype, "residual": residual, "train": train}


def norm8(n, d, dtype, residual):
    return {"op": "norm8", "n": n, "d": d, "dtype": dtype, "residual": residual}


def gate(n, clusters, k, dtype, normalize, masked, train):
    return {"op": "gate", "n": n, "clusters": clusters, "k": k, "dtype": dtype,
            "normalize": normalize, "masked": masked, "train": train}


def route(part, n, clusters, k, d, dtype, train, dropped=0.0):
    return {"op": part, "n": n, "clusters": clusters, "k": k, "d": d, "dtype": dtype,
            "train": train, "dropped": dropped}


def listed():
    return [
        # the norm in front of a layer while one token is decoded: launch latency
        dict(norm(1, 1024, "bf16", True, False), name="norm one token"),
        # a training step's norm over the rows of a batch, residual stream kept
        dict(norm(32768, 1024, "bf16", True, True), name="norm train"),
        # rows whose width fits no vector: 2-byte alignment of every other row
        dict(norm(6007, 1001, "fp16", False, True), name="norm train odd width"),
        # rows of a serving request, normalised into the operand of the fp8 assignment
        dict(norm8(16, 1024, "bf16", True), name="norm8 request"),
        # the embedding workload's width, a large chunk of rows
        dict(norm8(262144, 768, "bf16", True), name="norm8 embeddings"),
        # routing of the few tokens of a decode step
        dict(gate(4, 64, 2, "bf16", True, False, False), name="gate request"),
        # routing of a training batch, weights over the chosen
        dict(gate(65536, 256, 8, "fp32", True, False, True), name="gate train"),
        # many clusters, some not allowed for a row (capacity, padding), weights over all
        dict(gate(12289, 1000, 6, "bf16", False, True, True), name="gate train wide masked"),
        # a decode step's tokens to their clusters and back
        dict(route("route", 8, 64, 2, 1024, "bf16", False), name="route request"),
        # a training batch's rows copied to their clusters, and the copies' gradients summed
        dict(route("group", 16384, 256, 8, 1024, "bf16", True, 0.03), name="group train"),
        # rows laid out by cluster, K of the embedding workload (inverted lists)
        dict(route("group", 1000000, 65536, 1, 128, "bf16", False), name="group lists"),
        # the weighted way back with the gradients of rows and weights
        dict(route("combine", 16384, 256, 8, 1024, "bf16", True, 0.03), name="combine train"),
    ]


def spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "gate", "route", "group", "combine"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.6
    if op in ("norm", "norm8"):
        d = spread(rng, 48, 8192)
        if rng.random() < 0.6:
            d = max(64, d // 64 * 64)
        n = spread(rng, 1, max(2, min(262144, 24_000_000 // d)))
        residual = rng.random() < 0.6
        return norm(n, d, dtype, residual, train) if op == "norm" else norm8(n, d, dtype, residual)
    if op == "gate":
        clusters = spread(rng, 8, 4096)
        if rng.random() < 0.5:
            clusters = max(8, clusters // 8 * 8)
        n = spread(rng, 1, max(2, min(65536, 16_000_000 // clusters)))
        return gate(n, clusters, rng.randint(1, min(16, clusters // 2)), dtype,
                    rng.random() < 0.5, rng.random() < 0.4, train)
    k = rng.choice([1, 2, 4, 6, 8])
    clusters = spread(rng, max(8, k), 65536 if k == 1 else 512)
    d = spread(rng, 32, 4096)
    if rng.random() < 0.6:
        d = max(32, d // 32 * 32)
    n = spread(rng, 1, max(2, min(500000 // k, 64_000_000 // (d * k))))
    return route(op, n, clusters, k, d, dtype, train and op != "route",
                 rng.choice([0.0, 0.0, 0.02, 0.2]))


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, dtype=t, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    n = case["n"]
    if case["op"] in ("norm", "norm8"):
        d = case["d"]
        # activations: a common size with a few columns far above it
        size = torch.ones(d, device="cuda")
        size[:: max(1, d // 5)] = 12.0
        s["x"] = (torch.randn(n, d, generator=g, device="cuda") * size).to(t)
        s["residual"] = normal(n, d, scale=2.0) if case["residual"] else None
        s["weight"] = 1.0 + 0.2 * normal(d, dtype=torch.float32)
        if case.get("train"):
            s["x"].requires_grad_()
            s["weight"].requires_grad_()
            s["dy"] = normal(n, d, scale=0.1)
            s["dh"] = normal(n, d, scale=0.1) if case["residual"] else None
    elif case["op"] == "gate":
        s["scores"] = normal(n, case["clusters"])
        s["mask"] = None
        if case["masked"]:
            # about a fifth not allowed, and now and then a row (padding) with nothing allowed
            s["mask"] = torch.rand(n, case["clusters"], generator=g, device="cuda") > 0.2
            s["mask"] &= torch.rand(n, 1, generator=g, device="cuda") > 0.02
        if case["train"]:
            s["scores"].requires_grad_()
            s["dw"] = normal(n, case["k"], dtype=torch.float32)
    else:
        k, clusters, d = case["k"], case["clusters"], case["d"]
        # clusters are not used evenly
        if k == 1:
            u = torch.rand(n, 1, generator=g, device="cuda", dtype=torch.float64)
            lab = (u.pow(1.5) * clusters).long().clamp_(max=clusters - 1)
        else:
            favour = torch.linspace(1.0, 0.0, clusters, device="cuda")
            lab = (torch.randn(n, clusters, generator=g, device="cuda") + favour).topk(k, 1)[1]
        if case["dropped"]:
            lab[torch.rand(n, k, generator=g, device="cuda") < case["dropped"]] = -1
        s["labels"] = lab.to(torch.int32)
        if case["op"] in ("route", "group"):
            s["x"] = normal(n, d)
        if case["op"] in ("route", "combine"):
            s["y"] = normal(n * k, d)
            s["weights"] = torch.softmax(normal(n, k, dtype=torch.float32), 1)
        if case["train"] and case["op"] == "group":
            s["x"].requires_grad_()
            s["dxg"] = normal(n * k, d)
        if case["train"] and case["op"] == "combine":
            s["y"].requires_grad_()
            s["weights"].requires_grad_()
            s["dout"] = normal(n, d)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return run_own(s) if own else run_plain(s)


def run_own(s):
    import tensorflow_distributed_clustering_amd as tdc
    op = s["op"]
    if op == "norm":
        out = tdc.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        if s["residual"] is None:
            if not s["train"]:
                return [out]
            return [out.detach(), *torch.autograd.grad(out, (s["x"], s["weight"]), s["dy"])]
        if not s["train"]:
            return list(out)
        return [out[0].detach(), out[1].detach(),
                *torch.autograd.grad(out, (s["x"], s["weight"]), (s["dy"], s["dh"]))]
    if op == "norm8":
        out = tdc.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        if s["residual"] is None:
            return [out.dequantize(torch.bfloat16)]
        return [out[0].dequantize(torch.bfloat16), out[1]]
    if op == "gate":
        weights, labels = tdc.topk_gate(s["scores"], s["k"], mask=s["mask"], normalize=s["normalize"])
        if not s["train"]:
            return [weights, labels]
        return [weights.detach(), labels, *torch.autograd.grad(weights, s["scores"], s["dw"])]
    groups = tdc.group_plan(s["labels"], s["clusters"])
    res = [groups.offsets, groups.order, groups.pos]
    if op in ("route", "group"):
        xg = tdc.group_rows(s["x"], groups)
        res.append(xg.detach())
        if s["train"]:
            res += torch.autograd.grad(xg, s["x"], s["dxg"])
    if op in ("route", "combine"):
        out = tdc.combine_rows(s["y"], groups, s["weights"])
        res.append(out.detach())
        if s["train"]:
            res += torch.autograd.grad(out, (s["y"], s["weights"]), s["dout"])
    return res


@torch.no_grad()
def run_plain(s):
    op = s["op"]
    if op in ("norm", "norm8"):
        return plain_norm(s)
    if op == "gate":
        return plain_gate(s)
    return plain_route(s)


def plain_norm(s):
    x, r, w = s["x"], s["residual"], s["weight"]
    # the sum is kept by the caller in its own type, and the norm is the kept row's
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS)
    hat = hf * rstd
    y = hat * w
    if s["op"] == "norm8":
        n, d = y.shape
        pad = -d % 32
        b = torch.cat([y, y.new_zeros(n, pad)], 1).view(n, -1, 32) if pad else y.view(n, -1, 32)
        top = b.abs().amax(2, keepdim=True)
        # the largest value of 32 lies between 2^7 and 2^8 after its power of two is taken out
        e = torch.where(top > 0, torch.frexp(top)[1] - 8, torch.full_like(top, -127).int())
        q = torch.ldexp(b, -e).to(torch.float8_e4m3fn)
        back = torch.ldexp(q.float(), e).view(n, -1)[:, :d].to(torch.bfloat16)
        return [back] if r is None else [back, h]
    res = [y.to(x.dtype)] if r is None else [y.to(x.dtype), h]
    if s["train"]:
        dy = s["dy"].float()
        gr = dy * w
        dx = rstd * (gr - hat * (gr * hat).mean(1, keepdim=True))
        if r is not None:
            dx = dx + s["dh"].float()
        res += [dx.to(x.dtype), (dy * hat).sum(0)]
    return res


def plain_gate(s):
    k = s["k"]
    v = s["scores"].float()
    if s["mask"] is not None:
        v = torch.where(s["mask"], v, float("-inf"))
    top, at = torch.sort(v, dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    there = top > float("-inf")
    best = torch.where(there[:, :1], top[:, :1], 0.0)
    e = torch.exp(v - best)
    of = torch.exp(top - best)
    total = (of if s["normalize"] else e).sum(1, keepdim=True)
    scale = torch.where(total > 0, 1.0 / total, 0.0)
    weights = of * scale
    res = [weights, torch.where(there, at, -1).to(torch.int32)]
    if s["train"]:
        mean = (weights * s["dw"]).sum(1, keepdim=True)
        if s["normalize"]:
            ds = torch.zeros_like(v)
        else:
            ds = -(e * scale) * mean
        near = weights * (s["dw"] - mean)
        ds.scatter_(1, at, torch.where(there, near, ds.gather(1, at)))
        res.append(ds.to(s["scores"].dtype))
    return res


def plain_route(s):
    n, k, clusters = s["n"], s["k"], s["clusters"]
    lab = s["labels"].reshape(-1).long()
    key = torch.where((lab >= 0) & (lab < clusters), lab, clusters)
    sorted_key, order = torch.sort(key, stable=True)
    place = torch.arange(n * k, device=lab.device)
    pos = torch.empty_like(order)
    pos[order] = place
    offsets = torch.searchsorted(sorted_key, torch.arange(clusters + 1, device=lab.device))
    kept = (sorted_key < clusters)[:, None]       # by place
    valid = (key < clusters).view(n, k, 1)        # by slot
    pos = pos.view(n, k)
    res = [offsets.to(torch.int32), order.to(torch.int32), pos.to(torch.int32)]
    row = order // k
    if s["op"] in ("route", "group"):
        x = s["x"]
        res.append(torch.where(kept, x[row], 0.0).to(x.dtype))
        if s["train"]:
            res.append(torch.where(valid, s["dxg"][pos].float(), 0.0).sum(1).to(x.dtype))
    if s["op"] in ("route", "combine"):
        y, w = s["y"], s["weights"]
        back = torch.where(valid, y[pos].float(), 0.0)
        res.append((back * w[:, :, None]).sum(1).to(y.dtype))
        if s["train"]:
            dout = s["dout"].float()
            dy = w.reshape(-1)[order][:, None] * dout[row]
            res.append(torch.where(kept, dy, 0.0).to(y.dtype))
            res.append((back * dout[:, None]).sum(2))
    return res


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm8"):
        return exact_norm(s)
    if case["op"] == "gate":
        return exact_gate(s)
    return exact_route(s)


def exact_norm(s):
    x, r = s["x"].detach(), s["residual"]
    h = x.double() if r is None else (x.double() + r.double()).to(x.dtype).double()
    h.requires_grad_()
    w = s["weight"].detach().double().requires_grad_()
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * w
    if s["op"] == "norm8":
        back = torch.cat([e4m3_block(b) for b in y.detach().split(32, 1)], 1)
        return [back] if r is None else [back, h.detach()]
    res = [y.detach()] if r is None else [y.detach(), h.detach()]
    if s["train"]:
        dx, dw = torch.autograd.grad(y, (h, w), s["dy"].double())
        res += [dx if r is None else dx + s["dh"].double(), dw]
    return res


def e4m3_block(b):
    """Up to 32 columns to the nearest values m * 2^(e + x), m of 4 bits and x from -9 up, ties
    to the even m, where 2^(e + 7) is the largest power of two in the row's largest value."""
    top = b.abs().amax(1, keepdim=True)
    e = torch.floor(torch.log2(top)) - 7
    e = e + (torch.exp2(e + 8) <= top).double() - (torch.exp2(e + 7) > top).double()
    v = b / torch.exp2(e)
    x = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6)
    step = torch.exp2(x - 3)
    return torch.where(top > 0, torch.round(v / step) * step * torch.exp2(e), 0.0)


def exact_gate(s):
    v = s["scores"].detach().double()
    n, clusters = v.shape
    if s["mask"] is not None:
        v = v.masked_fill(~s["mask"], float("-inf"))
    left, labels = v.clone(), []
    rows = torch.arange(n, device=v.device)
    for _ in range(s["k"]):
        best = left.amax(1)
        first = torch.where(left == best[:, None], torch.arange(clusters, device=v.device), clusters).amin(1)
        labels.append(torch.where(best > float("-inf"), first, -1))
        left[rows, first] = float("-inf")
    labels = torch.stack(labels, 1)
    chosen = torch.zeros(n, clusters + 1, dtype=torch.bool, device=v.device)
    chosen.scatter_(1, torch.where(labels < 0, clusters, labels), True)
    chosen = chosen[:, :clusters]
    z = v.masked_fill(~chosen, float("-inf")) if s["normalize"] else v
    p = torch.softmax(z, 1).nan_to_num(0.0)     # a row with nothing allowed has no weights
    there = labels >= 0
    weights = torch.where(there, p.gather(1, labels.clamp(min=0)), 0.0)
    res = [weights, labels.to(torch.int32)]
    if s["train"]:
        up = torch.zeros_like(p).scatter_add_(1, labels.clamp(min=0), torch.where(there, s["dw"].double(), 0.0))
        res.append(p * up - p * (p * up).sum(1, keepdim=True))
    return res


def exact_route(s):
    n, k, clusters = s["n"], s["k"], s["clusters"]
    lab = s["labels"].cpu().numpy().reshape(-1).astype(np.int64)
    lab[(lab < 0) | (lab >= clusters)] = clusters
    order = np.argsort(lab, kind="stable")
    pos = np.empty(n * k, np.int64)
    pos[order] = np.arange(n * k)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(lab, minlength=clusters + 1)[:clusters])])
    total = int(offsets[-1])
    res = [torch.from_numpy(v.astype(np.int32)) for v in (offsets, order, pos.reshape(n, k))]
    slot = torch.from_numpy(order[:total]).cuda()
    row = torch.div(slot, k, rounding_mode="floor")

    def behind(v):
        return torch.cat([v, v.new_zeros(n * k - total, v.shape[1])])

    if s["op"] in ("route", "group"):
        x = s["x"].detach().double()
        res.append(behind(x.index_select(0, row)))
        if s["train"]:
            res.append(torch.zeros_like(x).index_add_(0, row, s["dxg"][:total].double()))
    if s["op"] in ("route", "combine"):
        y, w = s["y"].detach()[:total].double(), s["weights"].detach().double().view(-1, 1)
        res.append(torch.zeros(n, y.shape[1], dtype=torch.float64, device="cuda").index_add_(
            0, row, y * w.index_select(0, slot)))
        if s["train"]:
            dout = s["dout"].double().index_select(0, row)
            res.append(behind(dout * w.index_select(0, slot)))
            dw = torch.zeros(n * k, dtype=torch.float64, device="cuda")
            res.append(dw.index_copy_(0, slot, torch.linalg.vecdot(y, dout)).view(n, k))
    return res


# ------------------------------------------------------------------ what a pass has to do
def work(case):
    n, es = case["n"], 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("norm", "norm8"):
        d = case["d"]
        size = n * d * es
        both = 1 if case["residual"] else 0
        if case["op"] == "norm8":
            # a value of 8 bits and a scale of 8 bits for 32 of them
            return {"bytes": size * (1 + 2 * both) + n * d + n * -(-d // 32) + 4 * d, "flops": 6 * n * d}
        total = size * (2 + 2 * both) + 4 * d
        if case["train"]:
            total += size * (2 + both) + 4 * d
        return {"bytes": total, "flops": n * d * (14 if case["train"] else 5)}
    if case["op"] == "gate":
        size, k = n * case["clusters"], case["k"]
        total = size * (es + (1 if case["masked"] else 0)) + 8 * n * k
        if case["train"]:
            total += size * es + 4 * n * k
        return {"bytes": total, "flops": size * (4 + (4 if case["train"] else 0))}
    k, d = case["k"], case["d"]
    one, many = n * d * es, n * k * d * es
    total, flops = 12 * n * k + 4 * case["clusters"], 0
    if case["op"] in ("route", "group"):
        total += one + many
        if case["train"]:
            total += many + one
            flops += n * k * d
    if case["op"] in ("route", "combine"):
        total += many + 4 * n * k + one
        flops += 2 * n * k * d
        if case["train"]:
            total += one + many + 4 * n * k
            flops += 3 * n * k * d
    return {"bytes": total, "flops": flops}
