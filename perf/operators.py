"""The routing and adapter operators of ``skmetal_amd.experts``, as cases to time.

Four kinds of pass, each through the entry points that a program calls:

===========  ======================================================================
kind         one pass
===========  ======================================================================
route        router scores to the experts of every row, their weights, the experts'
             counts and the balance loss
route_train  the same and the gradient of the scores from those of weights and loss
adapt        a shared projection's output plus the low-rank adapter of every row
adapt_train  the same and the gradients of rows, adapters and gates
===========  ======================================================================

Rows take their adapters by requests ("runs": stretches of rows with one adapter) or one
by one ("rows": skewed, as a router or cluster labels give them); some have none.
"""

from __future__ import annotations

import math

import torch

own = False  # False: the plain form below; True: the package's kernels

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MAX_ROUTE = 131_072 * 256  # n * e of a drawn case (the largest listed one)
MAX_ADAPT = 16_384 * 8_192  # n * (d + o) of a drawn case (the largest listed one)


def _route(name, kind, n, e, k, dtype, **kw):
    return dict(name=name, kind=kind, n=n, e=e, k=k, dtype=dtype, normalize=kw.get("normalize", True), padded=kw.get("padded", False),
                excluded=kw.get("excluded", False))


def _adapt(name, kind, n, d, o, r, a, dtype, law, **kw):
    return dict(name=name, kind=kind, n=n, d=d, o=o, r=r, a=a, dtype=dtype, law=law, gated=kw.get("gated", False))


def listed():
    return [
        # one generated token
        _route("route_1_e64_k2", "route", 1, 64, 2, "fp32"),
        # a decoding batch before many small experts
        _route("route_96_e256_k8", "route", 96, 256, 8, "bf16"),
        # one layer's router in a training step
        _route("route_train_16384_e64_k2", "route_train", 16_384, 64, 2, "bf16", normalize=False),
        # padded sequences, experts that some rows may not take, sizes a multiple of nothing
        _route("route_train_50003_e37_k3", "route_train", 50_003, 37, 3, "fp16", padded=True, excluded=True),
        # a large step over many small experts
        _route("route_train_131072_e256_k8", "route_train", 131_072, 256, 8, "bf16"),
        # one generated token of one request
        _adapt("adapt_1_1024_r8", "adapt", 1, 1024, 1024, 8, 16, "bf16", "rows"),
        # a decoding batch of 64 requests with adapters of their own
        _adapt("adapt_64_4096_r16", "adapt", 64, 4096, 4096, 16, 48, "bf16", "rows"),
        # rows of embeddings with an adapter per cluster, in fp32
        _adapt("adapt_5003_768_r12", "adapt", 5_003, 768, 768, 12, 50, "fp32", "rows"),
        # prompts of ragged lengths
        _adapt("adapt_8192_4096_r16", "adapt", 8_192, 4096, 4096, 16, 32, "bf16", "runs"),
        # rows and ranks that no tile divides
        _adapt("adapt_train_4099_777_r5", "adapt_train", 4_099, 777, 1001, 5, 7, "fp16", "rows", gated=True),
        # routed experts in a training step
        _adapt("adapt_train_8192_2048_r32", "adapt_train", 8_192, 2048, 2048, 32, 8, "bf16", "rows", gated=True),
        # adapters of many users trained at once
        _adapt("adapt_train_16384_4096_r64", "adapt_train", 16_384, 4096, 4096, 64, 64, "bf16", "runs"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route_train", "adapt", "adapt", "adapt_train", "adapt_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if kind.startswith("route"):
            n, e = _log(rng, 1, 131_072 if kind == "route_train" else 16_384), _log(rng, 2, 512)
            k = rng.randint(1, min(8, e))
            if n * e * (2 if dtype == "fp32" else 1) <= MAX_ROUTE:
                return dict(kind=kind, n=n, e=e, k=k, dtype=dtype, normalize=rng.random() < 0.5, padded=rng.random() < 0.3,
                            excluded=rng.random() < 0.3)
        else:
            n, d, o = _log(rng, 1, 16_384), _log(rng, 32, 4096), _log(rng, 32, 4096)
            if rng.random() < 0.7:  # widths of layers: mostly whole steps of 64
                d, o = -(-d // 64) * 64, -(-o // 64) * 64
            r, a = _log(rng, 1, 64), _log(rng, 1, 64)
            if n * (d + o) * (2 if dtype == "fp32" else 1) <= MAX_ADAPT:
                return dict(kind=kind, n=n, d=d, o=o, r=r, a=a, dtype=dtype, law=rng.choice(["runs", "rows"]), gated=rng.random() < 0.4)


# ---- inputs ----


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * (seed % 1_000_000) + 29)


def _ids(n, a, law, g):
    """The adapters of n rows: requests of exponential lengths about 256 rows, or skewed draws; one in 16 has none."""
    if law == "runs":
        m = max(1, n // 256)
        cuts = torch.empty(m, device="cuda").exponential_(generator=g).cumsum(0)
        req = torch.searchsorted((cuts / cuts[-1] * n).contiguous(), torch.arange(n, device="cuda", dtype=torch.float32), right=True).clamp_(max=m - 1)
        ids = torch.randint(0, a, (m,), device="cuda", generator=g)
        ids = torch.where(torch.rand(m, device="cuda", generator=g) < 1 / 16, -1, ids)[req]
    else:
        ids = (a * torch.rand(n, device="cuda", generator=g) ** 1.5).long().clamp_(max=a - 1)
        ids = torch.where(torch.rand(n, device="cuda", generator=g) < 1 / 16, -1, ids)
    return ids.int()


def prepare(case, seed):
    g, n, dtype = _generator(seed), case["n"], TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).to(dtype)

    state = dict(case=case)
    if case["kind"].startswith("route"):
        e, k = case["e"], case["k"]
        z = normal(n, e, std=1.5, dtype=torch.float32) + normal(1, e, std=0.5, dtype=torch.float32)  # some experts are liked more
        if case["excluded"]:
            z.masked_fill_(torch.rand(n, e, device="cuda", generator=g) < 1 / 16, -math.inf)
            z.masked_fill_(torch.rand(n, 1, device="cuda", generator=g) < 1 / 256, -math.inf)
        state["logits"] = z.to(dtype)
        at = torch.arange(n, device="cuda")
        state["mask"] = at % 512 < 512 - at // 512 * 37 % 200 if case["padded"] else None  # sequences of 512 rows, padded at their ends
        if case["kind"] == "route_train":
            state["grad_weights"] = normal(n, k, dtype=torch.float32)
            state["grad_loss"] = torch.full((), 0.01 * n, device="cuda")
        return state
    d, o, r, a = case["d"], case["o"], case["r"], case["a"]
    state["x"], state["base"] = normal(n, d), normal(n, o)
    state["down"], state["up"] = normal(a, r, d, std=1 / math.sqrt(d)), normal(a, r, o, std=1 / math.sqrt(r))
    state["scales"] = torch.rand(a, device="cuda", generator=g) + 0.5
    state["ids"] = _ids(n, a, case["law"], g)
    state["gates"] = torch.rand(n, device="cuda", generator=g) if case["gated"] else None
    if case["kind"] == "adapt_train":
        state["grad"], state["grad_base"] = normal(n, o), normal(n, d)
    return state


# ---- one pass ----


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_route(state) if kind.startswith("route") else _own_adapt(state)
    return _plain_route(state) if kind.startswith("route") else _plain_adapt(state)


def _own_route(s):
    from skmetal_amd import experts

    c = s["case"]
    r = experts.route(s["logits"], c["k"], mask=s["mask"], normalize=c["normalize"])
    out = dict(weights=r.weights, experts=r.experts, counts=r.counts, prob_sums=r.prob_sums, rows=r.rows, loss=r.loss)
    if c["kind"] == "route_train":
        out["grad_logits"] = experts.route_backward(s["logits"], r, grad_weights=s["grad_weights"], grad_loss=s["grad_loss"], mask=s["mask"],
                                                    normalize=c["normalize"])
    return out


def _own_adapt(s):
    from skmetal_amd import experts

    if s["case"]["kind"] == "adapt":
        return experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"], gates=s["gates"], scales=s["scales"])
    out, low = experts.adapt(s["x"], s["down"], s["up"], s["ids"], base=s["base"], gates=s["gates"], scales=s["scales"], return_low=True)
    grads = experts.adapt_backward(s["grad"], s["x"], s["down"], s["up"], s["ids"], low, base=s["grad_base"], gates=s["gates"], scales=s["scales"])
    return dict(out=out, grad_x=grads.x, grad_down=grads.down, grad_up=grads.up, grad_gates=grads.gates)


def _plain_route(s):
    c, z = s["case"], s["logits"].float()
    n, e, k = c["n"], c["e"], c["k"]
    live = z > -math.inf
    if s["mask"] is not None:
        live = live & s["mask"][:, None]
    live_row = live.any(1, keepdim=True)
    z = torch.where(live, z, -math.inf)
    p = torch.where(live, torch.exp(z - torch.where(live_row, z.amax(1, keepdim=True), 0.0)), 0.0)
    p = p / torch.where(live_row, p.sum(1, keepdim=True), 1.0)
    top = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    taken = live.gather(1, top)
    chosen = p.gather(1, top)
    total = torch.where(live_row, chosen.sum(1, keepdim=True), 1.0)
    weights = chosen / total if c["normalize"] else chosen
    counts = torch.zeros(e, dtype=torch.int32, device=z.device).index_add_(0, top.flatten(), taken.flatten().int())
    sums = p.sum(0)
    rows = live_row.sum(dtype=torch.int32).reshape(1)
    each = e / (k * rows.float().clamp(min=1.0).square())
    out = dict(weights=weights, experts=torch.where(taken, top, -1).int(), counts=counts, prob_sums=sums, rows=rows,
               loss=(each * (counts * sums).sum()).reshape(()))
    if c["kind"] == "route_train":
        G = (s["grad_loss"] * each * counts)[None, :]
        dz = p * (G - (p * G).sum(1, keepdim=True))
        dw = torch.where(taken, s["grad_weights"], 0.0)
        if c["normalize"]:
            dz = dz.scatter_add(1, top, weights * (dw - (weights * dw).sum(1, keepdim=True)))
        else:
            dz = dz.scatter_add(1, top, chosen * dw) - p * (chosen * dw).sum(1, keepdim=True)
        out["grad_logits"] = dz.to(s["logits"].dtype)
    return out


def _plain_adapt(s):
    c = s["case"]
    n, a, r = c["n"], c["a"], c["r"]
    x, base, down, up = s["x"].float(), s["base"].float(), s["down"].float(), s["up"].float()
    has = (s["ids"] >= 0) & (s["ids"] < a)
    ids = torch.where(has, s["ids"], 0).long()
    factor = torch.where(has, s["scales"][ids] if s["gates"] is None else s["scales"][ids] * s["gates"], 0.0)[:, None]
    train = c["kind"] == "adapt_train"
    if n * r * (c["d"] + c["o"]) <= 1 << 26:  # few rows: each with its adapter beside it
        A, B = down[ids], up[ids]
        t = (A * x[:, None, :]).sum(2)
        out = base + (B * (factor * t)[:, :, None]).sum(1)
        if train:
            dy, dxb = s["grad"].float(), s["grad_base"].float()
            u = (B * dy[:, None, :]).sum(2)
            dt = factor * u
            dx = dxb + (A * dt[:, :, None]).sum(1)
            dA = torch.zeros_like(down).index_add_(0, ids, dt[:, :, None] * x[:, None, :])
            dB = torch.zeros_like(up).index_add_(0, ids, (factor * t)[:, :, None] * dy[:, None, :])
    else:  # the rows of each adapter side by side, as many places each as the fullest has; rows without one share a last place
        key = torch.where(has, ids, a)
        order = torch.sort(key, stable=True).indices
        size = torch.zeros(a + 1, dtype=torch.long, device=x.device).index_add_(0, key, torch.ones_like(key))
        first = size.cumsum(0) - size
        rank = torch.empty_like(key).index_copy_(0, order, torch.arange(n, device=x.device) - first[key[order]])
        cap = max(1, int(size[:a].max()))
        place = torch.where(has, key * cap + rank, a * cap)

        def spread(v):
            return v.new_zeros(a * cap + 1, v.shape[1]).index_copy_(0, place, torch.where(has[:, None], v, 0.0))[:-1].view(a, cap, -1)

        def collect(v):
            return torch.cat([v.reshape(a * cap, -1), v.new_zeros(1, v.shape[2])])[place]

        X, F = spread(x), spread(factor)
        T = torch.matmul(X, down.transpose(1, 2))
        out = base + collect(torch.matmul(F * T, up))
        if train:
            dY, dxb = spread(s["grad"].float()), s["grad_base"].float()
            U = torch.matmul(dY, up.transpose(1, 2))
            dT = F * U
            dx = dxb + collect(torch.matmul(dT, down))
            dA, dB = torch.matmul(dT.transpose(1, 2), X), torch.matmul((F * T).transpose(1, 2), dY)
            t, u = collect(T), collect(U)
    if not train:
        return out.to(s["x"].dtype)
    gates = torch.where(has, s["scales"][ids] * (u * t).sum(1), 0.0) if s["gates"] is not None else None
    dtype = s["x"].dtype
    return dict(out=out.to(dtype), grad_x=dx.to(dtype), grad_down=dA.to(dtype), grad_up=dB.to(dtype), grad_gates=gates)


# ---- what a pass cannot do without ----


def work(case):
    n, size = case["n"], 4.0 if case["dtype"] == "fp32" else 2.0
    train = case["kind"].endswith("train")
    if case["kind"].startswith("route"):
        e, k = case["e"], case["k"]
        moved = size * n * e + (n if case["padded"] else 0) + 8.0 * n * k + 8.0 * e
        # exp, two sums and a product a score, comparisons for the chosen ones; as much again backward
        return dict(bytes=moved + (size * n * e + 4.0 * n * k if train else 0.0), flops=5.0 * n * e * (2 if train else 1))
    d, o, r, a = case["d"], case["o"], case["r"], case["a"]
    used = min(a, n if case["law"] == "rows" else max(1, n // 256))
    per_row = size * (d + 2 * o) + 4.0 + (4.0 if case["gated"] else 0.0)
    if not train:
        return dict(bytes=n * per_row + used * size * r * (d + o), flops=2.0 * n * r * (d + o))
    per_row += size * (o + 2 * d) + (4.0 if case["gated"] else 0.0)
    return dict(bytes=n * per_row + (used + a) * size * r * (d + o), flops=6.0 * n * r * (d + o))


# ---- the same results in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_route(s) if case["kind"].startswith("route") else _exact_adapt(s)


def _exact_route(s):
    c = s["case"]
    n, e, k = c["n"], c["e"], c["k"]
    z = s["logits"].double().cpu()
    if s["mask"] is not None:
        z[~s["mask"].cpu()] = -math.inf
    row = torch.isfinite(z).any(1)
    p = torch.zeros_like(z)
    p[row] = torch.softmax(z[row], 1)
    # ranks by value, then by place: the first k of each row with a finite score
    place = torch.argsort(-z, dim=1, stable=True)[:, :k]
    ok = torch.isfinite(torch.gather(z, 1, place))
    w = torch.gather(p, 1, place) * ok
    if c["normalize"]:
        w[row] /= w[row].sum(1, keepdim=True)
    experts = torch.where(ok, place, -1)
    counts = torch.bincount(experts[ok], minlength=e)
    N, sums = int(row.sum()), p.sum(0)
    scale = e / (k * max(N, 1) ** 2)
    out = dict(weights=w, experts=experts, counts=counts, prob_sums=sums, rows=torch.tensor([N]), loss=scale * (counts * sums).sum())
    if c["kind"] == "route_train":
        dp = (float(s["grad_loss"]) * scale * counts.double()).expand(n, e).clone()
        dw = s["grad_weights"].double().cpu() * ok
        if c["normalize"]:  # w = v / sum v
            v = torch.gather(p, 1, place) * ok
            total = v.sum(1, keepdim=True).clamp(min=1e-300)
            dw = (dw - (dw * v).sum(1, keepdim=True) / total) / total * ok
        dp.scatter_add_(1, place, dw)
        out["grad_logits"] = p * dp - p * (p * dp).sum(1, keepdim=True)
    return out


def _exact_adapt(s):
    c = s["case"]
    train = c["kind"] == "adapt_train"
    out = s["base"].double()
    if train:
        dx, dA, dB = s["grad_base"].double(), torch.zeros_like(s["down"], dtype=torch.float64), torch.zeros_like(s["up"], dtype=torch.float64)
        dg = torch.zeros(c["n"], dtype=torch.float64, device=out.device) if s["gates"] is not None else None
    for j in range(c["a"]):
        rows = torch.nonzero(s["ids"] == j).flatten()
        if not len(rows):
            continue
        A, B, x, scale = s["down"][j].double(), s["up"][j].double(), s["x"][rows].double(), float(s["scales"][j])
        gate = scale * (s["gates"][rows].double() if s["gates"] is not None else torch.ones(len(rows), dtype=torch.float64, device=x.device))
        t = x @ A.T.contiguous()
        out[rows] += gate[:, None] * (t @ B)
        if train:
            dy = s["grad"][rows].double()
            u = dy @ B.T.contiguous()
            dx[rows] += gate[:, None] * (u @ A)
            dA[j] = (gate[:, None] * u).T.contiguous() @ x
            dB[j] = (gate[:, None] * t).T.contiguous() @ dy
            if dg is not None:
                dg[rows] = scale * (t * u).sum(1)
    return dict(out=out, grad_x=dx, grad_down=dA, grad_up=dB, grad_gates=dg) if train else out
