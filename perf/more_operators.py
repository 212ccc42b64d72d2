"""Expert feed-forwards, dropout and log probabilities of ``skmetal_amd.experts``, as cases to time.

Six kinds of pass, each through the entry points that a program calls:

===========  ======================================================================
kind         one pass
===========  ======================================================================
feed         every row through the gated feed-forward block of each of its experts,
             weighted and added to the residual stream
feed_train   the same and the gradients of rows, the three matrices and the weights
rate         log probability of each row's target, entropy, and the top alternatives
rate_train   log probability and entropy, and the gradient of the scores from theirs
drop         dropout from a counter, added to the residual stream
drop_train   the same and the gradient of the rows, the mask made anew
===========  ======================================================================
"""

from __future__ import annotations

import math

import torch

own = False  # False: the plain form below; True: the package's kernels

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# What a drawn case costs at most: the largest listed one of its kind.
MAX_FEED = 16_384 * 2048 * 3 * 2048  # products of rows and matrices, a third of a training pass
MAX_MATRICES = 16 * 2048 * 3 * 4096  # elements
MAX_RATE = 4096 * 32_000
MAX_DROP = 16_384 * 4096


def _feed(name, kind, n, d, f, o, a, k, dtype, **kw):
    return dict(name=name, kind=kind, n=n, d=d, f=f, o=o, a=a, k=k, dtype=dtype, act=kw.get("act", "silu"))


def _rate(name, kind, n, v, k, dtype, **kw):
    return dict(name=name, kind=kind, n=n, v=v, k=k, dtype=dtype, excluded=kw.get("excluded", False), ignored=kw.get("ignored", False))


def _drop(name, kind, n, d, p, dtype, **kw):
    return dict(name=name, kind=kind, n=n, d=d, p=p, dtype=dtype, base=kw.get("base", False))


def listed():
    return [
        # one generated token that goes to two of eight experts
        _feed("feed_1_2048_e8_k2", "feed", 1, 2048, 1024, 2048, 8, 2, "bf16"),
        # a decoding batch of 64 requests, which between them use every expert
        _feed("feed_64_4096_e16_k2", "feed", 64, 4096, 2048, 4096, 16, 2, "bf16"),
        # a prompt through one block that all rows share
        _feed("feed_4096_2048_dense", "feed", 4096, 2048, 8192, 2048, 1, 1, "bf16", act="gelu"),
        # embeddings with an expert per cluster, trained in fp32
        _feed("feed_train_2048_512_e4", "feed_train", 2048, 512, 1024, 512, 4, 1, "fp32"),
        # widths that no tile and no load of 16 bytes divides
        _feed("feed_train_1031_777_e5_k3", "feed_train", 1031, 777, 501, 777, 5, 3, "fp16"),
        # routed experts in a training step
        _feed("feed_train_8192_2048_e8_k2", "feed_train", 8192, 2048, 2048, 2048, 8, 2, "bf16"),
        # one generated token before a large vocabulary, with its alternatives
        _rate("rate_1_131072_top5", "rate", 1, 131_072, 5, "bf16"),
        # a decoding batch, an odd vocabulary, scores that a grammar excludes
        _rate("rate_96_50257_top16", "rate", 96, 50_257, 16, "fp16", excluded=True),
        # fp32 scores of an odd vocabulary, prompts whose targets do not count
        _rate("rate_train_1999_50257", "rate_train", 1999, 50_257, 0, "fp32", ignored=True),
        # the loss of a training step
        _rate("rate_train_4096_32000", "rate_train", 4096, 32_000, 0, "bf16"),
        # the rows of a small batch before their adapters
        _drop("drop_64_1024", "drop", 64, 1024, 0.05, "bf16"),
        # the residual stream of a training step
        _drop("drop_train_16384_4096", "drop_train", 16_384, 4096, 0.1, "bf16", base=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["feed", "feed", "feed_train", "feed_train", "rate", "rate_train", "drop", "drop_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if kind.startswith("feed"):
            n, d, f, o = _log(rng, 1, 8192), _log(rng, 32, 4096), _log(rng, 32, 8192), _log(rng, 32, 4096)
            if rng.random() < 0.7:  # widths of layers: mostly whole steps of 64, and as wide behind the block as before it
                d, f = -(-d // 64) * 64, -(-f // 64) * 64
                o = d
            a = _log(rng, 1, 32)
            k = rng.randint(1, min(4, a))
            if n * k * f * (2 * d + o) <= MAX_FEED // (1 if dtype == "bf16" else 8) and a * f * (2 * d + o) <= MAX_MATRICES:
                return dict(kind=kind, n=n, d=d, f=f, o=o, a=a, k=k, dtype=dtype, act=rng.choice(["silu", "silu", "gelu", "relu"]))
        elif kind.startswith("rate"):
            n, v = _log(rng, 1, 8192), _log(rng, 16, 200_000)
            if n * v * (2 if dtype == "fp32" else 1) <= MAX_RATE:
                return dict(kind=kind, n=n, v=v, k=0 if kind == "rate_train" else rng.randint(0, 16), dtype=dtype, excluded=rng.random() < 0.3,
                            ignored=rng.random() < 0.3)
        else:
            n, d = _log(rng, 1, 16_384), _log(rng, 32, 8192)
            if n * d * (2 if dtype == "fp32" else 1) <= MAX_DROP:
                return dict(kind=kind, n=n, d=d, p=rng.choice([0.05, 0.1, 0.25, 0.5]), dtype=dtype, base=rng.random() < 0.5)


# ---- inputs ----


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1_000_003 * (seed % 1_000_000) + 31)
    n, dtype = case["n"], TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case=case)
    if case["kind"].startswith("feed"):
        d, f, o, a, k = (case[v] for v in "dfoak")
        s["x"], s["base"] = normal(n, d), normal(n, o)
        s["gate"], s["up"], s["down"] = normal(a, f, d, std=1 / math.sqrt(d)), normal(a, f, d, std=1 / math.sqrt(d)), normal(a, o, f, std=1 / math.sqrt(f))
        # some experts are liked more; one row in 32 is padding, which no expert takes
        scores = normal(1, a, std=0.5, dtype=torch.float32) - torch.log(-torch.log(uniform(n, a).clamp_(1e-7, 1 - 1e-7)))
        chosen = torch.topk(scores, k, dim=1).indices.int()
        s["chosen"] = torch.where(uniform(n, 1) < 1 / 32, -1, chosen) if n > 32 else chosen
        w = uniform(n, k) + 0.1
        s["weights"] = w / w.sum(1, keepdim=True) if k > 1 else w
        if case["kind"] == "feed_train":
            s["grad"], s["grad_base"] = normal(n, o), normal(n, d)
    elif case["kind"].startswith("rate"):
        v = case["v"]
        z = normal(n, v, std=2.0, dtype=torch.float32)
        target = torch.randint(0, v, (n,), device="cuda", generator=g)
        z.scatter_add_(1, target[:, None], 6.0 * uniform(n, 1))  # a model that has learned something
        if case["excluded"]:
            out = uniform(n, v) < 1 / 8
            out.scatter_(1, target[:, None], False)
            z.masked_fill_(out, -math.inf)
        s["logits"] = z.to(dtype)
        if case["ignored"]:
            target = torch.where(uniform(n) < 1 / 4, -100, target)
        s["targets"] = target.int()
        if case["kind"] == "rate_train":  # a policy's step: an advantage for each target, an entropy bonus
            s["grad_log_probs"], s["grad_entropy"] = normal(n, dtype=torch.float32), 0.01 * normal(n, dtype=torch.float32)
    else:
        d = case["d"]
        s["x"], s["base"] = normal(n, d), normal(n, d) if case["base"] else None
        s["key"] = torch.randint(0, 1 << 62, (2,), device="cuda", generator=g)  # the program's seed and its step
        if case["kind"] == "drop_train":
            s["grad"] = normal(n, d)
    return s


# ---- one pass ----


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own_feed(state) if kind.startswith("feed") else _own_rate(state) if kind.startswith("rate") else _own_drop(state)
    return _plain_feed(state) if kind.startswith("feed") else _plain_rate(state) if kind.startswith("rate") else _plain_drop(state)


def _own_feed(s):
    from skmetal_amd import experts

    c = s["case"]
    matrices = s["gate"], s["up"], s["down"]
    if c["kind"] == "feed":
        return experts.feed(s["x"], *matrices, s["chosen"], weights=s["weights"], base=s["base"], act=c["act"])
    out, pre = experts.feed(s["x"], *matrices, s["chosen"], weights=s["weights"], base=s["base"], act=c["act"], return_pre=True)
    g = experts.feed_backward(s["grad"], s["x"], *matrices, s["chosen"], pre, weights=s["weights"], base=s["grad_base"], act=c["act"])
    return dict(out=out, grad_x=g.x, grad_gate=g.gate, grad_up=g.up, grad_down=g.down, grad_weights=g.weights)


def _own_rate(s):
    from skmetal_amd import experts

    c = s["case"]
    r = experts.rate(s["logits"], s["targets"], top_k=c["k"])
    out = dict(log_probs=r.log_probs, entropy=r.entropy, lse=r.lse)
    if c["k"]:
        out |= dict(top=r.top, top_log_probs=r.top_log_probs)
    if c["kind"] == "rate_train":
        out["grad_logits"] = experts.rate_backward(s["logits"], s["targets"], r, grad_log_probs=s["grad_log_probs"], grad_entropy=s["grad_entropy"])
    return out


def _own_drop(s):
    from skmetal_amd import experts

    c = s["case"]
    out = experts.drop(s["x"], c["p"], s["key"], site=7, base=s["base"])
    return dict(out=out, grad_x=experts.drop(s["grad"], c["p"], s["key"], site=7)) if c["kind"] == "drop_train" else out


def _act(z, act):
    """The activation and its derivative."""
    if act == "silu":
        t = 1 / (1 + torch.exp(-z))
        return z * t, t * (1 + z * (1 - t))
    if act == "gelu":
        t = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * t, t + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0)


def _plain_feed(s):
    c = s["case"]
    n, a, k = c["n"], c["a"], c["k"]
    x, base, gate, up, down = s["x"].float(), s["base"].float(), s["gate"].float(), s["up"].float(), s["down"].float()
    # the rows of each expert side by side, as many places each as the fullest has; those without one share a last place
    chosen = s["chosen"].long().flatten()
    has = (chosen >= 0) & (chosen < a)
    key = torch.where(has, chosen, a)
    order = torch.sort(key, stable=True).indices
    size = torch.zeros(a + 1, dtype=torch.long, device=x.device).index_add_(0, key, torch.ones_like(key))
    first = size.cumsum(0) - size
    rank = torch.empty_like(key).index_copy_(0, order, torch.arange(n * k, device=x.device) - first[key[order]])
    cap = max(1, int(size[:a].max()))
    place = torch.where(has, key * cap + rank, a * cap)
    weight = s["weights"].flatten()[:, None]

    def spread(v):
        return v.new_zeros(a * cap + 1, v.shape[1]).index_copy_(0, place, torch.where(has[:, None], v, 0.0))[:-1].view(a, cap, -1)

    def collect(v):
        return torch.cat([v.reshape(a * cap, -1), v.new_zeros(1, v.shape[2])])[place]

    X, W = spread(x.repeat_interleave(k, 0)), spread(weight)
    G, U = torch.matmul(X, gate.transpose(1, 2)), torch.matmul(X, up.transpose(1, 2))
    A, dA = _act(G, c["act"])
    H = A * U
    Y = torch.matmul(H, down.transpose(1, 2))
    out = base + collect(W * Y).view(n, k, -1).sum(1)
    dtype = s["x"].dtype
    if c["kind"] == "feed":
        return out.to(dtype)
    dY = spread(s["grad"].float().repeat_interleave(k, 0))
    dH = torch.matmul(dY, down)
    dw = collect((dH * H).sum(2, keepdim=True)).view(n, k)
    dH = W * dH
    dG, dU = dH * U * dA, dH * A
    dx = s["grad_base"].float() + collect(torch.matmul(dG, gate) + torch.matmul(dU, up)).view(n, k, -1).sum(1)
    dgate, dup = torch.matmul(dG.transpose(1, 2), X), torch.matmul(dU.transpose(1, 2), X)
    ddown = torch.matmul((W * dY).transpose(1, 2), H)
    return dict(out=out.to(dtype), grad_x=dx.to(dtype), grad_gate=dgate.to(dtype), grad_up=dup.to(dtype), grad_down=ddown.to(dtype), grad_weights=dw)


def _plain_rate(s):
    c = s["case"]
    n, v, k = c["n"], c["v"], c["k"]
    z = s["logits"].float()
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    below = torch.where(e > 0, e * (z - m), 0.0).sum(1, keepdim=True)
    lse = m + torch.log(total)
    entropy = torch.log(total) - below / total
    target = s["targets"].long()[:, None]
    counts = (target >= 0) & (target < v)
    at = torch.where(counts, target, 0)
    log_probs = torch.where(counts, (z.gather(1, at) - m) - torch.log(total), 0.0)
    out = dict(log_probs=log_probs[:, 0], entropy=entropy[:, 0], lse=lse[:, 0])
    if k:
        top = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
        out |= dict(top=top.int(), top_log_probs=(z.gather(1, top) - m) - torch.log(total))
    if c["kind"] == "rate_train":
        p = e / total
        gl, ge = torch.where(counts, s["grad_log_probs"][:, None], 0.0), s["grad_entropy"][:, None]
        logp = torch.where(e > 0, (z - m) - torch.log(total), 0.0)
        dz = -p * (gl + ge * (logp + entropy))
        out["grad_logits"] = dz.scatter_add_(1, at, gl).to(s["logits"].dtype)
    return out


def _plain_drop(s):
    c = s["case"]
    n, d, p = c["n"], c["d"], c["p"]
    keep = _words(n * d, s["key"], 7).view(n, d) >= round(p * 2**32)

    def dropped(x):
        return torch.where(keep, x.float() * (1 / (1 - p)), 0.0)

    out = dropped(s["x"])
    if s["base"] is not None:
        out = out + s["base"].float()
    dtype = s["x"].dtype
    return dict(out=out.to(dtype), grad_x=dropped(s["grad"]).to(dtype)) if c["kind"] == "drop_train" else out.to(dtype)


def _words(count, key, site):
    """`count` words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): four for each counter (index / 4, site, step), as int64."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 3) // 4, device=key.device)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, site), (key[1] & low).expand_as(block)
    k0, k1 = key[0] & low, (key[0] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 32 x 32 bits: the low 64 are right, whichever sign they show
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).flatten()[:count]


# ---- what a pass cannot do without ----


def work(case):
    n, size = case["n"], 4.0 if case["dtype"] == "fp32" else 2.0
    train = case["kind"].endswith("train")
    if case["kind"].startswith("feed"):
        d, f, o, a, k = (case[v] for v in "dfoak")
        matrices = min(a, n * k) * f * (2 * d + o)
        moved = size * n * (d + 2 * o) + 8.0 * n * k + size * matrices
        if train:  # out's gradient, x's base, x's gradient and those of all matrices
            moved += size * n * (o + 2 * d) + 4.0 * n * k + size * a * f * (2 * d + o)
        return dict(bytes=moved, flops=2.0 * n * k * f * (2 * d + o) * (3 if train else 1))
    if case["kind"].startswith("rate"):
        v, k = case["v"], case["k"]
        # exp, the sums of exp and of its product, their product; as much again backward
        return dict(bytes=size * n * v * (2 if train else 1) + 16.0 * n + 8.0 * n * k + (8.0 * n if train else 0.0), flops=6.0 * n * v * (2 if train else 1))
    d = case["d"]
    moved = size * n * d * (2 + (1 if case["base"] else 0) + (2 if train else 0))
    # ten rounds of two products, four exclusive ors and two sums for four elements
    return dict(bytes=moved + 16.0, flops=20.0 * n * d * (2 if train else 1))


# ---- the same results in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_feed(s) if case["kind"].startswith("feed") else _exact_rate(s) if case["kind"].startswith("rate") else _exact_drop(s)


def _exact_feed(s):
    c = s["case"]
    train = c["kind"] == "feed_train"
    out = s["base"].double()
    if train:
        dx, dw = s["grad_base"].double(), torch.zeros(s["weights"].shape, dtype=torch.float64, device=out.device)
        dmat = [torch.zeros(s[v].shape, dtype=torch.float64, device=out.device) for v in ("gate", "up", "down")]
    for q in range(c["a"]):
        rows, places = torch.nonzero(s["chosen"] == q, as_tuple=True)
        if not len(rows):
            continue
        P, Q, R = (s[v][q].double() for v in ("gate", "up", "down"))
        x, w = s["x"][rows].double(), s["weights"][rows, places].double()[:, None]
        g, u = x @ P.T.contiguous(), x @ Q.T.contiguous()
        g.requires_grad_(train)
        f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[c["act"]](g)
        act = f.detach()
        out.index_add_(0, rows, w * ((act * u) @ R.T.contiguous()))
        if train:
            dy = s["grad"][rows].double()
            dh = dy @ R
            dw[rows, places] = (dh * act * u).sum(1)
            (dg,) = torch.autograd.grad(f, g, w * dh * u)
            du = w * dh * act
            dx.index_add_(0, rows, dg @ P + du @ Q)
            dmat[0][q], dmat[1][q] = dg.T.contiguous() @ x, du.T.contiguous() @ x
            dmat[2][q] = (w * dy).T.contiguous() @ (act * u)
    return dict(out=out, grad_x=dx, grad_gate=dmat[0], grad_up=dmat[1], grad_down=dmat[2], grad_weights=dw) if train else out


def _exact_rate(s):
    c = s["case"]
    lp = torch.log_softmax(s["logits"].double(), 1)
    p = lp.exp()
    plp = torch.nan_to_num(p * lp, nan=0.0)  # 0 where the probability is
    entropy = -plp.sum(1)
    rows = torch.nonzero((s["targets"] >= 0) & (s["targets"] < c["v"])).flatten()
    at = s["targets"][rows].long()
    log_probs = torch.zeros_like(entropy)
    log_probs[rows] = lp[rows, at]
    out = dict(log_probs=log_probs, entropy=entropy, lse=torch.logsumexp(s["logits"].double(), 1))
    if c["k"]:
        top = torch.argsort(-s["logits"].double(), dim=1, stable=True)[:, : c["k"]]
        out |= dict(top=top, top_log_probs=torch.gather(lp, 1, top))
    if c["kind"] == "rate_train":
        gl, ge = torch.zeros_like(entropy), s["grad_entropy"].double()
        gl[rows] = s["grad_log_probs"].double()[rows]
        dz = -p * gl[:, None] - ge[:, None] * (plp + p * entropy[:, None])
        dz[rows, at] += gl[rows]
        out["grad_logits"] = dz
    return out


def _exact_drop(s):
    import numpy as np

    c = s["case"]
    n, d, p = c["n"], c["d"], c["p"]
    seed, step = (int(v) for v in s["key"].tolist())
    low, bits = np.uint64(0xFFFFFFFF), np.uint64(32)
    i = np.arange(-(-n * d // 4), dtype=np.uint64)
    w = [i & low, i >> bits, np.full_like(i, 7), np.full_like(i, step & 0xFFFFFFFF)]
    for r in range(10):
        k0, k1 = np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(b >> bits) ^ w[1] ^ k0, b & low, (a >> bits) ^ w[3] ^ k1, a & low]
    keep = np.stack(w, 1).reshape(-1)[: n * d].reshape(n, d) >= round(p * 2**32)
    factor = torch.from_numpy(keep).to(s["x"].device).double() / (1 - p)
    out = factor * s["x"].double()
    if s["base"] is not None:
        out += s["base"].double()
    return dict(out=out, grad_x=factor * s["grad"].double()) if c["kind"] == "drop_train" else out
