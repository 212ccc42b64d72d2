"""Experts placed at the centres of a KMeans fit: train their adapters, then serve them.

Rows of embeddings are clustered on the GPU, the router scores a row by its product with
every centre, and each cluster's expert is a low-rank adapter beside a projection that
all rows share.  Training steps route the rows with the balance loss and pass them
through their experts; a served row takes the same calls without gradients.

    python examples/cluster_experts.py [--rows N] [--width D] [--experts E] [--steps S]
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import skmetal_amd as skmetal  # noqa: E402
from skmetal_amd import experts  # noqa: E402


def embeddings(rows, width, clusters, seed=0):
    """Unit rows around `clusters` directions, and targets that differ by cluster."""
    g = torch.Generator().manual_seed(seed)
    centre = torch.nn.functional.normalize(torch.randn(clusters, width, generator=g), dim=1)
    label = torch.randint(0, clusters, (rows,), generator=g)
    x = torch.nn.functional.normalize(centre[label] + 0.3 / math.sqrt(width) * torch.randn(rows, width, generator=g), dim=1)
    shift = torch.randn(clusters, 4, width, generator=g) / math.sqrt(width)
    out = torch.randn(clusters, 4, width, generator=g)
    return x, x + torch.einsum("nrd,nd,nro->no", shift[label], x, out[label]) / 2


class Experts(torch.nn.Module):
    """A shared projection, a router that starts at given centres, an adapter per centre."""

    def __init__(self, centres, width, rank, top_k, dtype=torch.bfloat16):
        super().__init__()
        e = centres.shape[0]
        self.top_k = top_k
        self.router = torch.nn.Parameter(centres.clone())                     # [e, d] fp32
        self.shared = torch.nn.Linear(width, width, bias=False, device="cuda", dtype=dtype)
        self.down = torch.nn.Parameter((torch.randn(e, rank, width, device="cuda") / math.sqrt(width)).to(dtype))
        self.up = torch.nn.Parameter(torch.zeros(e, rank, width, device="cuda", dtype=dtype))

    def forward(self, x):
        q = experts.routed(8.0 * (x.float() @ self.router.T), self.top_k, normalize=True)
        y = self.shared(x)
        for t in range(self.top_k):
            y = experts.adapted(x, self.down, self.up, q.experts[:, t], base=y, gates=q.weights[:, t])
        return y, q

    @torch.no_grad()
    def serve(self, x):
        """The same for rows that need no gradient, down to a single one."""
        q = experts.route(8.0 * (x.float() @ self.router.T), self.top_k, normalize=True)
        y = self.shared(x)
        for t in range(self.top_k):
            experts.adapt(x, self.down, self.up, q.experts[:, t], base=y, gates=q.weights[:, t], out=y)
        return y


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=16_384)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--experts", type=int, default=32)
    ap.add_argument("--steps", type=int, default=60)
    args = ap.parse_args(argv)
    from sklearn.cluster import KMeans

    x, target = embeddings(args.rows, args.width, args.experts)
    model = skmetal.accelerate(KMeans(n_clusters=args.experts, n_init=1, random_state=0)).fit(x.numpy())
    torch.manual_seed(1)
    net = Experts(torch.from_numpy(model.cluster_centers_).cuda(), args.width, rank=8, top_k=2)
    opt = torch.optim.Adam(net.parameters(), lr=3e-3)
    x, target = x.cuda().bfloat16(), target.cuda()
    losses = []
    for step in range(args.steps):
        y, q = net(x)
        fit = (y.float() - target).square().mean()
        loss = fit + 0.01 * q.loss
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(fit.item())
        if step % 20 == 0 or step == args.steps - 1:
            print(f"step {step}: loss {losses[-1]:.4f}, balance {q.loss.item():.3f}, rows of the busiest expert {int(q.counts.max())}")
    one = net.serve(x[:1])
    print(f"one row served: off its target by {(one.float() - target[:1]).square().mean().item():.4f}")
    return losses, net, x


if __name__ == "__main__":
    main()
