"""Trains a GCN with learned node rows on a batch of synthetic graphs:

    python -m tcc_amd.train_embeddings --graphs 200 --nodes 50000 --steps 20

Every graph is a random subset of the nodes of one table with R-MAT edges
among them, and its nodes' labels follow two hidden classes of the table, so
that only the embeddings can tell them apart.  Prints the loss and the gradient
norm of every step.
"""
from __future__ import annotations

import argparse

import torch

from . import gcn
from .graphs import rmat_graph


def batch_of_graphs(num_nodes: int, graphs: int, mean_rows: int, seed: int):
    """(rows, cols, ids, offsets, max_rows): the block-diagonal edges of
    `graphs` graphs of uneven size, the node id of every row, the graphs' first
    rows (int32) and the longest one's rows."""
    g = torch.Generator().manual_seed(seed)
    sizes = torch.randint(max(2, mean_rows // 4), 2 * mean_rows, (graphs,), generator=g)
    first = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    rows, cols = [], []
    for k in range(graphs):
        n = int(sizes[k])
        r, c = rmat_graph(n, min(4 * n, n * n // 2), seed + 1 + k)
        rows.append(r + first[k])
        cols.append(c + first[k])
    ids = torch.randint(0, num_nodes, (int(first[-1]),), generator=g)
    return torch.cat(rows), torch.cat(cols), ids, first.to(torch.int32), int(sizes.max())


def train(nodes: int = 50_000, graphs: int = 200, mean_rows: int = 60, dim: int = 64, hidden: int = 128, steps: int = 20,
          lr: float = 1e-2, max_norm: float = 1.0, seed: int = 0, log=print):
    """The losses and gradient norms of `steps` steps, and the model."""
    torch.manual_seed(seed)
    rows, cols, ids, offsets, max_rows = batch_of_graphs(nodes, graphs, mean_rows, seed)
    n = ids.numel()
    graph = gcn.LayerGraph(rows, cols, n, n)
    labels = (ids % 2).cuda()
    ids, offsets = ids.cuda(), offsets.cuda()
    model = gcn.EmbeddingGCN(nodes, dim, hidden, 2)
    optimizer = gcn.ClippedAdam(model.parameters(), lr=lr, max_norm=max_norm)
    losses, norms = [], []
    for step in range(steps):
        loss, norm = gcn.train_embedding_epoch(model, graph, ids, labels, optimizer, offsets, max_rows)
        losses.append(float(loss))
        norms.append(float(norm))
        log(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norms[-1]:.3f}")
    if model.embedding.error():
        raise RuntimeError("a node id lies outside the embedding table")
    return losses, norms, model


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--nodes", type=int, default=50_000)
    p.add_argument("--graphs", type=int, default=200)
    p.add_argument("--mean-rows", type=int, default=60)
    p.add_argument("--dim", type=int, default=64)
    p.add_argument("--hidden", type=int, default=128)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--lr", type=float, default=1e-2)
    p.add_argument("--max-norm", type=float, default=1.0)
    a = p.parse_args(argv)
    train(a.nodes, a.graphs, a.mean_rows, a.dim, a.hidden, a.steps, a.lr, a.max_norm,
          log=lambda s: print(s, flush=True))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
