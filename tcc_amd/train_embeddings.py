"""Trains a GCN with learned node rows on a batch of synthetic graphs:

    python -m tcc_amd.train_embeddings --graphs 200 --nodes 50000 --steps 20
    python -m tcc_amd.train_embeddings --norm layer --blocks 2 --distill 4

Every graph is a random subset of the nodes of one table with R-MAT edges
among them, and its nodes' labels follow hidden classes of the table (two, 3 K with
--distill K, or --classes), so that only the embeddings can tell them apart.  Prints
the loss and the gradient norm of every step.  With --norm layer the model has layer
norms and --blocks residual ones; with --distill K a model of one quarter of its
widths then learns from its K largest logits of every node.
"""
from __future__ import annotations

import argparse

import torch

from . import gcn, training
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


def checked(norm: str, blocks: int, classes: int | None, distill: int, temperature: float) -> int:
    """How many classes there are; ValueError for what the model or the student
    would refuse when their turn comes."""
    if blocks < 0 or (blocks > 0 and norm != "layer"):
        raise ValueError("residual blocks go with layer norms")
    if distill < 0:
        raise ValueError(f"a student learns from one logit of a node or more (got {distill})")
    if classes is None:
        classes = max(2, 3 * distill)
    if classes < 1:
        raise ValueError(f"there is one class at least (got {classes})")
    if distill > min(classes, 64):
        raise ValueError(f"the {distill} largest of {classes} logits: at most as many as there are classes, and 64")
    if distill and not 1e-18 <= temperature <= 1e18:
        raise ValueError(f"the temperature lies between 1e-18 and 1e18 (got {temperature})")
    return classes


def train(nodes: int = 50_000, graphs: int = 200, mean_rows: int = 60, dim: int = 64, hidden: int = 128, steps: int = 20,
          lr: float = 1e-2, max_norm: float = 1.0, seed: int = 0, log=print, norm: str = "group", blocks: int = 0,
          classes: int | None = None, distill: int = 0, temperature: float = 2.0):
    """The losses and gradient norms of `steps` steps, and the model; with
    `distill`, those of the student that learns from its `distill` largest logits,
    and the student."""
    classes = checked(norm, blocks, classes, distill, temperature)
    torch.manual_seed(seed)
    rows, cols, ids, offsets, max_rows = batch_of_graphs(nodes, graphs, mean_rows, seed)
    n = ids.numel()
    graph = gcn.LayerGraph(rows, cols, n, n)
    labels = (ids % classes).cuda()
    ids, offsets = ids.cuda(), offsets.cuda()

    def run(model, targets, loss_fcn, name):
        optimizer = gcn.ClippedAdam(model.parameters(), lr=lr, max_norm=max_norm)
        losses, norms = [], []
        for step in range(steps):
            loss, total = gcn.train_embedding_epoch(model, graph, ids, targets, optimizer, offsets, max_rows, loss_fcn)
            losses.append(float(loss))
            norms.append(float(total))
            log(f"{name}step {step}: loss {losses[-1]:.4f}, gradient norm {norms[-1]:.3f}")
        if model.embedding.error():
            raise RuntimeError("a node id lies outside the embedding table")
        return losses, norms, model

    teacher = run(gcn.EmbeddingGCN(nodes, dim, hidden, classes, norm=norm, blocks=blocks), labels, gcn.cross_entropy, "")
    if distill == 0:
        return teacher
    with torch.no_grad():
        entries = training.top_logits(teacher[2](graph, ids, offsets, max_rows), distill, temperature=temperature)
    small = [max(8, w // 4 // 8 * 8) for w in (dim, hidden)]  # 8 groups, where they are asked for
    return run(gcn.EmbeddingGCN(nodes, *small, classes, norm=norm), entries, gcn.DistillationLoss(temperature), "student: ")


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
    p.add_argument("--norm", choices=("group", "layer"), default="group")
    p.add_argument("--blocks", type=int, default=0, help="residual blocks (with --norm layer)")
    p.add_argument("--classes", type=int, help="2 by default, 3 K with --distill K")
    p.add_argument("--distill", type=int, default=0, metavar="K", help="train a student from the K largest logits")
    p.add_argument("--temperature", type=float, default=2.0)
    a = p.parse_args(argv)
    try:
        checked(a.norm, a.blocks, a.classes, a.distill, a.temperature)
    except ValueError as e:
        p.error(str(e))
    train(a.nodes, a.graphs, a.mean_rows, a.dim, a.hidden, a.steps, a.lr, a.max_norm,
          log=lambda s: print(s, flush=True), norm=a.norm, blocks=a.blocks, classes=a.classes, distill=a.distill,
          temperature=a.temperature)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
