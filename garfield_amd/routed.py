"""Searches over cells that a learned router chooses.

Stage B of the search orders a query's cells by the nearest cluster centres,
which are given.  Here the choice is learned: a linear map in front of the
cells' mean vectors, held at four bits, scores the cells of a query; ``route``
keeps the k best of those that the query's range allows, and the search visits
these alone (``Batch.set_cells``).

- training: ``mx_product`` of the mapped queries with the centres, ``route``'s
  softmax weights (of more than 64 cells, which ``route`` does not choose at
  once, the cross entropy of the scores), and their gradients
  (``mx_product_grad``, ``route_grad`` behind autograd) through the frozen
  centres to the map;
- serving: the mapped queries quantised (``mx_quantise``), both sides at four
  bits, cells outside a range masked, at most ``keep_groups`` of ``groups`` runs
  of cells (shards) a query.

``python -m garfield_amd.routed`` trains one on a synthetic index and searches
with it.
"""
import math

import numpy as np

from . import operators as ops


class CellRouter:
    """Scores of P cells, at most 1024, for D-dimensional queries: (q @ map) . centre / temperature."""

    def __init__(self, centres, temperature=0.1, seed=0):
        """centres: (P, D) mean vectors of the cells, on the GPU; kept at four bits."""
        import torch
        self.centres = ops.mx_quantise(centres)
        self.temperature = float(temperature)
        g = torch.Generator().manual_seed(seed)
        d = centres.shape[1]
        # near the identity: untrained, the cells with the nearest centres
        start = torch.eye(d) + 0.1 / math.sqrt(d) * torch.randn(d, d, generator=g)
        self.map = start.to(centres.device).requires_grad_()

    def train(self, queries, target, steps=100, lr=0.01):
        """Moves the map so that the softmax weight of each query's target cell
        grows; returns the loss (mean negative log weight) of every step."""
        import torch
        opt = torch.optim.Adam([self.map], lr=lr)
        losses = []
        for _ in range(steps):
            logits = ops.mx_product(queries @ self.map, self.centres) / self.temperature
            if self.centres.rows <= ops.MAX_CHOICES:
                r = ops.route(logits, self.centres.rows)   # all cells, best first
                weight = torch.where(r.ids == target[:, None], r.weights, 0).sum(1)
                loss = -weight.clamp_min(1e-20).log().mean()
            else:                                          # a target need not be among the best
                loss = torch.nn.functional.cross_entropy(logits, target)
            opt.zero_grad(set_to_none=True)
            loss.backward()
            opt.step()
            losses.append(loss.detach())
        return [float(v) for v in losses]

    def route(self, queries, allowed, k, groups=1, keep_groups=None):
        """The k best cells of each query among those allowed ((Q, P) truth
        values), with their weights; ids -1 where a query has fewer."""
        import torch
        with torch.no_grad():
            logits = ops.mx_product(ops.mx_quantise(queries @ self.map), self.centres) / self.temperature
            return ops.route(logits.masked_fill(~allowed, -math.inf), k, groups=groups, keep_groups=keep_groups)


def search_routed(batch, router, queries, k, K=10, groups=1, keep_groups=None):
    """The exact K nearest in range over each query's k routed cells: stage A's
    cell lists of the batch, masked scores, the chosen cells as the new lists.
    queries: the batch's, on the GPU.  Returns (ids, dists, Routes)."""
    import torch
    P = batch.index.P
    cells, counts, _, _ = batch.get_cells()
    allowed = np.zeros((batch.Q, P), bool)
    listed = np.arange(P)[None] < counts[:, None]
    allowed[np.nonzero(listed)[0], cells[listed]] = True
    r = router.route(queries, torch.from_numpy(allowed).to(queries.device), k, groups, keep_groups)
    ids = r.ids.cpu().numpy()
    found = (ids >= 0).sum(1).astype(np.uint32)            # a row's -1 come last
    lists = np.zeros((batch.Q, P), np.uint32)
    lists[:, :k] = np.maximum(ids, 0)
    batch.set_cells(lists, found, found)                   # every cell by brute force: exact
    out, dists, _ = batch.search(L=64, K=K)
    return out, dists, r


def cell_means(vectors, cell_of, P):
    """Mean vector of each cell (zeros for an empty one), on the GPU."""
    import torch
    v = torch.from_numpy(np.ascontiguousarray(vectors, np.float32)).cuda()
    c = torch.from_numpy(np.asarray(cell_of, np.int64)).cuda()
    total = torch.zeros(P, v.shape[1], device=v.device).index_add_(0, c, v)
    return total / torch.bincount(c, minlength=P).clamp(min=1)[:, None]


def demo(N=20000, D=96, P=16, Q=512, steps=60, seed=3, log=print):
    """A mixture of Gaussians whose component decides a point's attribute and so
    its cell; queries through a fixed random rotation, as from an encoder that
    the index was not built with.  Returns what it measured."""
    import torch

    from . import synth
    rng = np.random.default_rng(seed)
    vec, comp = synth.gmm_vectors(N, D, 4 * P, seed)
    att = synth.component_attrs(comp, 1, seed + 1)
    ix = synth.build_index(vec, att, [P], 16, 2, device="hip")
    dev = synth.open_device_index(ix)
    # the encoder's space: a rotation of the index's
    turn = np.linalg.qr(rng.standard_normal((D, D)))[0].astype(np.float32)
    near = vec[rng.integers(0, N, 2 * Q)] + 0.05 * rng.standard_normal((2 * Q, D)).astype(np.float32)
    everything = np.zeros((Q, 1), np.float32), np.full((Q, 1), att.max(), np.float32)
    # training targets: the cell of each query's nearest neighbour
    b = dev.batch(near[:Q], *everything)
    b.mark_cells(1.0)
    nearest, _, _ = b.search(L=64, K=1)
    b.close()
    gpid = np.asarray(ix["global_pid"], np.int64)
    target = torch.from_numpy(gpid[nearest[:, 0].astype(np.int64)]).cuda()
    router = CellRouter(cell_means(vec, gpid, P))
    losses = router.train(torch.from_numpy(near[:Q] @ turn).cuda(), target, steps=steps)
    # searches of the other half, half of the attribute's range each
    lo, hi = synth.ranges_for_selectivity(Q, 1, 0.5, seed + 2, hi=int(att.max()) + 1)
    q = torch.from_numpy(near[Q:] @ turn).cuda()
    b = dev.batch(near[Q:], lo.astype(np.float32), hi.astype(np.float32))
    b.mark_cells(1.0)
    full, _, _ = b.search(L=64, K=10)
    recall = {}
    for k in (1, 2, 4):
        b.mark_cells(1.0)
        got, _, r = search_routed(b, router, q, k, groups=4, keep_groups=2)
        recall[k] = float(np.mean([len(set(a[a != ops._lib.NO_RESULT]) & set(g[g != ops._lib.NO_RESULT]))
                                   / max(1, (g != ops._lib.NO_RESULT).sum()) for a, g in zip(got, full)]))
    b.close()
    dev.close()
    log(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}; recall@10 of 1, 2, 4 of {P} cells: "
        + ", ".join(f"{recall[k]:.3f}" for k in (1, 2, 4)), flush=True)
    return dict(losses=losses, recall=recall)


if __name__ == "__main__":
    demo()
