"""The router of more cells than one call of route chooses: training, and the
choice that it serves."""
import numpy as np
import pytest
import torch

import operators_oracle as orc
from garfield_amd import routed
from garfield_amd.operators import mx_dequantise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [64, 65, 256])
def test_training(P):
    """The first loss is the mean negative logarithm of the target's softmax
    score; training through a rotation lowers it."""
    print("case router of", P, flush=True)
    D, Q = 32, 512
    g = torch.Generator().manual_seed(P)
    centres = torch.nn.functional.normalize(torch.randn(P, D, generator=g), dim=1)
    target = torch.randint(0, P, (Q,), generator=g)
    turn = torch.linalg.qr(torch.randn(D, D, generator=g))[0]
    q = ((centres[target] + 0.05 * torch.randn(Q, D, generator=g)) @ turn).cuda()
    router = routed.CellRouter(centres.cuda(), temperature=0.25)
    w = mx_dequantise(router.centres).double().cpu().numpy()
    s = q.double().cpu().numpy() @ router.map.detach().double().cpu().numpy() @ w.T / 0.25
    top = s.max(1, keepdims=True)
    first = np.mean(top[:, 0] + np.log(np.exp(s - top).sum(1)) - s[np.arange(Q), target.numpy()])
    losses = router.train(q, target.cuda(), steps=40, lr=0.02)
    # scores of up to 50 in fp32 (the queries' own mapping is a fp32 product too)
    assert abs(losses[0] - first) <= 1e-3 * first
    assert losses[-1] < 0.7 * losses[0]
    r = router.route(q, torch.ones(Q, P, dtype=torch.bool, device="cuda"), 4)
    assert (r.ids.cpu() == target[:, None]).any(1).float().mean() > 0.5
    assert int(r.load.sum()) == 4 * Q and r.load.shape == (P,)


def test_search_lists():
    """search_routed passes what route chose among 256 cells to the batch."""
    print("case routed lists", flush=True)
    P, Q, D = 256, 40, 16

    class Index:
        pass

    class Batch:
        index = Index()

        def get_cells(self):
            counts = np.arange(Q, dtype=np.uint32) * 6
            cells = np.stack([np.random.default_rng(i).permutation(P) for i in range(Q)]).astype(np.uint32)
            return cells, counts, None, None

        def set_cells(self, lists, counts, little):
            self.lists, self.counts = lists, counts

        def search(self, L, K):
            return None, None, None

    Batch.index.P, Batch.Q = P, Q
    g = torch.Generator().manual_seed(1)
    router = routed.CellRouter(torch.randn(P, D, generator=g).cuda())
    b, q = Batch(), torch.randn(Q, D, generator=g).cuda()
    _, _, r = routed.search_routed(b, router, q, 12, groups=16, keep_groups=4)
    with torch.no_grad():
        from garfield_amd import mx_product, mx_quantise
        s = mx_product(mx_quantise(q @ router.map), router.centres) / router.temperature
    s = s.double().cpu().numpy()
    cells, counts, _, _ = b.get_cells()
    for i in range(Q):
        s[i, cells[i, counts[i]:]] = -np.inf
    ids, _, _ = orc.route(s, 12, groups=16, keep_groups=4)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    assert np.array_equal(b.counts, (ids >= 0).sum(1))
    for i in range(Q):
        assert b.lists[i, :b.counts[i]].tolist() == ids[i][ids[i] >= 0].tolist()
