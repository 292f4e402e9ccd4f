"""A learned router over the cells of an index: trained through the frozen
4-bit centres, then used to search (garfield_amd/routed.py)."""
import numpy as np
import pytest
import torch

import operators_oracle as orc
from garfield_amd import routed, synth

pytestmark = pytest.mark.gpu


def test_router_learns_and_searches():
    print("case routed demo", flush=True)
    out = routed.demo(N=8000, Q=256, steps=60)
    # the loss of a uniform choice among 16 cells is log 16 = 2.77; the queries
    # come rotated, so the untrained map is no better than that
    assert out["losses"][0] > 2.0 and out["losses"][-1] < 0.5 * out["losses"][0]
    assert out["recall"][1] <= out["recall"][2] <= out["recall"][4]
    assert out["recall"][4] > 0.8


def test_routed_cells_stay_in_range():
    """Routed cells are cells of the query's range, at most k of them, in at
    most keep_groups groups; a query whose range holds no cell finds nothing."""
    print("case routed cells", flush=True)
    P = 16
    vec, comp = synth.gmm_vectors(6000, 64, 64, 11)
    att = synth.component_attrs(comp, 1, 12)
    ix = synth.build_index(vec, att, [P], 16, 2, device="hip")
    dev = synth.open_device_index(ix)
    Q = 100
    lo, hi = synth.ranges_for_selectivity(Q, 1, 0.4, 13, hi=int(att.max()) + 1)
    lo[0], hi[0] = 5, 4                      # empty
    lo[1], hi[1] = -20, -10                  # beyond the attribute's values
    q = vec[:Q]
    b = dev.batch(q, lo.astype(np.float32), hi.astype(np.float32))
    b.mark_cells(1.0)
    cells, counts, _, _ = b.get_cells()
    router = routed.CellRouter(routed.cell_means(vec, ix["global_pid"], P))
    ids, dists, r = routed.search_routed(b, router, torch.from_numpy(q).cuda(), 3, groups=8, keep_groups=2)
    chosen = r.ids.cpu().numpy()
    gpid = np.asarray(ix["global_pid"])
    for i in range(Q):
        allowed = set(cells[i, :counts[i]])
        mine = [c for c in chosen[i] if c >= 0]
        assert set(mine) <= allowed and len({c // 2 for c in mine}) <= 2
        assert len(mine) == len(set(mine))
        got = ids[i][ids[i] != 0x7FFFFFFF]
        assert set(gpid[got.astype(np.int64)]) <= set(mine)
        assert all(lo[i, 0] <= att[p, 0] <= hi[i, 0] for p in got.astype(np.int64))
    assert (ids[0] == 0x7FFFFFFF).all() and (ids[1] == 0x7FFFFFFF).all()
    # what it chose is what the definition gives for the masked scores
    with torch.no_grad():
        from garfield_amd import mx_product, mx_quantise
        s = mx_product(mx_quantise(torch.from_numpy(q).cuda() @ router.map), router.centres) / router.temperature
    s = s.double().cpu().numpy()
    for i in range(Q):
        s[i, [c for c in range(P) if c not in set(cells[i, :counts[i]])]] = -np.inf
    want, _, _ = orc.route(s, 3, groups=8, keep_groups=2)
    assert np.array_equal(chosen, want)
    b.close()
    dev.close()
