"""Beam search's kernels (csrc/beam_*.cu) and searches on the GPU at their edges: scores in 64 bits and chains of selections."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from beam_edges import LastTokenModel, best_chains
from plain import beam_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("G,held,B,V,pad,stops", [(1, 1, 4, 151936, 0, ()), (3, 4, 4, 5000, 0, (7, 20)), (2, 5, 6, 3001, 2, ()), (2, 32, 32, 33000, 1, (5,)),
                                                  (1, 3, 3, 2, 0, (1,))])
def test_select_with_scores_in_64_bits(G, held, B, V, pad, stops):
    """Scores apart by less than 32 bits tell: 1e-6 at -5,000.  A total is off by the row's sum, whose terms are off by 4e-11 at most, and by
    a few roundings of 2^-53 of what is added up."""
    from toyinfer_b200.kernels import beam as KB
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (torch.randn(G * held, V + pad, generator=g, device=DEV) * 2.5)[:, :V]
    x[:] = x[::held].repeat_interleave(held, 0) if held > 1 else x           # equal rows: the scores decide
    s = -5000 + torch.randperm(G * held, generator=g, device=DEV).double().view(G, held) * 1e-6
    if held > 2:
        s[0, 1], s[-1, 0] = -float("inf"), float("nan")
    ids = torch.tensor(list(stops), dtype=torch.int32, device=DEV) if stops else None
    got = KB.select(x, s, B, ids, wide=True)
    want = plain.select(x.cpu().numpy(), s.cpu().numpy(), B, stops)
    assert got.scores.dtype == got.ended_scores.dtype == torch.float64
    for i, (a, b) in enumerate(zip(got, want)):
        a, b = a.cpu(), torch.from_numpy(np.asarray(b))
        if i in (0, 3):
            f = torch.isfinite(b)
            assert torch.equal(a[~f], b[~f])
            assert ((a[f] - b[f]).abs() <= 5e-11 + 2 ** -50 * b[f].abs()).all()
        else:
            assert a.dtype == torch.int32 and torch.equal(a.long(), b)
    narrow = KB.select(x, s.float(), B, ids)
    assert narrow.scores.dtype == narrow.ended_scores.dtype == torch.float32


def test_two_thousand_selections_in_a_row():
    """Running scores handed on as they come: each selection is the plain one's from the same scores, and at -7,400, where a step of 32 bits
    is 5e-4 and beams are about 1e-3 apart, the scores are still their tokens' sums: 5e-11 and one rounding of 2^-41 a selection."""
    from toyinfer_b200.kernels import beam as KB
    V, B, n = 40, 4, 2000
    pool = torch.randn(64, B, V, generator=torch.Generator().manual_seed(1)) * 1e-3
    on_gpu = pool.to(DEV)
    true = np.zeros((1, 1))
    scores = torch.zeros(1, 1, dtype=torch.float64, device=DEV)
    for k in range(n):
        held = scores.shape[1]
        rows = pool[k % 64, :held]
        got = KB.select(on_gpu[k % 64, :held].contiguous(), scores, B, wide=True)
        parents, tokens = got.parents[0].tolist(), got.tokens[0].tolist()
        want = plain.select(rows.numpy(), scores.cpu().numpy(), B)
        assert parents == want[1][0].tolist() and tokens == want[2][0].tolist(), k
        lp = [plain.log_probs(r) for r in rows.numpy()]
        true = np.array([[true[0, p] + lp[p][t] for p, t in zip(parents, tokens)]])
        scores = got.scores
        assert np.abs(scores.cpu().numpy() - true).max() <= (k + 1) * (5e-11 + 2 * 2 ** -41), k
    assert true.max() < -7000


def test_scores_of_a_long_search_are_sums_in_64_bits():
    """As the test of this name without a device, by the kernel, whose rows' sums are off by 5e-11 a step."""
    from toyinfer_b200 import BeamParams
    from toyinfer_b200.engine.beam import BeamLoop, BeamStepper
    V, n, B = 40, 1500, 4
    table = torch.randn(V, V, generator=torch.Generator().manual_seed(0)) * 1e-3
    params = BeamParams(B, n_best=B)
    loop = BeamLoop(BeamStepper(LastTokenModel(table.to(DEV)), params, []), params, [], 8, 1 << 20, 1 << 20)
    got = loop.run([[3]], n)[0]
    lp, live = best_chains(table, 3, B, n)
    for h, (score, tokens) in zip(got, live):
        path = [3] + h.tokens
        assert abs(h.score - sum(lp[a, b] for a, b in zip(path, path[1:]))) <= n * 5e-11 + 1e-8
        assert abs(h.score - score) <= n * 5e-11 + 1e-8 and h.tokens == tokens[1:]


def test_select_refuses_scores_of_other_types():
    from toyinfer_b200.kernels import KernelError
    from toyinfer_b200.kernels import beam as KB
    x = torch.zeros(4, 10, device=DEV)
    wide = torch.zeros(2, 4, dtype=torch.float64, device=DEV)
    for s, w in ((wide[:, :2].contiguous(), False), (wide[:, :2].contiguous().float(), True), (wide[:, ::2], True),
                 (wide[:, :2].contiguous().half(), True)):
        with pytest.raises(KernelError, match="scores"):
            KB.select(x, s, 2, wide=w)
