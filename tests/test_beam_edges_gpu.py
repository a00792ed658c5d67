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


def groups_with_homes(G, B, width, length, seed):
    """Slots, homes (a page of its own per place and column), tables as a search leaves them, and parents with places that move."""
    rng = np.random.RandomState(seed)
    slots = rng.permutation(G * B + 1)[:G * B].reshape(G, B).astype(np.int32)
    home = np.zeros((G * B + 2, width), dtype=np.int32)
    home[:-1] = 1 + rng.permutation((G * B + 1) * width).reshape(-1, width)
    table = home.copy()
    for g in range(G):
        for c in range(width):
            pick = rng.permutation(B) if c == length // 64 else rng.randint(0, B, B)
            table[slots[g], c] = home[slots[g][pick], c]
    parents = np.tile(np.arange(B, dtype=np.int32), (G, 1))
    parents[:, 1:B:2] = 0
    return slots, home, table, parents


@pytest.mark.parametrize("B,n_tables,which,fault", [(4, 1, 0, "none"), (4, 1, 0, "twice"), (3, 2, 1, "none"), (32, 2, 0, "twice"), (5, 8, 6, "none"),
                                                    (2, 5, 4, "negative")])
def test_a_group_without_a_page_per_beam_is_left_as_it_was(B, n_tables, which, fault):
    """One of three groups lacks a page of its own at the column that is written, in one table of several: the group is reported, and nothing
    of it changes or moves in any table; the other two groups go on."""
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    length, width = 150, 4
    made = [groups_with_homes(3, B, width, length, 7) for _ in range(n_tables)]
    slots, _, _, parents = made[0]
    homes, tables = [m[1].copy() for m in made], [m[2].copy() for m in made]
    homes[which][slots[1, B - 1], length // 64] = {"none": 0, "negative": -3, "twice": homes[which][slots[1, 0], length // 64]}[fault]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)       # noqa: E731
    on_gpu = [dev(t) for t in tables]
    moves = KB.tables(dev(slots), dev(parents), dev(np.full(3, length, dtype=np.int32)), 0,
                      [KB.Table(t, dev(h)) for t, h in zip(on_gpu, homes)])
    with pytest.raises(K.KernelError, match="out of place"):
        K.check_status()
    rest = [0, 2]
    want_tables = [t.copy() for t in tables]
    want = plain.tables(want_tables, homes, [0] * n_tables, slots[rest], parents[rest], [length] * 2).reshape(1 + n_tables, 2, B, 3)
    got = moves.cpu().numpy().reshape(1 + n_tables, 3, B, 3)
    assert np.array_equal(got[:, rest], want) and not got[:, 1].any()
    for t, w in zip(on_gpu, want_tables):
        assert np.array_equal(t.cpu().numpy(), w)            # (the plain form has left the group's rows alone)


def test_a_group_in_which_nothing_moves_needs_no_pages():
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    slots, home, table, _ = groups_with_homes(2, 4, 3, 70, 3)
    parents = np.tile(np.arange(4, dtype=np.int32), (2, 1))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)       # noqa: E731
    t = dev(table)
    moves = KB.tables(dev(slots), dev(parents), dev(np.full(2, 70, dtype=np.int32)), 0, [KB.Table(t, torch.zeros_like(t))])
    K.check_status()
    assert not moves.any().item() and np.array_equal(t.cpu().numpy(), table)


@pytest.mark.parametrize("G,B,V,stops", [(1, 32, 151936, (7, 100000)), (2, 24, 200000, (0, 199999)), (1, 32, 152000, tuple(range(0, 16 * 9000, 9000)))])
def test_wide_groups_whose_best_beams_are_the_last(G, B, V, stops):
    """Tiles of the last rows find no room among the keys that are kept, and bound the choice all the same: with stop tokens the selection
    takes about as long as without (1.1 times; 58 times where they did not count), and the results are the plain form's."""
    from toyinfer_b200.kernels import beam as KB
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(G * B, V, generator=g, device=DEV) * 2.5
    s = torch.randn(G, B, generator=g, device=DEV) - 20
    s[:, :B - 6] -= 30
    for i, t in enumerate(stops[:4]):
        x[-1 - i, t] = 14.0 - i                             # sequences that are over, in the last tiles of all
    ids = torch.tensor(stops, dtype=torch.int32, device=DEV)
    got = KB.select(x, s, B, ids)
    for a, b in zip(got, plain.select(x.cpu().numpy(), s.cpu().numpy(), B, stops)):
        a, b = a.cpu().double(), torch.from_numpy(np.asarray(b)).double()
        f = torch.isfinite(b)
        assert torch.equal(a[~f], b[~f]) and ((a[f] - b[f]).abs() <= 1.01 * 2 ** -24 * b[f].abs() + 5e-11).all()

    def time(ids):
        times = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(20):
                KB.select(x, s, B, ids)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    time(None)
    assert time(ids) < 5 * time(None)


def test_selections_with_wide_scores_in_one_graph():
    """Two steps captured together, the second from the first one's scores where they lie; replayed with other logits."""
    from toyinfer_b200.kernels import beam as KB
    G, B, V = 3, 4, 20001
    make = lambda seed: torch.randn(2, G * B, V, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * 2.5      # noqa: E731
    start = -3000 + torch.arange(G * B, device=DEV, dtype=torch.float64).view(G, B) * 1e-5
    two = lambda x: KB.select(x[1], KB.select(x[0], start, B, wide=True).scores, B, wide=True)                                  # noqa: E731
    x = make(1)
    two(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = two(x)
    for seed in (2, 3):
        x.copy_(make(seed))
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, two(x.clone())))
