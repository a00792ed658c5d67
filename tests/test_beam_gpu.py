"""Beam search's kernels (csrc/beam_*.cu) against the plain form in 64 bits (tests/plain/beam_plain.py): the selection at sizes and
masks where it can go wrong, page tables of groups that share pages and of rings, the move of pages and states, and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from plain import beam_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 64
NAMES = ("scores", "parents", "tokens", "ended_scores", "ended_parents", "ended_tokens")


def check_select(logits, scores, beams, stops=(), ending=True):
    from toyinfer_b200.kernels import beam as KB
    ids = torch.tensor(list(stops), dtype=torch.int32, device=DEV) if len(stops) else None
    got = KB.select(logits, scores, beams, ids, ending)
    want = plain.select(logits.cpu().numpy(), scores.cpu().numpy(), beams, stops, ending)
    for name, x, y in zip(NAMES, got, want):
        x, y = x.cpu(), torch.from_numpy(np.asarray(y))
        if "scores" not in name:
            assert torch.equal(x.long(), y), name
        else:
            # one rounding to 32 bits: half a step, 2^-24 of the value; before it the row's sum, whose terms are off by
            # (ln 2 / 32)^5 / 120 = 4e-11 at most (csrc/beam_select.cu), and its logarithm by as much: it counts where a total is
            # near zero
            assert torch.equal(torch.isfinite(x), torch.isfinite(y)), name
            f = torch.isfinite(y)
            assert torch.equal(x[~f].double(), y[~f]), name
            assert ((x[f].double() - y[f]).abs() <= 1.01 * 2 ** -24 * y[f].abs() + 5e-11).all(), name
    return got


def inputs(G, held, V, seed=0, pad=0, width=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(G * held, V + pad, generator=g, device=DEV)[:, :V] * width if not pad else \
        (torch.randn(G * held, V + pad, generator=g, device=DEV) * width)[:, :V]
    return x, torch.randn(G, held, generator=g, device=DEV) - 7


@pytest.mark.parametrize("G,held,B,V,n_stops,pad", [
    (1, 1, 1, 1, 0, 0), (1, 1, 4, 2, 0, 0), (1, 1, 8, 5, 2, 0), (2, 3, 3, 7, 1, 3), (3, 4, 4, 520, 1, 0), (5, 2, 7, 1023, 3, 1),
    (1, 4, 4, 8192, 1, 0), (1, 4, 4, 8193, 1, 0), (2, 5, 5, 8191, 0, 1), (4, 4, 4, 32000, 2, 0), (2, 8, 8, 16384, 2, 4),
    (1, 1, 32, 20001, 16, 0), (2, 32, 32, 9001, 16, 2), (3, 24, 24, 4099, 5, 0), (1, 4, 4, 151936, 1, 0), (70, 3, 3, 300, 1, 0),
    (3000, 4, 4, 130, 1, 1)])
def test_select_sizes(G, held, B, V, n_stops, pad):
    x, s = inputs(G, held, V, seed=V + G, pad=pad)
    rng = np.random.RandomState(V)
    stops = rng.choice(V, size=min(n_stops, max(0, V - 1)), replace=False).tolist()
    for i, t in enumerate(stops[:3]):
        x[i % x.shape[0], t] = 12.0 - i                    # a beam that is over
    check_select(x, s, B, stops)
    check_select(x, s, B, stops, ending=False)


@pytest.mark.parametrize("held,B,V", [(1, 8, 5000), (1, 32, 20001), (1, 32, 3000), (2, 30, 40000), (1, 24, 1024 * 23), (3, 32, 152000), (32, 32, 152000)])
def test_select_with_fewer_tiles_than_beams(held, B, V):
    x, s = inputs(2, held, V, seed=V, pad=B % 3)
    s[1, 1:] = -float("inf")                     # one beam left
    x[0, 5] = 15.0
    check_select(x, s, B, [5, 17])


@pytest.mark.parametrize("kind", ["equal", "coarse", "rising", "falling", "one thread", "lowest", "few allowed", "peaked", "tiny range", "far apart"])
@pytest.mark.parametrize("V", [50, 3000, 20000, 200000])
def test_select_values(kind, V):
    G, B = 3, 6
    x, s = inputs(G, B, V, seed=5)
    at = torch.arange(V, device=DEV, dtype=torch.float32)
    if kind == "equal":
        x = torch.full_like(x, 0.25)
        s = torch.zeros_like(s) - 3          # all totals equal: the lowest (beam, token)
    elif kind == "coarse":
        x = (x * 2).round() / 2              # many ties inside a row
    elif kind == "rising":
        x = (at * 1e-3).expand(G * B, V).contiguous()
    elif kind == "falling":
        x = (-at * 1e-3).expand(G * B, V).contiguous()
    elif kind == "one thread":
        x = x.clone()
        x[:, ::256] += 50                    # one thread's entries hold all the large ones
    elif kind == "lowest":
        x[:, 3:] = torch.finfo(torch.float32).min
    elif kind == "few allowed":
        x[:, 2:] = -float("inf")
    elif kind == "peaked":
        x[:, 7] = 80.0
    elif kind == "tiny range":
        x = x * 1e-30
        x[:, 11] += 1.0
        x[:, 20] += 0.5
        x[:, 31] += 0.25
        x[:, 33:36] += 0.125
    elif kind == "far apart":
        x = x * 1e30
    check_select(x, s, B, [1, 7])


@pytest.mark.parametrize("V", [700, 40000, 151936])
@pytest.mark.parametrize("width,shift", [(0.3, 0.0), (2.5, 0.0), (8.0, 30.0), (2.5, -60.0), (3.0, 150.0), (30.0, -20.0)])
def test_select_near_ties_between_rows(V, width, shift):
    """Beams whose rows hold the same logits in another order, and whose scores differ by one step of 32 bits: each token's totals in
    the two rows are 6e-8 apart, a thousand times what the rows' sums may be off by."""
    G, B = 3, 6
    g = torch.Generator(device=DEV).manual_seed(V)
    base = torch.randn(V, generator=g, device=DEV) * width + shift
    x = torch.stack([base[torch.randperm(V, generator=g, device=DEV)] for _ in range(G * B)])
    one = torch.tensor(-0.75)
    steps = [one]
    for _ in range(B - 1):
        steps.append(torch.nextafter(steps[-1], torch.tensor(0.0)))
    s = torch.stack([torch.stack(steps)[torch.randperm(B)] for _ in range(G)]).to(DEV)
    check_select(x, s, B, [3])


def test_select_masks_and_missing_beams():
    inf, nan = float("inf"), float("nan")
    x, s = inputs(4, 4, 700, seed=9)
    s[0, 1] = -inf
    s[0, 3] = nan                             # no beam either
    x[1] = nan                                # whose row is not read
    s[1] = -inf                               # a group without beams
    s[2, 0] = -inf
    x[8, :] = 1e38
    x[9] = -inf                               # a beam whose row allows nothing
    x[10, ::2] = nan
    x[10, 5] = inf
    x[10, 9] = inf                            # two certain tokens
    x[12:16, 4:] = -inf
    x[12, :4] = nan
    got = check_select(x, s, 4, [2])
    assert got.parents[1].tolist() == [0, 1, 2, 3] and got.tokens[1].tolist() == [0] * 4
    check_select(x[:, :3], s, 4, [0, 1, 2])   # nothing but stop tokens: all end, none goes on
    check_select(x, s, 9, [2])


def test_select_is_the_same_every_time_and_reads_its_own_rows_only():
    from toyinfer_b200.kernels import beam as KB
    x, s = inputs(6, 4, 30001, seed=3, pad=3)
    a = KB.select(x, s, 4, None)
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(a, KB.select(x, s, 4, None)))
    b = KB.select(x[8:16], s[2:4].contiguous(), 4, None)
    assert all(torch.equal(p[2:4], q) for p, q in zip(a, b))
    # on a stream of its own, and captured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = KB.select(x, s, 4, None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d = KB.select(x, s, 4, None)
    x.copy_(x.flip(0))
    s.copy_(s.flip(0).flip(1))
    g.replay()
    e = KB.select(x, s, 4, None)
    assert all(torch.equal(p, q) for p, q in zip(d, e)) and not torch.equal(d.tokens, a.tokens)


def test_select_of_odd_views():
    """One row whose distance to the next is anything; a column of a wider tensor; a score that no logarithm has."""
    x, s = inputs(1, 1, 5000, seed=2)
    check_select(x[0].unsqueeze(1).t(), s, 4)                  # stride 1 along both
    check_select(x.expand(1, -1)[:, 7:4001], s, 3)
    wide = torch.randn(6, 9000, device=DEV)
    check_select(wide[:, 100:8101], torch.zeros(3, 2, device=DEV), 2)
    check_select(wide[::2, 4:4100], torch.zeros(1, 3, device=DEV), 3)
    from toyinfer_b200.kernels import beam as KB
    got = KB.select(wide[:2], torch.tensor([[float("inf"), 0.0]], device=DEV), 3, None)
    assert got.scores.tolist() == [[float("inf")] * 3] and got.tokens.tolist() == [[0, 1, 2]] and got.parents.tolist() == [[0, 0, 0]]


def test_two_selections_at_once():
    """On two streams, and from two graphs replayed side by side: each has scratch of its own."""
    from toyinfer_b200.kernels import beam as KB
    made = [inputs(8, 4, 60000, seed=k) for k in (1, 2)]
    want = [KB.select(x, s, 4, None) for x, s in made]
    streams, graphs = [torch.cuda.Stream() for _ in made], []
    for (x, s), st in zip(made, streams):
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            graphs.append((g, KB.select(x, s, 4, None)))
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, (_, got) in zip(want, graphs):
        assert all(torch.equal(a, b) for a, b in zip(w, got))
    for _ in range(5):
        got = []
        for (x, s), st in zip(made, streams):
            with torch.cuda.stream(st):
                got.append(KB.select(x, s, 4, None))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, k in zip(want, got) for a, b in zip(w, k))


# -- tables ------------------------------------------------------------------------------------------------------------
class Made:
    """Slots, homes and tables of groups that have searched for a while, with pages shared as a search leaves them."""

    def __init__(self, seed, G, B, lengths, width, ring=0, fork=None, share_at_write=False):
        rng = np.random.RandomState(seed)
        self.G, self.B, self.lengths, self.ring = G, B, lengths, ring
        self.n_slots = G * B + 2
        self.slots = rng.permutation(self.n_slots)[:G * B].reshape(G, B).astype(np.int32)
        self.home = np.zeros((self.n_slots + 1, width), dtype=np.int32)
        self.home[:-1] = 1 + rng.permutation(self.n_slots * width).reshape(self.n_slots, width)
        self.table = self.home.copy()
        for g in range(G):
            L = lengths[g]
            w = (L % ring if ring else L) // PAGE
            for c in range(width):
                pick = rng.permutation(B) if c == w and not share_at_write else rng.randint(0, B, B)
                if fork is not None and c < fork // PAGE:
                    pick = np.zeros(B, dtype=int)
                self.table[self.slots[g], c] = self.home[self.slots[g][pick], c]
        self.parents = np.tile(np.arange(B, dtype=np.int32), (G, 1))
        for g in range(G):
            lost = rng.permutation(B)[:rng.randint(0, B)]
            stay = [b for b in range(B) if b not in lost]
            self.parents[g, lost] = rng.choice(stay, len(lost))

    def dev(self, a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def run_tables(made, extra=0):
    """One call over tables of the same slots, against the plain form."""
    from toyinfer_b200.kernels import beam as KB
    m = made[0]
    tables = [x.dev(x.table) for x in made]
    got = KB.tables(m.dev(m.slots), m.dev(m.parents), m.dev(np.array(m.lengths, dtype=np.int32) - extra), extra,
                    [KB.Table(t, x.dev(x.home), x.ring) for t, x in zip(tables, made)])
    want_tables = [x.table.copy() for x in made]
    want = plain.tables(want_tables, [x.home for x in made], [x.ring for x in made], m.slots, m.parents, m.lengths)
    for t, w in zip(tables, want_tables):
        assert np.array_equal(t.cpu().numpy(), w)
    assert np.array_equal(got.cpu().numpy(), want)
    return want


@pytest.mark.parametrize("G,B", [(1, 1), (1, 4), (3, 2), (5, 8), (2, 32), (40, 3)])
@pytest.mark.parametrize("ring", [0, 64, 192])
def test_tables(G, B, ring):
    from toyinfer_b200 import kernels as K
    for seed, base in enumerate((1, 63, 64, 65, 128, 191, 192, 193, 256, 500)):
        lengths = [base + 17 * g % 120 for g in range(G)]
        width = ring // PAGE if ring else 11
        m = Made(seed, G, B, lengths, width, ring, fork=base // 2, share_at_write=bool(ring) and base % PAGE == 0 and base >= ring and G == 1)
        run_tables([m], extra=seed)
    K.check_status()


def test_tables_of_several_groups_and_none():
    from toyinfer_b200.kernels import beam as KB
    lengths = [100, 640, 0, 703]
    made = [Made(1, 4, 5, lengths, 12), Made(1, 4, 5, lengths, 2, 128), Made(1, 4, 5, lengths, 3, 192), Made(1, 4, 5, lengths, 1, 64),
            Made(1, 4, 5, lengths, 40), Made(1, 4, 5, lengths, 4, 256)]
    for m in made[1:]:
        m.slots, m.parents = made[0].slots, made[0].parents
    # (each table's pages were dealt out with its own slots: the same seed draws the same ones)
    run_tables(made)
    m = made[0]
    moves = KB.tables(m.dev(m.slots), m.dev(m.parents), m.dev(np.array(lengths, dtype=np.int32)), 0, [])
    assert np.array_equal(moves.cpu().numpy(), plain.tables([], [], [], m.slots, m.parents, lengths))


def test_a_sequence_at_the_end_of_its_table():
    m = Made(3, 2, 4, [256, 255], 4)            # all columns full: there is no column to write next
    run_tables([m])


def test_parents_out_of_place_are_reported_and_left_out():
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    m = Made(4, 2, 4, [70, 70], 3)
    for bad in ([1, 0, 2, 3], [0, 0, 1, 3], [0, 1, 2, 7], [-1, 1, 2, 3]):
        parents = np.array([bad, [0, 0, 2, 2]], dtype=np.int32)
        table = m.dev(m.table)
        moves = KB.tables(m.dev(m.slots), m.dev(parents), m.dev(np.array(m.lengths, dtype=np.int32)), 0, [KB.Table(table, m.dev(m.home))])
        with pytest.raises(K.KernelError, match="out of place"):
            K.check_status()
        good = np.array([[b if p < 0 or p > 3 or bad[p] != p else p for b, p in enumerate(bad)], [0, 0, 2, 2]], dtype=np.int32)
        want_table = m.table.copy()
        want = plain.tables([want_table], [m.home], [0], m.slots, good, m.lengths)
        assert np.array_equal(moves.cpu().numpy(), want) and np.array_equal(table.cpu().numpy(), want_table)


def test_slots_and_homes_out_of_place_are_reported_and_left_out():
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    m = Made(5, 1, 3, [70], 3)
    lengths, parents = m.dev(np.array([70], dtype=np.int32)), m.dev(np.array([[0, 0, 0]], dtype=np.int32))
    for bad in ([m.n_slots + 1, 0, 1], [0, -1, 1], [0, 1, 1]):
        table = m.dev(m.table)
        moves = KB.tables(m.dev(np.array([bad], dtype=np.int32)), parents, lengths, 0, [KB.Table(table, m.dev(m.home))])
        with pytest.raises(K.KernelError, match="out of place"):
            K.check_status()
        rows = [s for s in bad if 0 <= s <= m.n_slots and bad.count(s) == 1]
        other = [s for s in range(m.n_slots + 1) if s not in rows]
        assert np.array_equal(table.cpu().numpy()[other], m.table[other])
        assert all(0 <= x <= m.n_slots for x in moves[0, :, :2].flatten().tolist())
    home = m.home.copy()
    home[m.slots[0, 1:], 1] = 0                       # slots that brought no page for the column that is written
    table = m.dev(m.table)
    table[torch.from_numpy(m.slots[0]).long().to(DEV), 1] = int(m.home[m.slots[0, 0], 1])
    moves = KB.tables(m.dev(m.slots), parents, lengths, 0, [KB.Table(table, m.dev(home))])
    with pytest.raises(K.KernelError, match="out of place"):
        K.check_status()
    assert moves[1].abs().sum().item() == 0


def test_captured_and_replayed_with_other_parents():
    """The three kernels in one graph: a replay reads the parents and lengths that are there then, and gives what plain calls give."""
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    G, B, V = 4, 4, 3000
    m = Made(8, G, B, [100, 64, 130, 191], 4)
    pages = torch.randn(2, m.n_slots * 4 + 1, 2, PAGE, 16, device=DEV)
    state = torch.randn(m.n_slots + 1, 33, device=DEV)
    x, s = inputs(G, B, V, seed=4)
    slots, home, lengths = m.dev(m.slots), m.dev(m.home), m.dev(np.array(m.lengths, dtype=np.int32))

    def memory_of():
        return m.dev(m.table), pages.clone(), state.clone()

    def search(x, s, table, page, st, areas):
        c = KB.select(x, s, B, None)
        KB.reorder(areas, KB.tables(slots, c.parents, lengths, 0, [KB.Table(table, home)]))
        return c

    table, page, st = memory_of()
    areas = KB.Areas([st], [[page]])
    search(x, s, table, page, st, areas)              # (sets everything up)
    table.copy_(m.dev(m.table)), page.copy_(pages), st.copy_(state)
    xs, ss = x.clone(), s.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = search(xs, ss, table, page, st, areas)
    for seed in (11, 12):
        nx, ns = inputs(G, B, V, seed=seed)
        xs.copy_(nx), ss.copy_(ns)
        table.copy_(m.dev(m.table)), page.copy_(pages), st.copy_(state)
        g.replay()
        t2, p2, s2 = memory_of()
        want = search(nx, ns, t2, p2, s2, KB.Areas([s2], [[p2]]))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(table, t2) and torch.equal(page, p2) and torch.equal(st, s2) and not torch.equal(table, m.dev(m.table))
    K.check_status()


# -- the move ----------------------------------------------------------------------------------------------------------
def memory(dtype, layers, n_pages, heads, dims, n_slots, states, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages = [torch.randn(layers, n_pages, heads, PAGE, d, generator=g, device=DEV).to(dtype) for d in dims]
    return pages, [torch.randn(n_slots, *shape, generator=g, device=DEV) for shape in states]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,heads,dims,states", [
    (1, 1, (16,), []), (3, 2, (32, 32), [(5,)]), (2, 8, (128, 128), [(3, 4, 5), (1,)]), (5, 1, (576,), [(40000,)]), (2, 3, (48, 24), [(2049,)]),
    (1, 2, (7, 9), [(3,)]), (36, 2, (128, 128), [])])
def test_reorder(dtype, layers, heads, dims, states):
    from toyinfer_b200.kernels import beam as KB
    rng = np.random.RandomState(layers)
    n_pages, n_slots = 23, 13
    pages, state = memory(dtype, layers, n_pages, heads, dims, n_slots, states)
    order, slots = rng.permutation(n_pages), rng.permutation(n_slots)
    rows = [1, 63, 64, 17, 0, 40]
    paged = [(int(order[0]), int(order[1 + i]), n) for i, n in enumerate(rows)]        # one source, several destinations
    of_slots = [(int(slots[0]), int(slots[3]), 1), (0, 0, 0), (int(slots[1]), int(slots[4]), 1), (0, 0, 0), (int(slots[1]), int(slots[5]), 1), (0, 0, 0)]
    moves = np.array([of_slots, paged], dtype=np.int32)
    want_pages, want_state = [p.clone() for p in pages], [s.clone() for s in state]
    plain.move(want_state, [want_pages], moves)
    KB.reorder(KB.Areas(state, [pages]), torch.from_numpy(moves).to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(pages + state, want_pages + want_state))


def test_reorder_of_several_tables_and_many_moves():
    from toyinfer_b200.kernels import beam as KB
    pages = [memory(torch.bfloat16, n, 401, h, d, 1, [])[0] for n, h, d in ((2, 2, (64, 64)), (1, 1, (72,)), (3, 1, (16, 8)))]
    pages.insert(1, [])                                     # a table whose layers keep nothing here
    rng = np.random.RandomState(0)
    moves = np.zeros((5, 200, 3), dtype=np.int32)
    for k in range(5):
        p = rng.permutation(401)
        on = rng.rand(200) < 0.4
        moves[k][on] = np.stack([p[:200], p[200:400], rng.randint(0, 65, 200)], 1)[on]
    moves[0] = 0
    want = [[t.clone() for t in of_table] for of_table in pages]
    plain.move([], want, moves)
    KB.reorder(KB.Areas([], pages), torch.from_numpy(moves).to(DEV))
    assert all(torch.equal(a, b) for x, y in zip(pages, want) for a, b in zip(x, y))


def test_units_outside_the_memory_are_reported_and_left_out():
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    pages, state = memory(torch.bfloat16, 2, 6, 2, (64,), 4, [(10,)])
    keep = [t.clone() for t in pages + state]
    areas = KB.Areas(state, [pages])
    for bad in ((6, 1, 3), (1, 6, 3), (-1, 2, 64), (2, -5, 1)):
        moves = torch.tensor([[(0, 0, 0)], [bad]], dtype=torch.int32, device=DEV)
        KB.reorder(areas, moves)
        with pytest.raises(K.KernelError, match="out of place"):
            K.check_status()
        KB.reorder(areas, torch.tensor([[(0, 9, 1)], [(0, 0, 0)]], dtype=torch.int32, device=DEV))
        with pytest.raises(K.KernelError, match="out of place"):
            K.check_status()
    assert all(torch.equal(a, b) for a, b in zip(pages + state, keep))


@pytest.mark.parametrize("ring", [0, 128])
def test_run_of_all_three_keeps_every_history(ring):
    """Sequences whose every position holds a value of its own, beams chosen at random step after step: after each step every place's
    history, read through its table, is its parent's with the new value behind it."""
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    G, B, V, start, steps = 3, 5, 700, 50, 170
    width = ring // PAGE if ring else (start + steps) // PAGE + 1
    slots = np.random.RandomState(1).permutation(G * B).reshape(G, B).astype(np.int32)
    home = np.zeros((G * B + 1, width), dtype=np.int32)
    home[:-1] = 1 + np.arange(G * B * width).reshape(G * B, width)
    table = torch.from_numpy(home).to(DEV)
    home_d, slots_d = table.clone(), torch.from_numpy(slots).to(DEV)
    page = torch.zeros(1, G * B * width + 1, 1, PAGE, 1, device=DEV)
    state = torch.zeros(G * B + 1, 1, device=DEV)
    areas = KB.Areas([state], [[page]])
    lengths = torch.full((G,), start, dtype=torch.int32, device=DEV)
    history = [[[float(p) + 1000 * g for p in range(start)] for _ in range(B)] for g in range(G)]

    def row(p):
        return p % ring if ring else p

    t = table.cpu().numpy()
    for g in range(G):
        for p in range(max(0, start - ring) if ring else 0, start):
            page[0, int(t[slots[g][0], row(p) // PAGE]), 0, p % PAGE, 0] = history[g][0][p]
        state[int(slots[g][0])] = float(g + 1)
    gen = torch.Generator(device=DEV).manual_seed(2)
    scores = torch.zeros(G, 1, device=DEV)
    value = 0.0
    for step in range(steps):
        held = scores.shape[1]
        logits = torch.randn(G * held, V, generator=gen, device=DEV) * 3
        choice = KB.select(logits, scores, B, None)
        moves = KB.tables(slots_d, choice.parents, lengths, step, [KB.Table(table, home_d, ring)])
        KB.reorder(areas, moves)
        scores = choice.scores.clone()
        scores -= scores.amax(1, keepdim=True)
        parents = choice.parents.tolist()
        t = table.cpu().numpy()
        at = start + step
        write = [int(t[slots[g][b], row(at) // PAGE]) for g in range(G) for b in range(B)]
        assert len(set(write)) == G * B                     # a page of its own for every place
        history = [[list(history[g][parents[g][b]]) for b in range(B)] for g in range(G)]
        pages = page[0, :, 0, :, 0].cpu().numpy()
        st = state.cpu().numpy()
        for g in range(G):
            for b in range(B):
                first = max(0, at - ring + 1) if ring else 0
                got = [pages[t[slots[g][b], row(p) // PAGE], p % PAGE] for p in range(first, at)]
                assert got == history[g][b][first:], (step, g, b)
                assert st[slots[g][b], 0] == float(g + 1)
                value += 1.0
                history[g][b].append(value)
        new = torch.tensor([history[g][b][-1] for g in range(G) for b in range(B)], device=DEV)
        page[0, torch.tensor(write, device=DEV), 0, at % PAGE, 0] = new
    K.check_status()


def test_refusals():
    from toyinfer_b200 import kernels as K
    from toyinfer_b200.kernels import beam as KB
    x, s = inputs(2, 3, 40)
    ids = torch.zeros(17, dtype=torch.int32, device=DEV)
    many = torch.zeros(70000, 2, device=DEV)
    for args in ((many, torch.zeros(17500, 4, device=DEV), 4), (x.double(), s, 3), (x.t(), s, 3), (x, s.double(), 3), (x[:5], s, 3), (x, s, 2), (x, s, 33), (x, s.t(), 3), (x, s, 3, ids),
                 (x, s, 3, ids[:2].long()), (x.cpu(), s, 3), (x[:, :0], s, 3), (x, s[:0], 3)):
        with pytest.raises(K.KernelError):
            KB.select(*args)
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)      # noqa: E731
    good = (i(2, 3), i(2, 3), i(2), 0, [KB.Table(i(7, 4), i(7, 4), 0)])
    KB.tables(i(2, 3) + torch.arange(3, dtype=torch.int32, device=DEV), i(2, 3) + torch.arange(3, dtype=torch.int32, device=DEV), *good[2:])
    for at, bad in ((0, i(2, 3).long()), (1, i(2, 4)), (2, i(3)), (0, i(0, 3)), (4, [KB.Table(i(7, 4), i(7, 5), 0)]),
                    (4, [KB.Table(i(7, 4), i(7, 4), 100)]), (4, [KB.Table(i(7, 4), i(7, 4), 0), KB.Table(i(6, 4), i(6, 4), 0)]),
                    (4, [KB.Table(i(7, 4), i(7, 4), 0)] * 9), (0, i(2, 3).cpu())):
        args = list(good)
        args[at] = bad
        with pytest.raises(K.KernelError):
            KB.tables(*args)
    with pytest.raises(K.KernelError):
        KB.tables(i(1, 33), i(1, 33), i(1), 0, [])
    for states, pages in (([torch.zeros(3, 4, device=DEV).t()], []), ([], [[torch.zeros(1, 2, 1, 32, 4, device=DEV)]]),
                          ([torch.zeros(3, 4)], []), ([torch.zeros(3, 4, dtype=torch.uint8, device=DEV)[:, :3].contiguous()], []),
                          ([], [[torch.zeros(2, 1, 64, 4, device=DEV)]]), ([], [[]] * 9)):
        with pytest.raises(K.KernelError):
            KB.Areas(states, pages)
    areas = KB.Areas([torch.zeros(3, 4, device=DEV)], [])
    for moves in (i(2, 3, 3), i(1, 3, 2), i(1, 0, 3), i(1, 9000, 3), i(1, 3, 3).long(), i(1, 3, 3).cpu()):
        with pytest.raises(K.KernelError):
            KB.reorder(areas, moves)
    KB.reorder(KB.Areas([], [[], []]), i(3, 2, 3))
    K.check_status()
