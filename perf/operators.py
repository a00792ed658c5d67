"""What the speed of beam search's operators is measured on.

A case is a dict of plain values.  ``op`` says which operator one pass runs:

  select    the selection over beams and vocabulary: log-probabilities, the best continuations, their placement, the ended ones
  tables    the page tables and the map of what has to move, from the sequences' lengths and the beams' parents
  reorder   the move itself: the rows of the pages that are being written, and whole states, of all layers
  step      the three after one another, as the search runs them between two steps of the model

``groups`` requests hold ``beams`` beams each (``held`` of them before a selection: 1 when a request's prompt has just run).
Sequences hold between ``short`` and ``long`` positions (spread evenly in an irregular order), the last ``gen`` of them drawn.
``dead`` beams of each group lose their place to another beam's second child.  The sizes are those of the Qwen3 shapes, of the
layers of width 2,048 and 4,096 that ``bench.py`` measures, and of the tests' small models."""
import math

import numpy as np
import torch

own = False
PAGE = 64
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LOWEST = -3.4028234663852886e38


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the first selection of one request, right after its prompt: four beams from one row of logits; latency counts
        dict(name="select_first", op="select", groups=1, held=1, beams=4, dead=0, vocab=151936, stops=1, pad=0, masked="none"),
        # four requests of four beams, the Qwen3 vocabulary with its two stop tokens
        dict(name="select_4x4", op="select", groups=4, held=4, beams=4, dead=0, vocab=151936, stops=2, pad=0, masked="none"),
        # a full batch of 64 sequences
        dict(name="select_16x4", op="select", groups=16, held=4, beams=4, dead=0, vocab=151936, stops=1, pad=0, masked="none"),
        # as many beams as the reference takes, half of a smaller vocabulary masked (constrained output), beams without a future among them
        dict(name="select_32x8_masked", op="select", groups=32, held=8, beams=8, dead=2, vocab=32000, stops=1, pad=0, masked="lowest"),
        # rows of an odd length that start at any 4 bytes, many stop tokens, two wide groups
        dict(name="select_wide_odd", op="select", groups=2, held=24, beams=24, dead=0, vocab=123373, stops=5, pad=2, masked="inf"),
        # one request of four beams over one table: a launch's latency
        dict(name="tables_1x4", op="tables", groups=1, beams=4, dead=2, short=700, long=700, gen=37, window=0),
        # 64 requests of eight beams up to the benchmark's context, with a windowed group beside the one that keeps all positions
        dict(name="tables_64x8", op="tables", groups=64, beams=8, dead=3, short=40, long=8191, gen=30, window=1024),
        # the smallest model of the configurations, in the 32-bit engine, one request
        dict(name="reorder_small_f32", op="reorder", groups=1, beams=3, dead=1, short=50, long=50, gen=7, window=0, dtype="f32", layers=3,
             kv_heads=2, head_dim=32, value_dim=0, state=0, state_layers=0),
        # the 4B shape, sixteen requests of four beams: two of four beams move in every layer
        dict(name="reorder_4b_16x4", op="reorder", groups=16, beams=4, dead=2, short=70, long=290, gen=40, window=0, dtype="bf16", layers=36,
             kv_heads=8, head_dim=128, value_dim=0, state=0, state_layers=0),
        # linear-attention layers with a state per sequence beside latent ones that keep one row per position under a window
        dict(name="reorder_states_6x4", op="reorder", groups=6, beams=4, dead=2, short=30, long=1500, gen=25, window=1024, dtype="bf16",
             layers=6, kv_heads=1, head_dim=576, value_dim=-1, state=32 * 128 * 128 + 7, state_layers=18),
        # all of it for one request of four beams on the 4B shape
        dict(name="step_4b_1x4", op="step", groups=1, held=4, beams=4, dead=1, vocab=151936, stops=1, pad=0, masked="none", short=1000,
             long=1000, gen=25, window=0, dtype="bf16", layers=36, kv_heads=8, head_dim=128, value_dim=0, state=0, state_layers=0),
        # ... and for eight requests of eight beams
        dict(name="step_4b_8x8", op="step", groups=8, held=8, beams=8, dead=3, vocab=151936, stops=1, pad=0, masked="none", short=65,
             long=190, gen=33, window=0, dtype="bf16", layers=36, kv_heads=8, head_dim=128, value_dim=0, state=0, state_layers=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(("select", "select", "tables", "reorder", "step"))
    beams = rng.choice((1, 2, 3, 4, 4, 5, 6, 8, 8, 11, 16, 24))
    case = dict(op=op, beams=beams, dead=rng.randint(0, max(0, beams // 2)), groups=_log(rng, 1, max(1, 64 // beams)))
    if op == "tables":
        case["groups"] = _log(rng, 1, 512 // beams)
    if op in ("select", "step"):
        vocab = _log(rng, 300, 152000)
        case.update(held=1 if op == "select" and rng.random() < 0.2 else beams, vocab=vocab, stops=rng.randint(0, 6), pad=rng.choice((0, 0, 1, 5, 8)),
                    masked=rng.choice(("none", "none", "inf", "lowest")) if op == "select" else "none")
        if case["held"] == 1 and beams > 1:
            case["dead"] = 0
        elif op == "select":
            case["dead"] = min(case["dead"], beams - 1)
    if op != "select":
        long = _log(rng, 10, 8191 if op == "tables" else 300)
        case.update(short=rng.randint(1, long), long=long, window=rng.choice((0, 0, 64, 100, 128, 200, 1024)))
        case["gen"] = rng.randint(0, min(60, case["short"] - 1))
    if op in ("reorder", "step"):
        case.update(dtype=rng.choice(("bf16", "bf16", "f32")), layers=_log(rng, 1, 16), kv_heads=rng.choice((1, 2, 4, 8)),
                    head_dim=rng.choice((16, 48, 64, 72, 128, 128)), value_dim=rng.choice((0, 0, 0, -1, 64)))
        case.update(state=0, state_layers=0)
        if rng.random() < 0.5:
            case.update(state=_log(rng, 100, 200000), state_layers=_log(rng, 1, 12))
    return case


def _lengths(case):
    """Positions that each group's sequences hold."""
    n, lo, hi = case["groups"], case["short"], case["long"]
    return [lo + (g * 7919 % n) * (hi - lo) // max(1, n - 1) for g in range(n)]


def _move_rows(case, ring):
    """Rows of its write page that each group's moving sequences take along."""
    return [PAGE if ring and n >= ring else n % PAGE for n in _lengths(case)]


def _ring(case):
    return -(-case["window"] // PAGE) * PAGE


def work(case):
    moved = flops = 0
    op = case["op"]
    if op in ("select", "step"):
        rows = case["groups"] * (case["held"] - (case["dead"] if op == "select" and case["held"] > 1 else 0))
        moved += rows * case["vocab"] * 4 + case["groups"] * (case["held"] * 4 + case["beams"] * 24)
        flops += 3 * rows * case["vocab"]
    if op in ("tables", "step"):
        used = [-(-n // PAGE) for n in _lengths(case)]
        ring = _ring(case) // PAGE
        for cap in ([10 ** 9] if not ring else [10 ** 9, ring]):
            moved += sum(case["dead"] * 8 * min(u, cap) + case["beams"] * 32 for u in used)
    if op in ("reorder", "step"):
        e = 2 if case["dtype"] == "bf16" else 4
        both = case["head_dim"] + {0: case["head_dim"], -1: 0}.get(case["value_dim"], case["value_dim"])
        full, ring = _split(case)
        per_row = case["kv_heads"] * both * e
        moved += 2 * case["dead"] * per_row * (full * sum(_move_rows(case, 0)) + ring * sum(_move_rows(case, _ring(case))))
        moved += 2 * case["dead"] * case["groups"] * case["state"] * 4 * case["state_layers"]
        moved += case["groups"] * case["beams"] * 12
    return {"bytes": moved, "flops": flops}


def _split(case):
    """Layers that keep all positions, and layers under the window."""
    n = case["layers"]
    return (n, 0) if not case["window"] else ((n + 1) // 2, n // 2)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))
    s = {"case": case}
    op = case["op"]
    parents = _parents(case, rng)
    if op in ("select", "step"):
        s.update(_logits(case, gen, rng, parents))
    if op != "select":
        s.update(_pages(case, rng))
        s["parents"] = torch.from_numpy(parents).to(DEV)
    if op in ("reorder", "step"):
        s.update(_memory(case, gen, s["n_pages"]))
        if op == "reorder":
            s["moves"] = _tables_plain([t.clone() for t in s["tables"]], s, s["parents"])
    return s


def _parents(case, rng):
    """[groups, beams] int32: ``dead`` places of each group go to children of the others."""
    G, B, dead = case["groups"], case["beams"], case["dead"]
    p = np.tile(np.arange(B, dtype=np.int32), (G, 1))
    for g in range(G):
        order = rng.permutation(B)
        lost, live = order[:dead], order[dead:]
        if len(live):
            p[g, lost] = live[rng.randint(0, len(live), dead)]
    return p


def _logits(case, gen, rng, parents):
    G, H, B, V = case["groups"], case["held"], case["beams"], case["vocab"]
    R = G * H
    x = torch.randn(R, V + case["pad"], generator=gen, device=DEV)[:, :V].mul_(2.5)
    scores = torch.randn(G, H, generator=gen, device=DEV) - 20
    stops = torch.from_numpy(rng.choice(V, size=case["stops"], replace=False).astype(np.int32)).to(DEV)
    if case["stops"]:
        # in every third row the sequence may well be over
        over = torch.arange(0, R, 3, device=DEV)
        x[over, stops[0].long()] = 10 + torch.randn(len(over), generator=gen, device=DEV)
    if case["masked"] != "none":
        hide = torch.rand(V, generator=gen, device=DEV) < 0.5
        hide[stops.long()] = False
        x[:, hide] = LOWEST if case["masked"] == "lowest" else -math.inf
    if case["op"] == "step":
        # a model that knows its next tokens: the continuations that the search takes stand out, each in its parent's row
        child = torch.from_numpy((np.arange(G)[:, None] * H + parents).reshape(-1)).to(DEV).long()
        open_ids = np.setdiff1d(np.arange(V), stops.cpu().numpy())
        ids = torch.from_numpy(np.concatenate([rng.choice(open_ids, size=B, replace=False) for _ in range(G)])).to(DEV)
        x[child, ids] = 17 + 0.5 * torch.randn(G * B, generator=gen, device=DEV)
        scores = -20 + 0.1 * scores - 30 * torch.from_numpy((parents != np.arange(B)).astype(np.float32)).to(DEV)
    elif case["dead"] and H > 1:
        lost = np.stack([rng.permutation(H)[:case["dead"]] for _ in range(G)])
        scores.scatter_(1, torch.from_numpy(lost).to(DEV), -math.inf)
    return {"logits": x, "scores": scores, "stops": stops if case["stops"] else None}


def _pages(case, rng):
    """Slots, and per table the pages that each slot brought along (home) and the present rows."""
    G, B = case["groups"], case["beams"]
    lengths = _lengths(case)
    n_slots = G * B + 3
    slots = rng.permutation(n_slots)[:G * B].reshape(G, B).astype(np.int32)
    width = max(lengths) // PAGE + 2
    homes, rows, counts = [], [], []
    for ring in [0] if not case["window"] else [0, min(_ring(case) // PAGE, width)]:
        w = ring or width
        home = np.zeros((n_slots + 1, w), dtype=np.int32)
        row = np.zeros((n_slots + 1, w), dtype=np.int32)
        need = []
        for g in range(G):
            first = 0 if ring else (lengths[g] - case["gen"]) // PAGE      # columns before it are the prompt's, in the first place's row
            last = min(w, lengths[g] // PAGE + 1)
            need += [(slots[g, 0], c) for c in range(min(first, last))] + [(slots[g, b], c) for b in range(B) for c in range(first, last)]
        numbers = 1 + rng.permutation(len(need)).astype(np.int32)
        at = np.array(need)
        home[at[:, 0], at[:, 1]] = numbers
        for g in range(G):
            first = 0 if ring else (lengths[g] - case["gen"]) // PAGE
            last = min(w, lengths[g] // PAGE + 1)
            write = lengths[g] // PAGE % w if ring else lengths[g] // PAGE
            own_rows = home[slots[g]]                                       # [B, w]
            pick = rng.randint(0, B, (B, w))
            pick[:, :first] = 0
            pick[:, write] = rng.permutation(B)
            new = np.take_along_axis(own_rows, pick, 0)
            fresh = lengths[g] % PAGE == 0 and not (ring and lengths[g] >= ring * PAGE)
            if fresh:
                new[:, write] = own_rows[:, write]
            new[:, last:] = 0
            row[slots[g]] = new
        homes.append(torch.from_numpy(home).to(DEV))
        rows.append(torch.from_numpy(row).to(DEV))
        counts.append(len(need))
    base = torch.tensor([n - case["gen"] for n in lengths], dtype=torch.int32, device=DEV)
    rings = [0] if not case["window"] else [0, _ring(case)]
    if case["window"]:
        rings[1] = min(rings[1], rows[1].shape[1] * PAGE)
    return {"slots": torch.from_numpy(slots).to(DEV), "lengths": base, "homes": homes, "tables": rows, "rings": rings, "n_pages": counts,
            "n_slots": n_slots}


def _memory(case, gen, n_pages):
    dt = DTYPES[case["dtype"]]
    layers = _split(case)
    pages = []
    for n, count in zip(layers, n_pages):
        of_table = []
        if n:
            for dim in (case["head_dim"], case["value_dim"] or case["head_dim"]):
                if dim > 0:
                    of_table.append(torch.randn(n, count + 1, case["kv_heads"], PAGE, dim, generator=gen, device=DEV, dtype=dt))
        pages.append(of_table)
    n_slots = case["groups"] * case["beams"] + 3
    states = [torch.randn(n_slots + 1, case["state"], generator=gen, device=DEV) for _ in range(case["state_layers"])]
    return {"pages": pages, "states": states}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "select":
        return _select_own(s) if own else _select_plain(s)
    if op == "tables":
        moves = _tables_own(s["tables"], s, s["parents"]) if own else _tables_plain(s["tables"], s, s["parents"])
        return {"tables": s["tables"], "moves": moves}
    if op == "reorder":
        moves, out = s["moves"], {}
    else:
        out = _select_own(s) if own else _select_plain(s)
        moves = _tables_own(s["tables"], s, out["parents"]) if own else _tables_plain(s["tables"], s, out["parents"])
        out["tables"] = s["tables"]
    if own:
        from toyinfer_b200.kernels import beam
        if "areas" not in s:
            s["areas"] = beam.Areas(s["states"], s["pages"])      # a program makes it once, of its cache
        beam.reorder(s["areas"], moves)
    else:
        _reorder_plain(s["states"], s["pages"], moves)
    return {**out, "pages": s["pages"], "states": s["states"]}


def _select_own(s):
    from toyinfer_b200.kernels import beam
    return beam.select(s["logits"], s["scores"], s["case"]["beams"], s["stops"])._asdict()


def _tables_own(tables, s, parents):
    from toyinfer_b200.kernels import beam
    return beam.tables(s["slots"], parents, s["lengths"], s["case"]["gen"],
                       [beam.Table(t, h, r) for t, h, r in zip(tables, s["homes"], s["rings"])])


# -- plain forms -------------------------------------------------------------------------------------------------------
def _first(t, k):
    """Values and places of the k largest of each row of t [G, N], descending, the lowest place first on ties."""
    N = t.shape[1]
    bound = t.topk(k, dim=1).values[:, -1:]
    above, level = t > bound, t == bound
    take = above | (level & (level.cumsum(1) <= k - above.sum(1, keepdim=True)))
    order = torch.arange(N, 0, -1, device=t.device)
    at = N - torch.where(take, order, 0).topk(k, dim=1).values
    values, by = t.gather(1, at).sort(dim=1, descending=True, stable=True)
    return values, at.gather(1, by)


def _select_plain(s):
    x, scores, stops = s["logits"], s["scores"], s["stops"]
    G, H = scores.shape
    B, V = s["case"]["beams"], x.shape[1]
    x = torch.where(x.isnan(), -math.inf, x).clamp(max=-LOWEST).double().view(G, H, V)
    x = x - x.amax(-1, keepdim=True).clamp(min=LOWEST)
    total = scores.double().unsqueeze(-1) + (x - x.exp().sum(-1, keepdim=True).log())
    total = torch.where(total.isnan(), -math.inf, total)
    stop = torch.zeros(V, dtype=torch.bool, device=x.device)
    if stops is not None:
        stop[stops.long()] = True
    short = max(0, B - H * V)
    every = torch.nn.functional.pad(total.reshape(G, H * V), (0, short), value=-math.inf)
    going = torch.nn.functional.pad(torch.where(stop, -math.inf, total).reshape(G, H * V), (0, short), value=-math.inf)

    value, at = _first(going, B)
    there = value > -math.inf
    parent, token = at // V, at % V
    same = (parent.unsqueeze(2) == parent.unsqueeze(1)) & there.unsqueeze(1)             # [G, rank, earlier rank]
    stays = there & ~(same & torch.ones(B, B, dtype=torch.bool, device=x.device).tril(-1)).any(2)
    place = torch.arange(B, device=x.device)
    kept = ((parent.unsqueeze(2) == place) & stays.unsqueeze(2)).any(1)                  # [G, place]
    free = torch.where(kept, -1, (~kept).cumsum(1) - 1)
    moves = there & ~stays
    turn = torch.where(moves, moves.cumsum(1) - 1, -2)
    goes = torch.where(stays.unsqueeze(2), parent.unsqueeze(2) == place, turn.unsqueeze(2) == free.unsqueeze(1)) & there.unsqueeze(2)
    taken = goes.any(1)
    rank = goes.long().argmax(1)
    out = {"scores": torch.where(taken, value.gather(1, rank), -math.inf).float(),
           "parents": torch.where(taken, parent.gather(1, rank), place).int(),
           "tokens": torch.where(taken, token.gather(1, rank), 0).int()}

    value, at = _first(every, B)
    ends = (value > -math.inf) & stop[(at % V)]
    out["ended_scores"] = torch.where(ends, value, -math.inf).float()
    out["ended_parents"] = torch.where(ends, at // V, -1).int()
    out["ended_tokens"] = torch.where(ends, at % V, -1).int()
    return out


def _tables_plain(tables, s, parents):
    slots, parents = s["slots"].long(), parents.long()
    G, B = slots.shape
    held = s["lengths"].long() + s["case"]["gen"]
    place = torch.arange(B, device=slots.device)
    moved = parents != place
    source = slots.gather(1, parents)
    moves = [torch.stack([torch.where(moved, source, 0), torch.where(moved, slots, 0), moved.long()], -1)]
    for table, home, ring in zip(tables, s["homes"], s["rings"]):
        W = table.shape[1]
        col = torch.arange(W, device=slots.device)
        write = held // PAGE % W if ring else (held // PAGE).clamp(max=W - 1)
        used = ((held + PAGE - 1) // PAGE).clamp(max=W)
        at = write.view(G, 1, 1).expand(G, B, 1)
        rows, old = table[slots], table[source]
        new = torch.where((col < used.view(G, 1, 1)) & (col != at) & moved.unsqueeze(2), old, rows)
        begun = (write < used) & (held // PAGE < W) if not ring else write < used
        page = old.gather(2, at).squeeze(2)                                              # what each place's sequence has there
        twin = (page.unsqueeze(2) == page.unsqueeze(1)) & ~moved.unsqueeze(1)            # [G, place, another survivor]
        keeps = ~moved & ~(twin & torch.ones(B, B, dtype=torch.bool, device=slots.device).tril(-1)).any(2)
        mine = home[slots].gather(2, at).squeeze(2)
        free = ~((mine.unsqueeze(2) == page.unsqueeze(1)) & keeps.unsqueeze(1)).any(2)
        turn = torch.where(keeps, -1, (~keeps).cumsum(1) - 1)
        offer = torch.where(free, free.cumsum(1) - 1, -2)
        given = torch.where(turn.unsqueeze(2) == offer.unsqueeze(1), mine.unsqueeze(1), 0).sum(2)
        to = torch.where(keeps, page, given)
        now = torch.where(begun.unsqueeze(1), to, rows.gather(2, at).squeeze(2))
        table[slots] = new.scatter(2, at, now.unsqueeze(2).to(new.dtype))
        count = torch.where(held >= ring, PAGE, held % PAGE) if ring else held % PAGE
        goes = begun.unsqueeze(1) & ~keeps & (count.unsqueeze(1) > 0)
        moves.append(torch.stack([torch.where(goes, page, 0), torch.where(goes, to, 0), torch.where(goes, count.unsqueeze(1), 0)], -1))
    return torch.stack(moves).reshape(len(moves), G * B, 3).int()


def _reorder_plain(states, pages, moves):
    moves = moves.long()
    for state in states:
        src, dst, n = moves[0].unbind(1)
        spare = state.shape[0] - 1                          # nobody's slot: what does not move is copied from there to there
        state[torch.where(n > 0, dst, spare)] = state[torch.where(n > 0, src, spare)]
    row = torch.arange(PAGE, device=moves.device)
    for group, of_table in enumerate(pages):
        src, dst, n = moves[1 + group].unbind(1)
        for t in of_table:
            t[:, dst] = torch.where((row < n.view(-1, 1)).view(1, -1, 1, PAGE, 1), t[:, src], t[:, dst])


# ---------------------------------------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    out = {}
    if op in ("select", "step"):
        out = _exact_select(s["logits"].cpu().numpy(), s["scores"].cpu().numpy(), case["beams"],
                            [] if s["stops"] is None else s["stops"].tolist())
        if op == "select":
            return out
    parents = out["parents"] if op == "step" else s["parents"].cpu().numpy()
    tables = [t.cpu().numpy() for t in s["tables"]]
    moves = _exact_tables(tables, [h.cpu().numpy() for h in s["homes"]], s["rings"], s["slots"].cpu().numpy(), parents,
                          [n + case["gen"] for n in s["lengths"].tolist()])
    if op == "tables":
        return {"tables": tables, "moves": moves}
    for src, dst, n in moves[0]:
        if n:
            for state in s["states"]:
                state[int(dst)] = state[int(src)]
    for k, of_table in enumerate(s["pages"]):
        for src, dst, n in moves[1 + k]:
            if n:
                for t in of_table:
                    t[:, int(dst), :, :int(n)] = t[:, int(src), :, :int(n)]
    if op == "step":
        out["tables"] = tables
    return {**out, "pages": [[t.double() for t in of_table] for of_table in s["pages"]], "states": [t.double() for t in s["states"]]}


def _exact_select(x, scores, B, stops):
    G, H = scores.shape
    V = x.shape[1]
    names = ("scores", "parents", "tokens", "ended_scores", "ended_parents", "ended_tokens")
    out = {n: np.zeros((G, B)) if "scores" in n else np.zeros((G, B), dtype=np.int64) for n in names}
    with np.errstate(invalid="ignore", over="ignore"):
        for g in range(G):
            total = np.full((H, V), -np.inf)
            for b in range(H):
                row = np.minimum(np.where(np.isnan(x[g * H + b]), -np.inf, x[g * H + b]).astype(np.float64), -LOWEST)
                if scores[g, b] > -np.inf and row.max() > -np.inf:
                    top = row.max()
                    total[b] = np.float64(scores[g, b]) + (row - top - np.log(np.exp(row - top).sum()))
            total = total.reshape(-1)
            some = min(total.size, 4 * B + H * len(stops) + 8)
            bound = np.partition(total, total.size - some)[total.size - some]
            near = np.nonzero(total >= bound)[0]
            near = near[total[near] > -np.inf]
            best = [int(i) for i in near[np.argsort(-total[near], kind="stable")]]
            going = [i for i in best if i % V not in stops][:B]
            left = set(range(B))
            placed, later = {}, []
            for i in going:
                p = i // V
                if p in left:
                    placed[p] = i
                    left.discard(p)
                else:
                    later.append(i)
            # a place may only be taken by another's child when it has none of its own
            for i, place in zip(later, sorted(left)):
                placed[place] = i
            for b in range(B):
                i = placed.get(b)
                out["scores"][g, b] = -np.inf if i is None else total[i]
                out["parents"][g, b] = b if i is None else i // V
                out["tokens"][g, b] = 0 if i is None else i % V
                e = best[b] if b < len(best) and best[b] % V in stops else None
                out["ended_scores"][g, b] = -np.inf if e is None else total[e]
                out["ended_parents"][g, b] = -1 if e is None else e // V
                out["ended_tokens"][g, b] = -1 if e is None else e % V
    return out


def _exact_tables(tables, homes, rings, slots, parents, lengths):
    """Changes the tables; returns the moves [1 + tables, groups * beams, 3]."""
    G, B = slots.shape
    moves = np.zeros((1 + len(tables), G, B, 3), dtype=np.int64)
    for g in range(G):
        for b in range(B):
            if parents[g, b] != b:
                moves[0, g, b] = (slots[g, parents[g, b]], slots[g, b], 1)
    for k, (table, home, ring) in enumerate(zip(tables, homes, rings)):
        W = table.shape[1]
        for g in range(G):
            n = lengths[g]
            write = n // PAGE % W if ring else n // PAGE
            used = min(-(-n // PAGE), W)
            before = table[slots[g]].copy()
            for b in range(B):
                for c in range(used):
                    if c != write:
                        table[slots[g, b], c] = before[parents[g, b], c]
            if write >= used:
                continue
            kept = {}
            for b in range(B):
                if parents[g, b] == b and before[b, write] not in kept:
                    kept[before[b, write]] = b
            spare = [p for p in (home[slots[g, b], write] for b in range(B)) if p not in kept]
            rows = PAGE if ring and n >= ring else n % PAGE
            for b in range(B):
                page = before[parents[g, b], write]
                if kept.get(page) != b:
                    new = spare.pop(0)
                    table[slots[g, b], write] = new
                    if rows:
                        moves[1 + k, g, b] = (page, new, rows)
    return moves.reshape(1 + len(tables), G * B, 3)
