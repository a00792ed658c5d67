"""Beam search's kernels: the selection over beams and vocabulary (csrc/beam_select.cu), page tables and moves from the
sequences' lengths and the beams' parents (csrc/beam_tables.cu), and the move of pages and states (csrc/beam_reorder.cu).

A *group* is one request's beams; a beam's *place* is its index in the group, and belongs to one slot of the cache.  After
``select`` the sequence at a place goes on from its parent's; ``tables`` and ``reorder`` let the cache follow, on the device:
nothing of a step has to pass through the host before the next one starts.

    choice = select(logits, scores, beams, stop_ids)
    moves = tables(slots, choice.parents, lengths, extra, [Table(...), ...])
    reorder(areas, moves)
"""
from __future__ import annotations

from ctypes import c_int, c_longlong, c_void_p
from typing import NamedTuple, Optional, Sequence

import torch

from . import KernelError, _call, _need_cuda, _ptr, _raw_device, _stream
from .wide import _fn
from ..cache.allocators import PAGE

P, I, L = c_void_p, c_int, c_longlong
_SELECT = [P, L, I, I, I, P, I, I, P, I, I, P, P, P, P]
_TABLES = [P, I, P, P, P, I, I, I, I, I, P, P]
_REORDER = [P, I, I, P, P, P, I, P]
BEAMS_MAX = 32          # beams of one group
STOPS_MAX = 16          # stop tokens
TABLES_MAX = 8          # page tables of one cache
ROWS_MAX = 65535        # rows of logits of one selection
VOCAB_MAX = 1 << 30     # logits of a row: places inside a row are 32-bit numbers
MOVES_MAX = 8192        # entries of one call's moves, over its lists
TILE, PART = 1024, 4    # logits of a row that csrc/beam_select.cu takes at a time, and the words of scratch for them
PIECE = 16384           # bytes that a warp moves at a time (csrc/beam_reorder.cu)


def _here(*tensors, what: str) -> None:
    """All on the current device: the launch goes to its stream."""
    devices = {t.get_device() for t in tensors if t is not None}
    if -1 in devices:                    # not a CUDA device
        _need_cuda(*tensors, what=what)
    now = _raw_device() if _raw_device is not None else torch.cuda.current_device()
    if devices - {now}:
        raise KernelError(f"{what}: tensors on cuda {sorted(devices)}, the current device is cuda:{now}")


class Choice(NamedTuple):
    """What ``select`` gives, [groups, beams] each.  By place: the next beams' scores (-inf: no beam), the places they come from (a
    place itself, or one whose parent is itself) and their tokens.  By rank: the candidates that ended, each at the rank it had among
    all candidates (-inf, -1 and -1 elsewhere)."""

    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor
    ended_scores: torch.Tensor
    ended_parents: torch.Tensor
    ended_tokens: torch.Tensor


def select(logits: torch.Tensor, scores: torch.Tensor, beams: int, stop_ids: Optional[torch.Tensor] = None, ending: bool = True,
           wide: bool = False) -> Choice:
    """The next ``beams`` beams of every group.  logits float32 [groups * held, vocab] (a group's rows follow one another), scores
    float32 [groups, held] with held <= beams: the logarithms of the beams' probabilities so far (-inf: no beam; its row is not read).

    A continuation's total is its beam's score plus log softmax of its row; larger totals come first, then lower (beam, token).  The
    first ``beams`` whose token is not in ``stop_ids`` (int32, at most 16) are the next beams; with ``ending`` those among the first
    ``beams`` of all whose token is in it are returned as ended.  NaN counts as -inf, +inf as the largest finite number, and what is
    at -inf is never chosen: a group with fewer continuations keeps places without a beam.  The first child of a beam stays at its
    place, the other children take the places of beams without one, in order.  Totals are formed in 64 bits and returned in 32.  With ``wide`` scores are float64, those
    given and those returned: for searches that hand them on from step to step, where each rounding to 32 bits would be one of the
    whole sum."""
    _here(logits, scores, stop_ids, what="beam select")
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise KernelError("beam select: expected float32 [rows, vocab] with dense rows")
    if scores.dtype != (torch.float64 if wide else torch.float32) or scores.dim() != 2 or not scores.is_contiguous():
        raise KernelError(f"beam select: scores must be dense {'float64' if wide else 'float32'} [groups, beams]")
    G, held = scores.shape
    R, V = logits.shape
    if R != G * held or R == 0 or V == 0:
        raise KernelError(f"beam select: {R} rows of {V} logits do not fit {G} groups of {held} beams")
    if V > VOCAB_MAX or R > ROWS_MAX:
        raise KernelError(f"beam select: {R} rows of {V} logits (at most {ROWS_MAX} of {VOCAB_MAX})")
    if not 1 <= held <= beams <= BEAMS_MAX:
        raise KernelError(f"beam select: {beams} beams from {held} (at most {BEAMS_MAX}, and no fewer than before)")
    n_stops = 0
    if stop_ids is not None:
        if stop_ids.dtype != torch.int32 or stop_ids.dim() != 1 or not stop_ids.is_contiguous():
            raise KernelError("beam select: stop tokens must be dense int32")
        n_stops = stop_ids.numel()
        if n_stops > STOPS_MAX:
            raise KernelError(f"beam select: {n_stops} stop tokens (at most {STOPS_MAX})")
    # results and scratch in one piece: each allocation takes the host as long as half a launch
    n = G * beams
    words = 4 * n if wide else 2 * n              # of the scores
    at = (words + 4 * n + 3) & ~3
    room = torch.empty(at + R * (-(-V // TILE)) * PART, dtype=torch.int32, device=logits.device)
    base = room.data_ptr()
    _call(_fn("ti_beam_select", _SELECT),
          logits.data_ptr(), logits.stride(0) if R > 1 else V, G, held, V, scores.data_ptr(), 1 if wide else 0, beams, _ptr(stop_ids), n_stops,
          1 if ending else 0, base, base + 4 * words, base + 4 * at, _stream(), launches=2)
    if wide:
        scores, ended_scores = room[:words].view(torch.float64).view(2, G, beams).unbind(0)
        parents, tokens, ended_parents, ended_tokens = room.as_strided((4, G, beams), (n, beams, 1), words).unbind(0)
        return Choice(scores, parents, tokens, ended_scores, ended_parents, ended_tokens)
    scores, ended_scores, parents, tokens, ended_parents, ended_tokens = room.as_strided((6, G, beams), (n, beams, 1)).unbind(0)
    return Choice(scores.view(torch.float32), parents, tokens, ended_scores.view(torch.float32), ended_parents, ended_tokens)


class Table(NamedTuple):
    """A cache group's page table as ``tables`` changes it, int32 [slots + 1, columns] on the device; ``home``: the same with the pages
    that each slot was given by the cache; ``ring_rows``: positions that a windowed group's ring holds (0: all positions are kept)."""

    table: torch.Tensor
    home: torch.Tensor
    ring_rows: int = 0


def tables(slots: torch.Tensor, parents: torch.Tensor, lengths: torch.Tensor, extra: int, page_tables: Sequence[Table]) -> torch.Tensor:
    """Lets the page tables follow the beams, in place, and returns what has to move: int32 [1 + tables, groups * beams, 3] with
    (source, destination, rows) per place, rows 0 where nothing does.  List 0 is slots (for states), list 1 + i pages of table i.

    slots and parents int32 [groups, beams], each slot in one group, parents as ``select`` gives them; lengths int32 [groups]: the
    positions that each group's sequences hold are lengths + extra.  A page that is not written any more is shared by the places that come from its
    beam; at the column that the next token goes to every place gets a page of its own, out of the group's homes there, and the
    rows that it holds so far are among the moves.  At that column the homes of a group are pages of its own, one per place; a group
    whose are not is reported (``check_status``) and left as it was, and so is a place whose parent or slot is out of place.
    ``reorder`` comes next, before anything reads the tables or writes the pages."""
    _here(slots, parents, lengths, what="beam tables")
    for t, what in ((slots, "slots"), (parents, "parents"), (lengths, "lengths")):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise KernelError(f"beam tables: {what} must be dense int32")
    shape = slots.shape
    if len(shape) != 2 or parents.shape != shape or lengths.shape != shape[:1] or 0 in shape:
        raise KernelError("beam tables: expected slots and parents [groups, beams] and lengths [groups]")
    G, B = shape
    n_tables = len(page_tables)
    if B > BEAMS_MAX or n_tables > TABLES_MAX:
        raise KernelError(f"beam tables: {B} beams, {n_tables} tables (at most {BEAMS_MAX} and {TABLES_MAX})")
    if not -(1 << 30) <= extra <= 1 << 30:
        raise KernelError(f"beam tables: {extra} positions behind the lengths")
    words = []
    n_slots = None
    for table, home, ring_rows in page_tables:
        _here(table, home, what="beam tables")
        shape = table.shape
        if table.dtype != torch.int32 or len(shape) != 2 or not table.is_contiguous() or home.dtype != torch.int32 \
                or home.shape != shape or not home.is_contiguous():
            raise KernelError("beam tables: a table and its homes must be dense int32 [slots + 1, columns] of one shape")
        if ring_rows < 0 or ring_rows % PAGE or (n_slots is not None and shape[0] != n_slots):
            raise KernelError(f"beam tables: a ring of {ring_rows} rows, {shape[0]} slots")
        n_slots = shape[0]
        words += (table.data_ptr(), home.data_ptr(), shape[1], ring_rows // PAGE)
    moves = torch.empty((1 + n_tables, G * B, 3), dtype=torch.int32, device=slots.device)
    _call(_fn("ti_beam_tables", _TABLES), (c_longlong * len(words))(*words), n_tables, slots.data_ptr(),
          parents.data_ptr(), lengths.data_ptr(), int(extra), G, B, PAGE, n_slots if n_slots is not None else 1 << 30, moves.data_ptr(),
          _stream())
    return moves


class Areas:
    """Where ``reorder`` finds a cache's memory; made once.  ``states``: tensors [slots, ...]; ``pages``: per table, in the order that
    ``tables`` gets them, its tensors [layers, pages, kv heads, PAGE, dim].  All dense, on one device; the tensors are kept alive."""

    FIELDS = 12

    def __init__(self, states: Sequence[torch.Tensor], pages: Sequence[Sequence[torch.Tensor]]):
        if len(pages) > TABLES_MAX:
            raise KernelError(f"beam areas: {len(pages)} page tables (at most {TABLES_MAX})")
        self.tensors = [list(states)] + [list(of_table) for of_table in pages]
        every = [t for tensors in self.tensors for t in tensors]
        _need_cuda(*every, what="beam areas")
        self.device = every[0].device if every else None
        records, self.first, self.pieces = [], [0], []
        for which, tensors in enumerate(self.tensors):
            before = 0
            for t in tensors:
                if not t.is_contiguous() or t.device != self.device or t.dim() < (1 if which == 0 else 5) or t.numel() == 0:
                    raise KernelError(f"beam areas: {tuple(t.shape)} is not a dense tensor of "
                                      f"{'states [slots, ...]' if which == 0 else 'pages [layers, pages, heads, rows, dim]'} on {self.device}")
                e = t.element_size()
                if which == 0:
                    row = t.stride(0) * e
                    n_outer, outer, n_inner, inner, unit, units, rows = 1, 0, 1, 0, row, t.shape[0], 1
                else:
                    if t.dim() != 5 or t.shape[3] != PAGE:
                        raise KernelError(f"beam areas: pages {tuple(t.shape)} are not [layers, pages, heads, {PAGE}, dim]")
                    n_outer, units, n_inner, rows, _ = t.shape
                    outer, unit, inner, row = t.stride(0) * e, t.stride(1) * e, t.stride(2) * e, t.stride(3) * e
                width = next((w for w in (16, 4, 2) if not any(x % w for x in (t.data_ptr(), outer, inner, unit, row))), 0)
                if width == 0 or units >= 1 << 31:
                    raise KernelError(f"beam areas: {tuple(t.shape)} of {t.dtype} cannot be moved (elements of 2 or 4 bytes)")
                per_run = -(-(rows * row) // PIECE)
                records.append([t.data_ptr(), outer, n_outer, inner, n_inner, unit, units, row, rows, width, per_run, before])
                before += n_outer * n_inner * per_run
            self.first.append(len(records))
            self.pieces.append(before)
        self.n_areas = len(records)
        self.records = torch.tensor(records, dtype=torch.int64, device=self.device) if records else None
        self._first = (c_int * len(self.first))(*self.first)
        self._pieces = (c_longlong * len(self.pieces))(*self.pieces)


def reorder(areas: Areas, moves: torch.Tensor) -> None:
    """Copies what ``moves`` (from ``tables``) names: states from slot to slot, and of every layer's pages the first rows from page
    to page.  No move may read what another one writes (``tables`` sees to that)."""
    lists, shape = len(areas.tensors), moves.shape
    if moves.dtype != torch.int32 or len(shape) != 3 or shape[0] != lists or shape[2] != 3 or not moves.is_contiguous():
        raise KernelError(f"beam reorder: moves must be dense int32 [{lists}, places, 3]")
    if shape[1] == 0 or lists * shape[1] > MOVES_MAX:
        raise KernelError(f"beam reorder: {lists} lists of {shape[1]} moves (at most {MOVES_MAX} in all)")
    if areas.n_areas == 0:
        return
    _here(moves, areas.records, what="beam reorder")
    _call(_fn("ti_beam_reorder", _REORDER), _ptr(areas.records), areas.n_areas, lists, areas._first, areas._pieces,
          moves.data_ptr(), shape[1], _stream())
