"""Stand-ins for toyinfer_b200.kernels.beam on the CPU, for tests only: the plain form of tests/plain/beam_plain.py behind the same
names, on the tensors in place.  ``install(monkeypatch)`` patches them in."""
from __future__ import annotations

import numpy as np
import torch

from plain import beam_plain as plain
from toyinfer_b200.kernels import beam as KB


def select(logits, scores, beams, stop_ids=None, ending=True):
    out = plain.select(logits.numpy(), scores.numpy(), beams, () if stop_ids is None else stop_ids.tolist(), ending)
    return KB.Choice(*(torch.from_numpy(np.asarray(x)).to(torch.float32 if i in (0, 3) else torch.int32) for i, x in enumerate(out)))


def tables(slots, parents, lengths, extra, page_tables):
    moves = plain.tables([t.table.numpy() for t in page_tables], [t.home.numpy() for t in page_tables], [t.ring_rows for t in page_tables],
                         slots.numpy(), parents.numpy(), [n + extra for n in lengths.tolist()])
    return torch.from_numpy(moves).to(torch.int32)


class Areas:
    def __init__(self, states, pages):
        self.states, self.pages = states, pages


def reorder(areas, moves):
    plain.move(areas.states, areas.pages, moves.numpy())


def install(monkeypatch) -> None:
    for name in ("select", "tables", "Areas", "reorder"):
        monkeypatch.setattr(KB, name, globals()[name])
