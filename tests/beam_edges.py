"""What the tests of beam search's edges share: a model whose searches are known without running it."""
from __future__ import annotations

import contextlib
import types

import torch


class LastTokenModel:
    """An engine whose logits depend on the last token alone; its cache takes anything."""

    def __init__(self, logits):
        self.logits, self.device, self.slots = logits, logits.device, 0
        self.tracer = types.SimpleNamespace(range=lambda name: contextlib.nullcontext())
        self.cache = types.SimpleNamespace(beam_groups=lambda beams: 64, beam_tokens=lambda prompt, length, beams: 64, reserve_beams=lambda *a: None,
                                           begin_beams=lambda *a: None, follow_parents=lambda *a: None, kv_groups=[])

    def new_sequence(self):
        self.slots += 1
        return self.slots

    def end_sequence(self, slot):
        pass

    def step(self, entries, want, token_source=None):
        last = torch.tensor([t[-1] for _, t in entries], device=self.device) if token_source is None else token_source.long()
        return self.logits[last]


def best_chains(table, first, beams, n):
    """log softmax of the table's rows, and the search of ``n`` steps over last tokens alone, in 64 bits: [(score, tokens)]."""
    lp = torch.log_softmax(table.double().cpu(), -1).numpy()
    live = [(0.0, [first])]
    for _ in range(n):
        cand = sorted((-(s + lp[t[-1], v]), b, v) for b, (s, t) in enumerate(live) for v in range(lp.shape[1]))
        live = [(-c[0], live[c[1]][1] + [c[2]]) for c in cand[:beams]]
    return lp, live
