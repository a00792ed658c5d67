"""Beam search's bookkeeping at its edges, without a device: scores over long searches, limits, options."""
from __future__ import annotations

import types

import numpy as np
import pytest
import torch

from beam_edges import LastTokenModel, best_chains
from plain import beam_plain
from toyinfer_b200 import BeamParams
from toyinfer_b200.engine.beam import BeamLoop, BeamStepper
from toyinfer_b200.kernels import beam as KB


def select_plain(logits, scores, beams, stop_ids=None, ending=True):
    """As kernels.beam.select: totals in 64 bits, handed over in the type of ``scores``."""
    out = beam_plain.select(logits.numpy(), scores.numpy(), beams, () if stop_ids is None else stop_ids.tolist(), ending)
    return KB.Choice(*(torch.from_numpy(np.asarray(x)).to(scores.dtype if i in (0, 3) else torch.int32) for i, x in enumerate(out)))


def test_scores_of_a_long_search_are_sums_in_64_bits(monkeypatch):
    """1,500 tokens of log-probabilities near -3.7 come to -5,500, where a step of 32 bits is 5e-4, as far as beams are apart here:
    the scores are their tokens' sums in 64 bits (1,500 roundings of half a step, 2^-41 each: 7e-10 on either side), and the beams are
    the best ones.  The model is a chain, so the best sequences are known from a search over last tokens alone."""
    monkeypatch.setattr(KB, "select", select_plain)
    V, n, B = 40, 1500, 4
    table = torch.randn(V, V, generator=torch.Generator().manual_seed(0)) * 1e-3
    params = BeamParams(B, n_best=B)
    loop = BeamLoop(BeamStepper(LastTokenModel(table), params, []), params, [], 8, 1 << 20, 1 << 20)
    got = loop.run([[3]], n)[0]
    lp, live = best_chains(table, 3, B, n)
    assert len(got) == B and {len(h.tokens) for h in got} == {n}
    for h, (score, tokens) in zip(got, live):
        path = [3] + h.tokens
        assert abs(h.score - sum(lp[a, b] for a, b in zip(path, path[1:]))) <= 1e-8
        assert abs(h.score - score) <= 1e-8
        assert h.tokens == tokens[1:]


@pytest.mark.parametrize("penalty", ["9", "-1", "nan", "0.5"])
def test_without_beam_search_any_length_penalty_is_taken(monkeypatch, capsys, penalty):
    import toyinfer_b200
    from toyinfer_b200.engine import cli

    class Fake:
        engine = types.SimpleNamespace(spec=types.SimpleNamespace(vocab_size=10))
        last_stats = types.SimpleNamespace(prompt_tokens=1, generated_tokens=2)

        def __init__(self, *args, **kw):
            pass

        def generate(self, prompts, *args, **kw):
            return [types.SimpleNamespace(tokens=[4, 5], finish_reason="length") for _ in prompts]

    monkeypatch.setattr(toyinfer_b200, "LLM", Fake)
    assert cli.main(["--model_dir", "x", "--prompt_ids", "1", "--length_penalty", penalty]) == 0
    assert '"tokens": [4, 5]' in capsys.readouterr().out
    if penalty != "0.5":
        assert cli.main(["--model_dir", "x", "--prompt_ids", "1", "--length_penalty", penalty, "--beam_size", "2"]) == 2


def test_a_folder_without_a_model_is_an_error_of_the_call(capsys):
    from toyinfer_b200.engine import cli
    assert cli.main(["--model_dir", "nowhere", "--prompt_ids", "1"]) == 2
    assert "nowhere" in capsys.readouterr().err
