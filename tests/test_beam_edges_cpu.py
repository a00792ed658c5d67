"""Beam search's bookkeeping at its edges, without a device: scores over long searches, limits, options."""
from __future__ import annotations

import types

import numpy as np
import pytest
import torch

import cpu_beam
import cpu_kernels
from beam_edges import LastTokenModel, best_chains
from conftest import prompts_for
from plain import beam_plain
from toyinfer_b200 import LLM, BeamParams
from toyinfer_b200.cache import CacheError
from toyinfer_b200.engine.beam import BeamLoop, BeamStepper, plan_beams
from toyinfer_b200.kernels import KernelError
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


@pytest.fixture()
def cpu_llm(monkeypatch, model_folders):
    cpu_kernels.install(monkeypatch)
    cpu_beam.install(monkeypatch)
    return lambda name, **kw: LLM(model_folders[name], dtype="float32", device="cpu", **{"max_batch": 8, "max_tokens": 2048, **kw})


def test_a_batch_holds_no_more_groups_than_one_move_takes(cpu_llm, monkeypatch):
    """The move takes so many entries over all lists (states and page tables): more requests run in further batches."""
    llm = cpu_llm("A", max_seq_len=64, max_batch=8)
    lists = 1 + len(llm.engine.cache.kv_groups)
    prompts = prompts_for("A", [5, 6, 7, 8, 9], seed=2)
    want = llm.beam_search(prompts, BeamParams(2, n_best=2), max_new_tokens=4, ignore_eos=True)
    assert llm.last_stats.batches == 2
    monkeypatch.setattr(KB, "MOVES_MAX", lists * 5)          # two groups of two beams, not three
    tables = KB.tables

    def limited(slots, *args):
        assert slots.numel() * lists <= KB.MOVES_MAX
        return tables(slots, *args)

    monkeypatch.setattr(KB, "tables", limited)
    got = llm.beam_search(prompts, BeamParams(2, n_best=2), max_new_tokens=4, ignore_eos=True)
    assert llm.last_stats.batches == 3
    assert [[h.tokens for h in g] for g in got] == [[h.tokens for h in g] for g in want]


def test_a_cache_that_cannot_hold_beams_is_refused_before_anything_runs(cpu_llm, monkeypatch):
    """More page tables than one call takes, or memory that cannot be moved."""
    llm = cpu_llm("C", max_seq_len=64)                        # full and windowed layers: two tables
    c = llm.engine.cache
    assert len(c.kv_groups) == 2
    monkeypatch.setattr(llm.engine, "step", lambda *a, **k: pytest.fail("a step ran"))
    monkeypatch.setattr(KB, "TABLES_MAX", 1)
    with pytest.raises(CacheError, match="page tables"):
        llm.beam_search([[1, 2]], BeamParams(2), ignore_eos=True)
    monkeypatch.setattr(KB, "TABLES_MAX", 8)

    def refusing(states, pages):
        raise KernelError("cannot be moved")

    monkeypatch.setattr(KB, "Areas", refusing)
    c._areas = None
    with pytest.raises(KernelError, match="cannot be moved"):
        llm.beam_search([[1, 2]], BeamParams(2), ignore_eos=True)
    assert c.slots.n_free == c.n_slots


def test_plan_by_positions():
    """A request that fills the cache to the last position shares a batch; one position less, and it does not."""
    assert plan_beams([64, 640, 64], 8, 704) == [[0, 1], [2]]
    assert plan_beams([64, 640, 64], 8, 703) == [[0], [1], [2]]
    assert plan_beams([64, 640, 64], 8, 768) == [[0, 1, 2]]


def test_sizes_that_pass_32_bits_are_refused(monkeypatch):
    """Sizes go to the kernels as 32-bit numbers: 2^32 + 5 logits must not be taken as 5, nor 2^32 positions as none."""
    monkeypatch.setattr(KB, "_here", lambda *tensors, what: None)
    monkeypatch.setattr(KB, "_call", lambda *a, **k: pytest.fail("a kernel was launched"))
    monkeypatch.setattr(KB, "_fn", lambda *a: None)
    for V in ((1 << 32) + 5, (1 << 31) - 1, (1 << 30) + 1):
        with pytest.raises(KernelError, match="logits"):
            KB.select(torch.empty(2, V, device="meta"), torch.empty(1, 2, device="meta"), 2)
    with pytest.raises(KernelError, match="rows"):
        KB.select(torch.empty(65536, 8, device="meta"), torch.empty(32768, 2, device="meta"), 2)
    slots = torch.zeros(1, 2, dtype=torch.int32)
    for extra in (1 << 32, (1 << 31) - 1, -(1 << 31)):
        with pytest.raises(KernelError, match="positions"):
            KB.tables(slots, slots, slots[0, :1], extra, [])
