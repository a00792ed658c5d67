"""Beam search without a device: the loop's decisions, the cache's bookkeeping for beams, and the whole search through the engine on
the CPU (kernels replaced by tests/cpu_kernels.py and tests/cpu_beam.py) against the plain search, which runs every prefix whole."""
from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

import cpu_beam
import cpu_kernels
from conftest import prompts_for
from plain import beam_plain
from plain import qwen3_plain as plain
from toyinfer_b200 import LLM, BeamParams
from toyinfer_b200.cache import CacheError, CacheManager
from toyinfer_b200.engine.beam import plan_beams
from toyinfer_b200.kernels import KernelError
from toyinfer_b200.parts.base import KVRequest, StateRequest


@pytest.fixture()
def cpu_llm(monkeypatch, model_folders):
    cpu_kernels.install(monkeypatch)
    cpu_beam.install(monkeypatch)
    return lambda name, **kw: LLM(model_folders[name], dtype="float32", device="cpu", **{"max_batch": 8, "max_tokens": 2048, **kw})


def plain_search(folder, prompt, beams, max_new, **kw):
    w, cfg = plain.read_weights(folder), plain.read_config(folder)
    return beam_plain.search(lambda ids: plain.forward(w, cfg, ids)[-1].float().numpy(), prompt, beams, max_new, **kw)


def same(got, want):
    assert [(h.tokens, h.finish_reason) for h in got] == [(t, r) for _, _, t, r in want]
    for h, (value, score, _, _) in zip(got, want):
        # 32-bit logits summed in another order, scores kept in 32 bits over the tokens
        assert abs(h.value - value) <= 1e-4 + 1e-4 * abs(value) and abs(h.score - score) <= 1e-4 + 1e-4 * abs(score)


def all_free(llm):
    c = llm.engine.cache
    return c.slots.n_free == c.n_slots and all(g.pool.n_free == g.pool.n_pages and not g.on_device and not g.slot_first for g in c.kv_groups)


@pytest.mark.parametrize("beams,penalty,early", [(1, 1.0, False), (3, 1.0, False), (4, 0.0, True), (2, 2.0, False)])
def test_search_matches_plain(cpu_llm, model_folders, beams, penalty, early):
    llm = cpu_llm("A", max_seq_len=128)
    prompts = prompts_for("A", [5, 1, 9, 64], seed=3)
    stops = [7, 100, 31]
    got = llm.beam_search(prompts, BeamParams(beams, penalty, early, beams), max_new_tokens=7, stop_token_ids=stops[1:])
    for p, g in zip(prompts, got):
        same(g, plain_search(model_folders["A"], p, beams, 7, stops=stops, length_penalty=penalty, early_stopping=early))
    assert all_free(llm) and llm.last_stats.batches == -(-4 // (8 // beams))


@pytest.mark.parametrize("name,lens,chunk", [("C", [61, 3], None), ("C", [126, 70], 50), ("B", [63, 64, 65], 40)])
def test_search_over_page_borders_and_windows(cpu_llm, model_folders, name, lens, chunk):
    """Prompts around page borders; model C has a window of 40 (a ring of one page) above its first layer."""
    llm = cpu_llm(name, max_seq_len=256, prefill_chunk=chunk, max_batch=6)
    prompts = prompts_for(name, lens, seed=4)
    got = llm.beam_search(prompts, BeamParams(3, n_best=3), max_new_tokens=6, ignore_eos=True)
    for p, g in zip(prompts, got):
        same(g, plain_search(model_folders[name], p, 3, 6))
    assert all_free(llm)


def test_limits_and_refusals(cpu_llm, model_folders):
    llm = cpu_llm("A", max_seq_len=16, max_batch=4)
    p = prompts_for("A", [14, 16, 3], seed=1)
    got = llm.beam_search(p, BeamParams(2, n_best=2), max_new_tokens=5, ignore_eos=True)
    same(got[0], plain_search(model_folders["A"], p[0], 2, 5, max_len=16))
    assert got[0][0].finish_reason == "context" and len(got[0][0].tokens) == 2
    assert got[1][0].finish_reason == "context" and got[1][0].tokens == []
    same(got[2], plain_search(model_folders["A"], p[2], 2, 5))
    assert [h.finish_reason for h in llm.beam_search(p[2:], BeamParams(2), max_new_tokens=0)[0]] == ["length"]
    for bad in (dict(beams=0), dict(beams=33), dict(length_penalty=-1.0), dict(length_penalty=6.0), dict(beams=2, n_best=3), dict(n_best=0)):
        with pytest.raises(ValueError):
            llm.beam_search(p[2:], BeamParams(**bad))
    with pytest.raises(ValueError):
        llm.beam_search(p[2:], BeamParams(5))                              # more than max_batch
    with pytest.raises(ValueError):
        llm.beam_search([[]], BeamParams(2))
    with pytest.raises(ValueError):
        llm.beam_search([[1] * 17], BeamParams(2))
    with pytest.raises(ValueError):
        llm.beam_search(p[2:], BeamParams(2), stop_token_ids=list(range(20)))
    small = cpu_llm("A", max_seq_len=128, max_batch=8, max_tokens=128)
    with pytest.raises(ValueError, match="do not fit"):
        small.beam_search(p[2:], BeamParams(4), max_new_tokens=100)
    assert all_free(small) and all_free(llm)


def test_a_failing_step_gives_everything_back(cpu_llm, monkeypatch):
    llm = cpu_llm("A", max_seq_len=64)
    step, calls = llm.engine.step, itertools.count()

    def failing(*a, **k):
        if next(calls) == 3:
            raise RuntimeError("stop here")
        return step(*a, **k)

    monkeypatch.setattr(llm.engine, "step", failing)
    with pytest.raises(RuntimeError, match="stop here"):
        llm.beam_search(prompts_for("A", [5, 6], seed=1), BeamParams(3), max_new_tokens=9, ignore_eos=True)
    assert all_free(llm)


def test_plan():
    assert plan_beams([64, 64, 64], 2, 1000) == [[0, 1], [2]]
    assert plan_beams([64, 640, 64], 8, 700) == [[0], [1], [2]] or plan_beams([64, 640, 64], 8, 704) == [[0, 1], [2]]
    assert plan_beams([], 2, 64) == []
    with pytest.raises(ValueError):
        plan_beams([128], 2, 64)


def test_pages_of_beams():
    """Every beam's own pages begin where the beams begin to write, are distinct there, and come back with the slots."""
    c = CacheManager([KVRequest(1, 8), KVRequest(1, 8, 100), StateRequest((3,))], 64 * 40, 6, 640, torch.float32, "cpu")
    full, ring = c.kv_groups
    for prompt, length, first, ring_first in ((130, 250, 2, 0), (64, 100, 1, 1), (5, 600, 0, 0), (63, 64, 0, 0), (64, 64, 1, 1)):
        slots = [c.allocate_slot() for _ in range(4)]
        before = full.pool.n_free, ring.pool.n_free
        c.reserve_beams(slots, prompt, length)
        pages = -(-length // 64)
        for g, f in ((full, first), (ring, ring_first)):
            n = g.pages_needed(length)
            assert g.beam_columns(prompt, length) == f
            rows = g.home[slots].numpy()
            assert np.array_equal(rows, g.table[slots].numpy())
            assert (rows[0, :n] > 0).all() and (rows[1:, f:n] > 0).all() and (rows[1:, :f] == 0).all()
            assert len(set(rows[:, f:n].reshape(-1))) == 4 * (n - f)
        assert before[0] - full.pool.n_free == pages + 3 * (pages - first)
        assert c.beam_tokens(prompt, length, 4) == 64 * max(before[0] - full.pool.n_free, before[1] - ring.pool.n_free)
        for s in slots:
            c.release(s)
        assert full.pool.n_free == 40 and not full.on_device and not full.slot_first
    with pytest.raises(CacheError):
        c.reserve_beams([0], 5, 10)
    s = c.allocate_slot()
    with pytest.raises(CacheError):
        c.reserve_beams([s], 5, 1000)


def test_other_sequences_do_not_touch_the_rows_of_beams():
    """The host uploads rows of page tables from the first to the last that changed: those that the device rewrites are not among them."""
    c = CacheManager([KVRequest(1, 8)], 64 * 40, 6, 640, torch.float32, "cpu")
    a = c.allocate_slot()
    beams = [c.allocate_slot() for _ in range(3)]
    b = c.allocate_slot()
    c.reserve_beams(beams, 10, 200)
    g = c.kv_groups[0]
    g.table[beams[1]] = g.table[beams[0]].clone()          # as the device does
    kept = g.table[beams].clone()
    c.reserve(a, 100)
    c.reserve(b, 100)
    c.flush()
    assert torch.equal(g.table[beams], kept)
    assert np.array_equal(g.table[a].numpy(), g.table_host[a]) and np.array_equal(g.table[b].numpy(), g.table_host[b])


def test_kernels_refuse_the_cpu():
    import importlib
    KB = importlib.import_module("toyinfer_b200.kernels.beam")
    x = torch.zeros(4, 10)
    i = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA"):
        KB.select(x, torch.zeros(2, 2), 2)
    with pytest.raises(KernelError, match="CUDA"):
        KB.tables(i, i, i[0], 0, [])
    with pytest.raises(KernelError, match="CUDA"):
        KB.Areas([x], [])


def test_cli_options():
    from toyinfer_b200.engine import cli
    for args in (["--beam_size", "0"], ["--beam_size", "40"], ["--length_penalty", "9"], ["--beam_size", "8", "--max_batch", "4"]):
        assert cli.main(["--model_dir", "nowhere", "--prompt_ids", "1"] + args) == 2
