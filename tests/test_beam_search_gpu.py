"""Beam search through the entry point and the command line on the GPU, against the plain search, which runs every prefix whole: the
dense model with and without graphs, windows whose rings wrap, and architectures with latents, windows and states."""
from __future__ import annotations

import importlib
import json
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT, TINY, prompts_for
from plain import beam_plain
from plain import qwen3_plain as plain

pytestmark = pytest.mark.gpu


def plain_search(folder, prompt, beams, max_new, **kw):
    w, cfg = plain.read_weights(folder), plain.read_config(folder)
    return beam_plain.search(lambda ids: plain.forward(w, cfg, ids)[-1].float().numpy(), prompt, beams, max_new, **kw)


def same(got, want):
    assert [(h.tokens, h.finish_reason) for h in got] == [(t, r) for _, _, t, r in want]
    for h, (value, score, _, _) in zip(got, want):
        assert abs(h.value - value) <= 1e-3 + 1e-3 * abs(value) and abs(h.score - score) <= 1e-3 + 1e-3 * abs(score)


def all_free(llm):
    c = llm.engine.cache
    return c.slots.n_free == c.n_slots and all(g.pool.n_free == g.pool.n_pages and not g.on_device for g in c.kv_groups)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("name,lens,beams,max_new", [("A", [5, 9, 64], 4, 8), ("B", [60, 1], 3, 12), ("C", [61, 126], 5, 10), ("E", [120, 63], 2, 20)])
def test_search_matches_plain(model_folders, graph, name, lens, beams, max_new):
    from toyinfer_b200 import LLM, BeamParams
    stops = [7, 30, 31] if name == "A" else []
    llm = LLM(model_folders[name], dtype="float32", max_seq_len=min(256, TINY[name]["max_position_embeddings"]), max_batch=16, max_tokens=4096,
              enable_cuda_graph=graph)
    prompts = prompts_for(name, lens, seed=8)
    for _ in range(2):                 # the second time on slots and pages that have been used
        got = llm.beam_search(prompts, BeamParams(beams, n_best=beams), max_new_tokens=max_new, stop_token_ids=stops or None, ignore_eos=not stops)
        for p, g in zip(prompts, got):
            same(g, plain_search(model_folders[name], p, beams, max_new, stops=stops))
        assert all_free(llm)


@pytest.mark.parametrize("penalty,early,chunk,dedicated", [(1.0, False, None, True), (0.0, True, 20, True), (2.5, False, 7, True), (0.7, False, None, False)])
def test_requests_that_end_at_different_steps(model_folders, penalty, early, chunk, dedicated):
    """Many stop tokens, more requests than a batch holds, prompts in pieces or token by token: requests leave a running batch while the
    others' next step is under way, and some meet the engine's length limit."""
    from toyinfer_b200 import LLM, BeamParams
    llm = LLM(model_folders["B"], dtype="float32", max_seq_len=96, max_batch=10, max_tokens=2048, prefill_chunk=chunk, use_dedicated_prefill=dedicated)
    prompts = prompts_for("B", [20, 60, 90, 5, 64, 1, 33], seed=12)
    stops = [11, 12] + list(range(100, 112))             # the model's own two and more
    got = llm.beam_search(prompts, BeamParams(3, penalty, early, 3), max_new_tokens=14, stop_token_ids=stops)
    ends = set()
    for p, g in zip(prompts, got):
        same(g, plain_search(model_folders["B"], p, 3, 14, stops=stops, length_penalty=penalty, early_stopping=early, max_len=96))
        ends.add(max(len(h.tokens) for h in g))
    assert len(ends) > 1 and any(h.finish_reason == "context" for g in got for h in g) and llm.last_stats.batches == 3
    assert all_free(llm)


def test_one_beam_is_greedy_and_batches_do_not_matter(model_folders):
    from toyinfer_b200 import LLM, BeamParams, SamplingParams
    llm = LLM(model_folders["B"], dtype="float32", max_seq_len=256, max_batch=8, max_tokens=4096)
    prompts = prompts_for("B", [17, 64, 3, 130, 40], seed=2)
    greedy = [r.tokens for r in llm.generate(prompts, SamplingParams(temperature=0.0), max_new_tokens=9, ignore_eos=True)]
    assert [g[0].tokens for g in llm.beam_search(prompts, BeamParams(1), max_new_tokens=9, ignore_eos=True)] == greedy
    together = llm.beam_search(prompts, BeamParams(4, n_best=4), max_new_tokens=9, ignore_eos=True)
    alone = [llm.beam_search([p], BeamParams(4, n_best=4), max_new_tokens=9, ignore_eos=True)[0] for p in prompts]
    assert [[h.tokens for h in g] for g in together] == [[h.tokens for h in g] for g in alone]


def test_sequences_beside_a_search_keep_their_rows(model_folders):
    """A sequence of the caller's own lives on through a search: its logits are those of its tokens alone."""
    from toyinfer_b200 import LLM, BeamParams
    llm = LLM(model_folders["B"], dtype="float32", max_seq_len=256, max_batch=8, max_tokens=8192)
    e = llm.engine
    ids = prompts_for("B", [100], seed=6)[0]
    slot = e.new_sequence()
    e.step([(slot, ids[:62])])
    p = prompts_for("B", [30, 70], seed=7)
    llm.beam_search(p, BeamParams(4), max_new_tokens=5, ignore_eos=True)
    got = e.step([(slot, ids[62:])], [[37]]).clone()
    w, cfg = plain.read_weights(model_folders["B"]), plain.read_config(model_folders["B"])
    torch.testing.assert_close(got[0].cpu(), plain.forward(w, cfg, ids)[-1].float(), rtol=1e-3, atol=1e-3)
    e.end_sequence(slot)
    same(llm.beam_search(p[1:], BeamParams(4, n_best=4), max_new_tokens=5, ignore_eos=True)[0], plain_search(model_folders["B"], p[1], 4, 5))


FAMILIES = ("kadodra", "tusasun", "bagasun", "bolisun", "mikipel", "vobolorn")


@pytest.mark.parametrize("family,name", [(f, n) for f in FAMILIES for n in importlib.import_module(f"{f}_cases").CASES])
def test_scores_are_those_of_the_tokens(family, name, tmp_path):
    """Models with states, latents and windows: a hypothesis's score is what its tokens score when they run through the engine as one
    sequence (the beams' states and pages were theirs all along)."""
    from toyinfer_b200 import LLM, BeamParams
    cases = importlib.import_module(f"{family}_cases")
    cases.write_folder(name, str(tmp_path))
    llm = LLM(str(tmp_path), dtype="float32", max_batch=8, max_tokens=4096, max_seq_len=256)
    prompts = cases.prompts(name, [61, 20], seed=3)
    got = llm.beam_search(prompts, BeamParams(4, n_best=4), max_new_tokens=8, ignore_eos=True)
    e = llm.engine
    for p, hyps in zip(prompts, got):
        assert len({tuple(h.tokens) for h in hyps}) == 4
        for h in hyps:
            slot = e.new_sequence()
            logits = e.step([(slot, p + h.tokens)], [list(range(len(p) - 1, len(p) + 7))])
            lp = torch.log_softmax(logits.double().cpu(), -1).gather(1, torch.tensor(h.tokens)[:, None]).sum().item()
            e.end_sequence(slot)
            assert abs(lp - h.score) <= 2e-3 + 2e-4 * abs(lp), (family, lp, h.score)
    assert all_free(llm)


def test_bfloat16_heads_of_128_and_long_prompts(model_folders):
    """The tensor-core decode attention over shared pages: scores against the plain model's in 32 bits."""
    from toyinfer_b200 import LLM, BeamParams
    llm = LLM(model_folders["D"], dtype="bfloat16", max_seq_len=640, max_batch=16, max_tokens=16384, prefill_chunk=200)
    prompts = prompts_for("D", [500, 127, 64], seed=9)
    got = llm.beam_search(prompts, BeamParams(5, n_best=5), max_new_tokens=70, ignore_eos=True)
    e = llm.engine
    for p, hyps in zip(prompts, got):
        for h in hyps[:2]:
            assert len(h.tokens) == 70
            slot = e.new_sequence()
            logits = e.step([(slot, p + h.tokens)], [list(range(len(p) - 1, len(p) + 69))])
            lp = torch.log_softmax(logits.double().cpu(), -1).gather(1, torch.tensor(h.tokens)[:, None]).sum().item()
            e.end_sequence(slot)
            # bfloat16 activations: each token's log-probability differs by a few hundredths between a whole prompt and single steps
            assert abs(lp - h.score) <= 70 * 0.04, (lp, h.score)
    assert all_free(llm)


def test_command_line(model_folders):
    env = dict(os.environ, PYTHONPATH=ROOT)
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "toyinfer"), "--model_dir", model_folders["A"], "--dtype", "float32",
                          "--max_seq_len", "128", "--prompt_ids", "5,6,7;1,2", "--max_new_tokens", "6", "--beam_size", "3",
                          "--length_penalty", "0.5", "--ignore_eos", "1"], capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = [json.loads(x) for x in out.stdout.splitlines() if x.startswith("{")]
    for line, p in zip(lines, ([5, 6, 7], [1, 2])):
        want = plain_search(model_folders["A"], p, 3, 6, length_penalty=0.5)[0]
        assert line["tokens"] == want[2] and abs(line["score"] - want[1]) < 1e-3
