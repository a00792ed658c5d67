"""What a search attends to, through its shared and moved pages, against sequences that have their pages to themselves."""
from __future__ import annotations

import importlib

import pytest
import torch

from conftest import prompts_for
from plain import beam_plain

pytestmark = pytest.mark.gpu


def log_prob(logits, token):
    return torch.log_softmax(logits.double().cpu(), -1)[token].item()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name,dtype,lens,max_new", [("D", "bfloat16", [500, 127, 64], 70), ("D", "float32", [60, 129, 3], 70), ("C", "bfloat16", [30, 100, 1], 70)])
def test_scores_are_those_of_the_same_steps_without_sharing(model_folders, name, dtype, lens, max_new, graph):
    """Every hypothesis runs again as a sequence of its own, in steps of the same shapes: the prompts as the search ran them, then single
    tokens of as many sequences.  A row of a step depends on its own sequence and the step's shape alone, so the logits are the same to
    the bit, whichever pages they come from, and scores differ by the selections' sums only: 5e-11 and a rounding of 2^-44 a token.  A row
    of a page that was not moved, or was moved short, shows."""
    from toyinfer_b200 import LLM, BeamParams
    llm = LLM(model_folders[name], dtype=dtype, max_seq_len=640 if name == "D" else 256, max_batch=16, max_tokens=16384, enable_cuda_graph=graph)
    e = llm.engine
    prompts = prompts_for(name, lens, seed=9)
    B = 5
    for _ in range(3 if graph else 1):           # with graphs: until the prompts' step is captured
        got = llm.beam_search(prompts, BeamParams(B, n_best=B), max_new_tokens=max_new, ignore_eos=True)
    assert all(len(h.tokens) == max_new for g in got for h in g) and all(len(g) == B for g in got)
    slots = [[e.new_sequence() for _ in range(B)] for _ in prompts]
    sums = [[0.0] * B for _ in prompts]
    for j in range(B):
        logits = e.step([(s[j], p) for s, p in zip(slots, prompts)])
        for i, g in enumerate(got):
            sums[i][j] += log_prob(logits[i], g[j].tokens[0])
    for k in range(max_new - 1):
        logits = e.step([(slots[i][j], [g[j].tokens[k]]) for i, g in enumerate(got) for j in range(B)])
        for i, g in enumerate(got):
            for j in range(B):
                sums[i][j] += log_prob(logits[i * B + j], g[j].tokens[k + 1])
    for of_prompt in slots:
        for s in of_prompt:
            e.end_sequence(s)
    for i, g in enumerate(got):
        for j, h in enumerate(g):
            assert abs(h.score - sums[i][j]) <= max_new * (5e-11 + 2 ** -44) + 1e-9, (i, j, h.score, sums[i][j])


FAMILIES = ("kadodra", "tusasun", "bagasun", "bolisun", "mikipel", "vobolorn")


@pytest.mark.parametrize("family,name", [(f, n) for f in FAMILIES for n in importlib.import_module(f"{f}_cases").CASES])
def test_hypotheses_are_those_of_a_search_that_runs_every_prefix_whole(family, name, tmp_path):
    """Models with states, latents and windows: not only do scores belong to their tokens, the tokens are the best ones."""
    from toyinfer_b200 import LLM, BeamParams
    cases = importlib.import_module(f"{family}_cases")
    cases.write_folder(name, str(tmp_path))
    llm = LLM(str(tmp_path), dtype="float32", max_batch=8, max_tokens=4096, max_seq_len=256)
    e = llm.engine

    def logits_of(ids):
        slot = e.new_sequence()
        logits = e.step([(slot, ids)])[0].cpu().numpy().copy()
        e.end_sequence(slot)
        return logits

    for p in cases.prompts(name, [61, 20], seed=5):
        got = llm.beam_search([p], BeamParams(3, n_best=3), max_new_tokens=6, ignore_eos=True)[0]
        want = beam_plain.search(logits_of, p, 3, 6)
        assert [h.tokens for h in got] == [t for _, _, t, _ in want]
        for h, (_, score, _, _) in zip(got, want):
            assert abs(h.score - score) <= 1e-3 + 1e-3 * abs(score)
