"""Beam search through the engine's entry point against a plain search over the plain models' logits."""
import dataclasses
import importlib
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import plain_beams

pytestmark = [pytest.mark.gpu, pytest.mark.needs_device]
ROOT = os.path.normpath(os.path.join(os.path.dirname(__file__), ".."))

DESIGNS = {"virudra": ("virudra_models", "CONFIG_X"), "pedatar": ("pedatar_models", "CONFIG_P"), "pafolorn": ("pafolorn_models", "CONFIG_F"),
           "salivik": ("salivik_models", "CONFIG_S"), "luvatar": ("luvatar_models", "CONFIG_A"), "mogevik": ("mogevik_models", "CONFIG_D")}


def load(folder, dtype="float32", **kw):
    from deliverance_amd import AutoModelForCausalLM
    kw.setdefault("max_cached_tokens", 1024)
    kw.setdefault("max_num_seqs", 16)
    return AutoModelForCausalLM.from_pretrained(str(folder), dtype=dtype, **kw)


def log_probability(logits_of, prompt, tokens):
    total = 0.0
    for i, t in enumerate(tokens):
        z = np.asarray(logits_of(list(prompt) + list(tokens[:i])), dtype=np.float64)
        total += z[t] - z.max() - math.log(np.exp(z - z.max()).sum())
    return total


def check(response, logits_of, prompt, n_beams, max_new, ends=(), slack=2e-4, **options):
    """Every hypothesis has the plain log-probability of its tokens (32-bit logits are off by some 1e-6 a token), and where the plain
    search's own choices are further apart than that they are its hypotheses."""
    want, gap = plain_beams.beam_search(logits_of, prompt, n_beams, max_new, ends, **options)
    got = response.hypotheses
    assert len(got) == len(want) and response.prompt_tokens == len(prompt)
    for h in got:
        assert abs(h.score - log_probability(logits_of, prompt, h.tokens)) <= slack
    assert abs(got[0].rank - want[0][0]) <= slack or gap <= slack
    if gap > slack:
        assert [h.tokens for h in got] == [t for _, _, t in want]
    return gap > slack


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("n_beams", [1, 3, 4])
def test_beam_search_is_the_plain_one(models, n_beams, graphs):
    import plain_gpt2 as P
    from deliverance_amd import BeamParameters
    m = models["A"]
    eng = load(m.folder, use_graphs=graphs)
    prompts, told = [m.prompt(n) for n in (5, 16, 33)], 0
    outs = eng.beam_search(prompts, BeamParameters(num_beams=n_beams, max_tokens=14))
    for prompt, out in zip(prompts, outs):
        told += check(out, lambda ids: P.forward_logits(m.plain_cfg, m.W, ids)[-1], prompt, n_beams, 14, (511,))
    assert told, "no prompt's choices were far enough apart to compare"
    eng.cache.manager.check()
    assert eng.cache.manager.live() == []
    # the same again, one prompt alone, and sampling still works beside it
    from deliverance_amd import GeneratorParameters
    alone = eng.beam_search(prompts[1], BeamParameters(num_beams=n_beams, max_tokens=14))
    assert [h.tokens for h in alone.hypotheses] == [h.tokens for h in outs[1].hypotheses]
    greedy = eng.generate(prompts[0], GeneratorParameters(max_tokens=6, ignore_eos=True))
    assert greedy.generated_tokens == P.greedy_generate(m.plain_cfg, m.W, prompts[0], 6)


@pytest.mark.parametrize("name", sorted(DESIGNS))
def test_beam_search_with_states_windows_and_chunks(name, tmp_path):
    """Designs that keep recurrent states, windows, chunks or latent rows: what a beam keeps follows it."""
    from deliverance_amd import BeamParameters
    from deliverance_amd.random_model import random_model
    module, attr = DESIGNS[name]
    cfg = getattr(importlib.import_module(module), attr)
    plain = importlib.import_module(f"plain_{name}")
    random_model(str(tmp_path), cfg, seed=21)
    pcfg, W = plain.read_model_folder(str(tmp_path))
    prompt = [int(t) for t in np.random.default_rng(3).integers(0, cfg["vocab"], size=29)]
    eng = load(tmp_path, poison_freed_pages=True)
    out = eng.beam_search(prompt, BeamParameters(num_beams=3, max_tokens=24, ignore_eos=True))
    check(out, lambda ids: plain.forward_logits(pcfg, W, ids)[-1], prompt, 3, 24)
    assert all(len(h.tokens) == 24 for h in out.hypotheses)
    eng.cache.manager.check()


def test_beam_search_in_bfloat16_scores_its_own_tokens(models):
    """bfloat16 may choose otherwise where two tokens are near; what it returns has that probability within the logits' rounding (4 %
    of their root mean square a token, the bound that the replay tests hold every bfloat16 logit to, twice for the sum's)."""
    import plain_gpt2 as P
    from deliverance_amd import BeamParameters
    m = models["A"]
    eng = load(m.folder, "bfloat16")
    prompt = m.prompt(40)
    logits_of = lambda ids: P.forward_logits(m.plain_cfg, m.W, ids)[-1]  # noqa: E731
    out = eng.beam_search(prompt, BeamParameters(num_beams=4, max_tokens=20, ignore_eos=True))
    near = 20 * 2 * 0.04 * float(np.sqrt((logits_of(prompt) ** 2).mean()))
    for h in out.hypotheses:
        assert abs(h.score - log_probability(logits_of, prompt, h.tokens)) <= near


@pytest.mark.parametrize("dtype,graphs,page", [("float32", True, 16), ("float32", False, 32), ("bfloat16", True, 64)])
def test_long_prompts_read_what_beams_share_once(dtype, graphs, page, tmp_path, monkeypatch):
    import helpers
    import plain_gpt2 as P
    from deliverance_amd import BeamParameters
    from deliverance_amd.kernels import ops
    m = helpers.make_model(tmp_path, dict(helpers.CONFIG_A, n_positions=2048), seed=5)
    calls = []
    kernel = ops.attention_beams
    monkeypatch.setattr(ops, "attention_beams", lambda *a, **k: (calls.append(1), kernel(*a, **k))[1])
    eng = load(m.folder, dtype, use_graphs=graphs, max_cached_tokens=8192, page_size=page)
    prompts = [m.prompt(n) for n in (530, 547)]
    outs = eng.beam_search(prompts, BeamParameters(num_beams=3, max_tokens=9))
    assert calls
    logits_of = lambda ids: P.forward_logits(m.plain_cfg, m.W, ids)[-1]  # noqa: E731
    for prompt, out in zip(prompts, outs):
        if dtype == "float32":
            check(out, logits_of, prompt, 3, 9, (511,))
        else:
            near = 9 * 2 * 0.04 * float(np.sqrt((logits_of(prompt) ** 2).mean()))
            assert all(abs(h.score - log_probability(logits_of, prompt, h.tokens)) <= near for h in out.hypotheses)


def test_prompts_wait_for_pages_and_places(models):
    import plain_gpt2 as P
    from deliverance_amd import BeamParameters
    m = models["A"]
    # ten pages: one prompt of 20 tokens with 3 beams of 12 more needs 1 + 3 * 1 pages; two live at a time by places
    eng = load(m.folder, max_cached_tokens=160, max_num_seqs=6, max_batch_tokens=16, max_chunk=7)
    prompts = [m.prompt(20) for _ in range(5)]
    outs = eng.beam_search(prompts, BeamParameters(num_beams=3, max_tokens=12))
    for p, o in zip(prompts, outs):
        check(o, lambda ids: P.forward_logits(m.plain_cfg, m.W, ids)[-1], p, 3, 12, (511,))
    assert eng.cache.manager.stats()["pages_free"] == [10]


def test_an_end_token_finishes_a_hypothesis(models):
    import plain_gpt2 as P
    from deliverance_amd import BeamParameters
    m = models["A"]
    eng = load(m.folder)
    prompt = m.prompt(9)
    logits_of = lambda ids: P.forward_logits(m.plain_cfg, m.W, ids)[-1]  # noqa: E731
    best = eng.beam_search(prompt, BeamParameters(num_beams=4, max_tokens=10, ignore_eos=True)).hypotheses
    end = best[1].tokens[4]                                 # a token that the search meets becomes the end
    eng.config = dataclasses.replace(eng.config, eos_token_ids=(end,))
    stopped = 0
    for options in ({}, {"length_penalty": 0.5}, {"early_stopping": True}, {"length_penalty": -1.0}):     # (the last prefers short ones)
        out = eng.beam_search(prompt, BeamParameters(num_beams=4, max_tokens=10, **options))
        check(out, logits_of, prompt, 4, 10, (end,), **options)
        assert all((h.finish_reason == "stop") == (h.tokens[-1] == end) for h in out.hypotheses)
        stopped += sum(h.finish_reason == "stop" for h in out.hypotheses)
    assert stopped


def test_refusals(models):
    from deliverance_amd import BeamParameters
    m = models["A"]
    eng = load(m.folder, max_cached_tokens=64, max_num_seqs=4)
    for prompt, p in (([1], BeamParameters(num_beams=5)), ([1] * 40, BeamParameters(num_beams=4, max_tokens=40)), ([], BeamParameters()),
                      ([1] * 128, BeamParameters()), ([600], BeamParameters()), ([1], BeamParameters(ntokens=1000)), ([1, 2], BeamParameters(num_beams=0))):
        with pytest.raises(ValueError):
            eng.beam_search([prompt], p)
    assert eng.beam_search([], BeamParameters()) == []
    eng.add_request([1, 2, 3])
    with pytest.raises(RuntimeError, match="without other requests"):
        eng.beam_search([1, 2])


def test_beam_search_from_the_command_line(models, tmp_path):
    m = models["A"]
    out = tmp_path / "out.jsonl"
    p = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "deliverance"), "generate", "--model", m.folder, "--prompt-ids", "5,17,3",
                        "--num-beams", "3", "--max-tokens", "8", "--working-dtype", "F32", "--max-cached-tokens", "512", "--jsonl-output", str(out)],
                       capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr
    row = json.loads(out.read_text())
    assert len(row["hypotheses"]) == 3 and [int(t) for t in p.stdout.strip().split(",")] == row["hypotheses"][0]["token_ids"]


def test_profile_of_a_beam_search(models):
    p = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "deliverance"), "generate", "--model", models["A"].folder, "--prompt-ids", "5,17,3",
                        "--num-beams", "3", "--max-tokens", "8", "--ignore-eos", "--working-dtype", "F32", "--max-cached-tokens", "512", "--profile-stages"],
                       capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr
    assert all(word in p.stderr for word in ("profile summary", "beam_search.prompts", "beam_search.step", "beam_select", "state_reorder"))


@pytest.mark.parametrize("graphs", [True, False])
def test_windows_and_grouped_heads_read_what_beams_share_once(graphs, tmp_path, monkeypatch):
    """A design with short and long windows and several query heads a key head, recurrent mixers beside them: its attention sent to the kernel
    that reads shared pages once whatever the estimate says, over pages that windows give back."""
    from deliverance_amd import BeamParameters
    from deliverance_amd.kernels import ops
    from deliverance_amd.random_model import random_model
    from pafolorn_models import attention, delta, parallel_layer
    import plain_pafolorn as plain
    cfg = {"architecture": "Pafolorn", "vocab": 300, "width": 64, "norm": {"eps": 1e-5}, "logit_scale": 0.7,
           "layers": [parallel_layer(attention(4, 2, 32, 32, 0.18, 40, 0, 10000.0, 16), delta(4, 2, 16, 32, 4), 1.3, 0.8, ff=96),
                      parallel_layer(attention(8, 2, 16, 16, 0.25, 4096, 0, 500.0, 16), delta(2, 2, 16, 16, 2), 1.0, 1.0)]}
    random_model(str(tmp_path), cfg, seed=23)
    pcfg, W = plain.read_model_folder(str(tmp_path))
    calls, kernel = [], ops.attention_beams
    monkeypatch.setattr(ops, "attention_beams", lambda *a, **k: (calls.append((a[6], a[8])), kernel(*a, **k))[1])
    monkeypatch.setattr(ops, "attention_beams_pays", lambda *a, **k: True)
    eng = load(tmp_path, use_graphs=graphs, poison_freed_pages=True)
    prompts = [[int(t) for t in np.random.default_rng(n).integers(0, 300, size=n)] for n in (29, 101)]
    outs = eng.beam_search(prompts, BeamParameters(num_beams=3, max_tokens=40, ignore_eos=True))
    assert set(calls) == {(4, 40), (8, 4096)}
    for prompt, out in zip(prompts, outs):
        check(out, lambda ids: plain.forward_logits(pcfg, W, ids)[-1], prompt, 3, 40)
    eng.cache.manager.check()
    assert eng.cache.manager.live() == []
