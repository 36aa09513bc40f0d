"""The running sums of beam search over long searches: a choice hands its scores to the next one without rounding them at their own size."""
import math

import pytest
import torch

from deliverance_amd.kernels import ops
from deliverance_amd.kernels.ops import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0" if torch.cuda.is_available() else "cpu"


def chain(steps, beams, vocab, start, seed):
    """``steps`` choices, each on the scores that the one before left.  Returns the beams' scores and what the 64-bit sums are along the
    beams that were chosen."""
    g = torch.Generator().manual_seed(seed)
    scores = torch.full((beams,), start, device=DEV)
    low = torch.zeros(beams, device=DEV)
    sums = torch.full((beams,), start, dtype=torch.float64)
    ws = torch.empty(ops.beam_select_floats(beams, beams, vocab), device=DEV)
    for _ in range(steps):
        logits = torch.randn(beams, vocab, generator=g) * 2
        out, left = torch.full((1, beams), math.nan, device=DEV), torch.full((1, beams), math.nan, device=DEV)
        parents, tokens = torch.zeros(1, beams, dtype=torch.int32, device=DEV), torch.zeros(1, beams, dtype=torch.int32, device=DEV)
        ops.beam_select(logits.to(DEV), scores, beams, out, parents, tokens, ws, scores_low=low, out_scores_low=left)
        p, t = parents.cpu().long()[0], tokens.cpu().long()[0]
        sums = sums[p] + torch.log_softmax(logits.double(), 1)[p, t]
        scores, low = out[0], left[0]
    assert torch.equal((scores.cpu().double() + low.cpu().double()).float(), scores.cpu()), "the first part is the nearest 32-bit number"
    return scores.cpu().double() + low.cpu().double(), sums


# A logarithm of a sum of exponentials is off by less than 2^-21 (32-bit exponentials, four of them added in 32-bit); the two parts carry a sum to
# 2^-48 of itself.  (A 32-bit sum near -60,000 has steps of 2^-8: with it alone these are off by 1e-2 and more.)
@pytest.mark.parametrize("steps,vocab,start", [pytest.param(25, 200, -60000.0, marks=pytest.mark.simt_quick), (3000, 5000, 0.0)])
def test_a_chain_of_choices_keeps_the_64_bit_sum(steps, vocab, start):
    got, want = chain(steps, 3, vocab, start, seed=steps)
    assert float((got - want).abs().max()) <= steps * (2.0 ** -21 + 2.0 ** -48 * float(want.abs().max()))


@pytest.mark.simt_quick
def test_scores_without_a_number_behind_them():
    """What an infinite score leaves is 0, and a place without a beam stays one whatever its second part is."""
    logits = torch.randn(4, 70, generator=torch.Generator().manual_seed(2)).to(DEV)
    scores = torch.tensor([-math.inf, -3.0, math.inf, -math.inf], device=DEV)
    low = torch.tensor([0.0, 2.0 ** -24, 0.0, math.nan], device=DEV)
    out, left = torch.full((2, 90), math.nan, device=DEV), torch.full((2, 90), math.nan, device=DEV)
    parents, tokens = torch.zeros(2, 90, dtype=torch.int32, device=DEV), torch.zeros(2, 90, dtype=torch.int32, device=DEV)
    ops.beam_select(logits, scores, 2, out, parents, tokens, torch.empty(ops.beam_select_floats(4, 2, 70), device=DEV), scores_low=low,
                    out_scores_low=left)
    assert parents.cpu().tolist() == [[1] * 70 + [-1] * 20, [0] * 70 + [-1] * 20]
    want = torch.sort(torch.log_softmax(logits[1].cpu().double(), 0) - 3.0 + 2.0 ** -24, descending=True).values
    got = out.cpu().double() + left.cpu().double()
    assert float((got[0, :70] - want).abs().max()) <= 2.0 ** -21
    assert bool((out[1, :70] == math.inf).all()) and bool((out[:, 70:] == -math.inf).all())
    assert bool((left[1] == 0).all()) and bool((left[0, 70:] == 0).all())


def test_refusals_of_second_parts():
    logits, scores = torch.zeros(6, 40, device=DEV), torch.zeros(6, device=DEV)
    out = (torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    ws = torch.zeros(ops.beam_select_floats(6, 3, 40), device=DEV)
    for bad in (dict(scores_low=scores[:5]), dict(scores_low=scores.double()), dict(scores_low=torch.zeros(12, device=DEV)[::2]),
                dict(out_scores_low=out[0].double()), dict(out_scores_low=out[0][:1]), dict(out_scores_low=torch.zeros(4, 2, device=DEV).t())):
        with pytest.raises(KernelError):
            ops.beam_select(logits, scores, 3, *out, ws, **bad)


@pytest.mark.needs_device
@pytest.mark.parametrize("graphs", [True, False])
def test_a_long_search_returns_the_sum_of_its_tokens(graphs, tmp_path):
    """1,500 tokens: a hypothesis' score is the sum that the plain model gives its tokens.  A logit here is a 32-bit sum of 64 products and of
    size 2: its error is about the root of 64 roundings of 2^-24 of that, 1e-6 at the most and half of it on average, and not of one sign.  (A sum
    kept in 32 bits rounds by up to 2^-12 a token at -4,096 to -8,192: it was off by 1.6e-3.)"""
    import numpy as np
    import helpers
    import plain_gpt2 as P
    from deliverance_amd import AutoModelForCausalLM, BeamParameters
    m = helpers.make_model(tmp_path, dict(helpers.CONFIG_A, n_positions=2048), seed=5)
    eng = AutoModelForCausalLM.from_pretrained(str(m.folder), dtype="float32", use_graphs=graphs, max_cached_tokens=8192, max_num_seqs=4)
    prompt = m.prompt(9)
    out = eng.beam_search(prompt, BeamParameters(num_beams=2, max_tokens=1500, ignore_eos=True))
    for h in out.hypotheses:
        z = np.asarray(P.forward_logits(m.plain_cfg, m.W, prompt + h.tokens[:-1]), dtype=np.float64)[len(prompt) - 1:]
        z -= z.max(1, keepdims=True)
        want = float((z[np.arange(1500), h.tokens] - np.log(np.exp(z).sum(1))).sum())
        assert abs(h.score - want) <= 1500 * 5e-7


@pytest.mark.needs_device
def test_a_search_takes_the_kernel_that_its_positions_pay_for(tmp_path, monkeypatch):
    """A model of 2,048 positions: short contexts stay with the decode kernel however wide the tables are, and a search that grows goes over to
    the kernel that reads shared pages once; a step of either kind is recorded for itself."""
    import numpy as np
    import helpers
    import plain_gpt2 as P
    from deliverance_amd import AutoModelForCausalLM, BeamParameters
    m = helpers.make_model(tmp_path, dict(helpers.CONFIG_A, n_positions=2048), seed=5)
    calls, kernel = [], ops.attention_beams
    monkeypatch.setattr(ops, "attention_beams", lambda *a, **k: (calls.append(1), kernel(*a, **k))[1])
    eng = AutoModelForCausalLM.from_pretrained(str(m.folder), dtype="float32", max_cached_tokens=8192, max_num_seqs=4)
    eng.beam_search(m.prompt(20), BeamParameters(num_beams=3, max_tokens=10, ignore_eos=True))
    assert not calls
    prompt = m.prompt(380)
    out = eng.beam_search(prompt, BeamParameters(num_beams=3, max_tokens=120, ignore_eos=True))
    assert calls and {bool(k[3]) for k in eng.runner._graphs if isinstance(k, tuple)} == {False, True}
    for h in out.hypotheses:
        z = np.asarray(P.forward_logits(m.plain_cfg, m.W, prompt + h.tokens[:-1]), dtype=np.float64)[len(prompt) - 1:]
        z -= z.max(1, keepdims=True)
        want = float((z[np.arange(120), h.tokens] - np.log(np.exp(z).sum(1))).sum())
        assert abs(h.score - want) <= 120 * 5e-7 + 2e-5


@pytest.mark.needs_device
def test_searches_of_many_kinds_keep_few_recordings(models):
    """One engine, searches of many numbers of beams and prompts, and the first of them again when its recording has gone."""
    from deliverance_amd import AutoModelForCausalLM, BeamParameters, GeneratorParameters
    m = models["A"]
    eng = AutoModelForCausalLM.from_pretrained(m.folder, dtype="float32", max_cached_tokens=2048, max_num_seqs=15)
    eng.runner.MAX_BEAM_RECORDINGS = 3
    greedy = eng.generate(m.prompt(5), GeneratorParameters(max_tokens=4, ignore_eos=True)).generated_tokens
    prompts = [m.prompt(n) for n in (5, 9, 17)]
    found = {}
    for beams, n in ((4, 1), (2, 2), (3, 3), (5, 3), (2, 1), (4, 1), (5, 3), (1, 3)):
        out = eng.beam_search(prompts[:n], BeamParameters(num_beams=beams, max_tokens=6, ignore_eos=True))
        for k, r in enumerate(out):
            assert found.setdefault((beams, k), [h.tokens for h in r.hypotheses]) == [h.tokens for h in r.hypotheses]
        keys = [k for k in eng.runner._graphs if isinstance(k, tuple)]
        assert len(keys) <= 3 and all(k[0] <= 15 for k in keys)
    assert eng.generate(m.prompt(5), GeneratorParameters(max_tokens=4, ignore_eos=True)).generated_tokens == greedy
