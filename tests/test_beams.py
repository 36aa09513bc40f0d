"""Beam search's host side (no GPU): requests that continue one another in the cache manager, and the search for one prompt."""
import math
import random

import numpy as np
import pytest

import plain_beams
from deliverance_amd.cache import CacheError, CacheManager, KVGroupSpec, OutOfPages, PagePool, StateSpec


def manager(pages=40, slots=0, window=None):
    return CacheManager([KVGroupSpec((0, 1), 2, 16, None), KVGroupSpec((2,), 2, 16, window)], 4, [pages, pages], [StateSpec(3, 5)] if slots else [], slots)


def test_shared_pages_go_back_with_their_last_holder():
    p = PagePool(3)
    a = p.take(2, "a")
    p.share(a, "b")
    p.share([a[0]], "c")
    with pytest.raises(CacheError, match="already"):
        p.share([a[0]], "c")
    with pytest.raises(CacheError, match="nobody's"):
        p.share([2], "b")
    with pytest.raises(CacheError, match="belongs to"):
        p.give([a[1]], "c")
    assert p.give(a, "a") == [] and p.n_free == 1
    assert p.owner_of(a[1]) == "b" and not p.held_by(a[0], "a")
    assert p.give([a[1]], "b") == [a[1]] and p.give([a[0]], "c") == [] and p.give([a[0]], "b") == [a[0]]
    with pytest.raises(CacheError, match="freed twice"):
        p.give([a[0]], "b")
    assert p.n_free == 3 and p._holders == {}


def test_a_fork_shares_full_pages_and_writes_its_own():
    m = manager(slots=3)
    m.open("a")
    m.extend("a", 10)
    with pytest.raises(CacheError, match="reserved"):
        m.fork("a", "b")
    m.commit("a")
    m.fork("a", "b")
    m.check()
    assert m.length("b") == 10 and m.table("b", 0)[:2] == m.table("a", 0)[:2] and m.table("b", 0)[2] != m.table("a", 0)[2]
    assert m.writing("a", 0) == m.table("a", 0)[2] and m.state_slot("a") != m.state_slot("b")
    freed = []
    m.on_release = lambda g, pages: freed.extend((g, p) for p in pages)
    shared, own = m.table("a", 0)[:2], m.table("a", 0)[2]
    m.close("a")
    assert (0, own) in freed and not any((0, p) in freed for p in shared)
    m.check()
    m.close("b")
    m.check()
    assert m.stats()["pages_free"] == [40, 40] and m.stats()["state_slots_free"] == 3


def test_a_fork_at_a_pages_end_takes_no_page():
    m = manager(pages=2)
    m.open("a")
    m.extend("a", 8)
    m.commit("a")
    m.fork("a", "b")
    assert m.table("b", 0) == m.table("a", 0) and m.writing("b", 0) == -1
    with pytest.raises(OutOfPages):
        m.extend("b", 1)
    m.check()


def test_a_fork_that_does_not_fit_changes_nothing():
    m = manager(pages=3)
    m.open("a")
    m.extend("a", 9)
    m.commit("a")
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    assert m.live() == ["a"]
    m.check()


@pytest.mark.parametrize("window", [None, 5])
@pytest.mark.parametrize("seed", range(6))
def test_tables_follow_their_parents(seed, window):
    """Random searches against a plain record of what every beam's positions are.  A page stands for the contents written there; the
    page that is being written is copied as the device does it."""
    rng = random.Random(seed)
    m = manager(pages=200, slots=8, window=window)
    B = rng.randint(2, 5)
    rids, rows, plain = [f"b{i}" for i in range(B)], [{}, {}], [[] for _ in range(B)]
    m.on_release = lambda g, pages: [rows[g].pop((p, i), None) for p in pages for i in range(4)]

    def write(rid, k, values):
        start = m.extend(rid, len(values))
        for g in (0, 1):
            for i, s in enumerate(m.slots_for(rid, g, start, len(values))):
                rows[g][(s // 4, s % 4)] = values[i]
        plain[k] += values

    m.open(rids[0])
    write(rids[0], 0, [rng.random() for _ in range(rng.randint(1, 9))])
    m.commit(rids[0])
    for r in rids[1:]:
        m.fork(rids[0], r)

    def reorder(parents):
        old = [[m.writing(r, g) for r in rids] for g in (0, 1)]
        m.reorder(rids, parents)
        for g in (0, 1):
            assert [m.writing(r, g) for r in rids] == old[g], "everyone keeps the page that it writes"
            before = dict(rows[g])
            for b, p in enumerate(parents):
                for i in range(4):
                    if old[g][b] >= 0 and (old[g][p], i) in before:
                        rows[g][(old[g][b], i)] = before[(old[g][p], i)]
        plain[:] = [list(plain[p]) for p in parents]

    reorder([0] * B)
    for step in range(25):
        for k, r in enumerate(rids):
            write(r, k, [rng.random()])
            m.commit(r)
        reorder([rng.randrange(B) for _ in range(B)])
        m.check()
        for k, r in enumerate(rids):
            n = m.length(r)
            assert n == len(plain[k])
            for g in (0, 1):
                for pos in range(0 if g == 0 or window is None else max(0, n - window + 1), n):
                    assert rows[g][(m.table(r, g)[pos // 4], pos % 4)] == plain[k][pos], (step, k, g, pos)
    for r in rids:
        m.close(r)
    m.check()
    assert m.stats()["pages_free"] == [200, 200]


def test_refusals_of_the_manager():
    m = manager()
    for r in "ab":
        m.open(r)
        m.extend(r, 3)
        m.commit(r)
    for rids, parents in ((["a", "b"], [0]), (["a", "b"], [0, 2]), (["a", "a"], [0, 0]), (["a", "b"], [-1, 0])):
        with pytest.raises(CacheError):
            m.reorder(rids, parents)
    m.extend("b", 1)
    with pytest.raises(CacheError, match="one length"):
        m.reorder(["a", "b"], [0, 0])
    m.commit("b")
    with pytest.raises(CacheError, match="one length"):
        m.reorder(["a", "b"], [0, 0])


def group_search(logits_of, prompt, n_beams, max_new, ends=(), **options):
    """The search through ``BeamGroup``, with the choice made here."""
    from deliverance_amd.engine.beams import BeamGroup, BeamParameters
    p = BeamParameters(num_beams=n_beams, max_tokens=max_new, **options)
    p.validate(len(ends))
    g = BeamGroup(p, ends, max_new)
    while not g.done:
        found = []
        for b, (score, tokens) in enumerate(zip(g.scores, g.tokens)):
            if score == -math.inf:
                continue
            z = np.asarray(logits_of(list(prompt) + tokens), dtype=np.float64)
            z = z - z.max()
            z = z - math.log(np.exp(z).sum())
            found += [(score + z[v], b, v) for v in range(len(z))]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        found = found[:p.candidates(len(ends))]
        found += [(-math.inf, -1, -1)] * (p.candidates(len(ends)) - len(found))
        before = list(g.tokens)
        parents = g.take(found)
        if not g.done:
            chosen = {q for s, q in zip(g.scores, parents) if s > -math.inf}
            assert all(parents[q] == q for q in chosen), "a beam that goes on keeps its place"
            for b, q in enumerate(parents):
                assert g.tokens[b][:-1] == before[q]
    return g.finished


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("options", [{}, {"length_penalty": 0.0}, {"length_penalty": 2.0, "early_stopping": True}])
def test_the_search_is_the_plain_one(seed, options):
    vocab, n_beams, max_new = [3, 7, 12, 30][seed % 4], 1 + seed % 5, 2 + seed
    ends = () if seed % 3 == 0 else tuple(range(seed % 3))

    def logits_of(ids):
        return np.random.default_rng([seed, *ids]).normal(size=vocab) * 2

    want, gap = plain_beams.beam_search(logits_of, [5, 1], n_beams, max_new, ends, **options)
    got = group_search(logits_of, [5, 1], n_beams, max_new, ends, **options)
    assert gap > 0
    assert [(h.tokens, h.finish_reason) for h in got] == [(t, "stop" if t[-1] in ends else "length") for _, _, t in want]
    assert np.allclose([h.score for h in got], [s for _, s, _ in want])


def test_refusals_of_the_parameters():
    from deliverance_amd.engine.beams import BeamParameters
    BeamParameters().validate(1)
    for bad in (dict(num_beams=0), dict(num_beams=65), dict(max_tokens=0), dict(ntokens=0), dict(length_penalty=math.nan)):
        with pytest.raises(ValueError):
            BeamParameters(**bad).validate(1)
    with pytest.raises(ValueError, match="candidates"):
        BeamParameters(num_beams=60).validate(2)
    BeamParameters(num_beams=60, ignore_eos=True).validate(2)


def test_shared_scores_and_positions_of_a_padded_step():
    from deliverance_amd.engine.step import BeamStep, StepRunner
    words = StepRunner._beam_words(BeamStep(2, 4, [-1.5, -math.inf], [[32], [16]]), 2)
    assert np.array(words[:4], dtype=np.int32).view(np.float32).tolist() == [-1.5, -math.inf, -math.inf, -math.inf]
    assert words[4:] == [32, 0, 16, 0]


def test_the_command_line_takes_beams_or_sampling():
    from deliverance_amd import cli
    for more in (["--temperature", "0.5"], ["--top-k", "4"], ["--top-p", "0.5"], ["--xtc-threshold", "0.1"]):
        assert cli.main(["generate", "--model", "/nonexistent", "--prompt-ids", "1,2", "--num-beams", "2", *more]) == 2


def test_the_command_line_refuses_what_only_beam_search_has(capsys):
    from deliverance_amd import cli
    for more in (["--length-penalty", "0.5"], ["--early-stopping"]):
        assert cli.main(["generate", "--model", "/nonexistent", "--prompt-ids", "1,2", *more]) == 2
        assert "--num-beams" in capsys.readouterr().err


def test_sizes_beyond_32_bits_do_not_wrap(monkeypatch):
    """The library takes sizes as 32-bit numbers: what passes them is refused, and a window that passes them sees everything."""
    import torch
    from deliverance_amd.kernels import ops
    called = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: (called.append((name, a)), 0)[1]
    monkeypatch.setattr(ops, "_lib", lambda: Library())
    monkeypatch.setattr(ops, "_dev_here", lambda *t: None)
    monkeypatch.setattr(ops, "_ptr", lambda t: 16)
    monkeypatch.setattr(ops, "_stream", lambda: None)

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    far = 2 ** 32
    i32 = lambda *s: empty(*s, dtype=torch.int32)  # noqa: E731
    f32 = lambda *s: empty(*s, dtype=torch.float32)  # noqa: E731
    attend = dict(q=empty(2, 64), cache_slot=empty(5, 2, 1, 16, 32), block_table=i32(2, 4), seq_lens=i32(2), shared=i32(1), n_beams=2, n_heads=2, scale=1.0,
                  window=None, out=empty(2, 64))
    ops.attention_beams(**{**attend, "window": far + 5})
    assert called.pop()[1][15] == 2 ** 31 - 1
    one = dict(attend, q=empty(1, far)[:, :64], seq_lens=i32(1), block_table=i32(1, 4), n_beams=1, out=empty(1, far)[:, :64])
    ops.attention_beams(**one)                               # (one row: how far the next would be does not matter)
    assert called.pop()[1][1] == 64
    for bad in (dict(q=empty(2, far)[:, :64]), dict(out=empty(2, far + 64)[:, :64]), dict(block_table=i32(2, far + 1))):
        with pytest.raises(ops.KernelError, match="32 bits"):
            ops.attention_beams(**{**attend, **bad})
    out = (f32(1, 4), i32(1, 4), i32(1, 4))
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.beam_select(f32(2, far + 5), f32(2), 2, *out, f32(99))
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.beam_select_floats(2, 2, far + 5)
    with pytest.raises(ops.KernelError, match="32 bits"):
        ops.state_reorder([empty(far + 5, 1)], i32(1, 2), i32(1, 2))
    assert not called


def test_operands_on_another_device_are_refused(monkeypatch):
    import torch
    from deliverance_amd.kernels import ops

    class Operand:
        def __init__(self, index):
            self.index, self.is_cuda, self.device = index, index >= 0, f"cuda:{index}"

        def get_device(self):
            return self.index

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    ops._dev_here(Operand(1), None, Operand(1))
    for bad in ((Operand(0),), (Operand(1), Operand(0)), (Operand(0), Operand(1))):
        with pytest.raises(ops.KernelError, match="current device is cuda:1"):
            ops._dev_here(*bad)
    with pytest.raises(ops.KernelError, match="on the GPU"):
        ops._dev_here(Operand(1), Operand(-1))


def test_length_penalties_whose_power_is_no_number_are_refused():
    from deliverance_amd.engine.beams import BeamGroup, BeamParameters
    for bad in (32.5, -400.0, 1e6, math.inf):              # (400 tokens: 10^1040, no float; -400: zero, a division by it)
        with pytest.raises(ValueError, match="length_penalty"):
            BeamParameters(length_penalty=bad).validate(1)
    for good in (32.0, -32.0):
        params = BeamParameters(num_beams=2, length_penalty=good)
        params.validate(1)
        group = BeamGroup(params, {7}, 10 ** 6)
        group.tokens = [[1] * (10 ** 6 - 1)] * 2
        group.take([(-1e5, 0, 7), (-1.1e5, 1, 7), (-2e5, 0, 3), (-2e5, 1, 3)])
        assert all(math.isfinite(h.rank) and h.rank < 0 for h in group.finished) and len(group.finished) >= 2


def test_entry_points_refuse_sizes_before_they_launch():
    """Sizes outside the kernels' limits end with a message, whatever the pointers (no GPU is touched)."""
    from deliverance_amd.kernels import build, ops
    try:
        build.build(only=["beam_select", "reorder", "attn_beams"], verbose=False)
    except build.KernelLibraryError as e:
        pytest.skip(str(e))
    lib = ops._lib()

    def refused(rc, word):
        assert rc != 0 and word in build.load().da_last_error().decode()

    def select(ldl=50, G=1, B=1, V=50, K=2, scratch=8, words=10 ** 6):
        return lib.da_beam_select(8, ldl, G, B, V, 8, K, 8, 8, 8, scratch, words, None)
    for bad in (dict(V=0), dict(ldl=49), dict(B=65), dict(B=0), dict(G=-1), dict(V=2 ** 31 - 1, ldl=2 ** 31), dict(B=64, V=2 ** 26, ldl=2 ** 26)):
        refused(select(**bad), "bad sizes")
    refused(select(K=0), "candidates")
    refused(select(K=129), "candidates")
    refused(select(G=1025, B=64), "rows")
    refused(select(scratch=12), "scratch")
    refused(select(words=3), "scratch")
    refused(select(scratch=None), "scratch")
    assert select(G=0) == 0 and lib.da_beam_select_words(-1, 1, 5) == -1 and lib.da_beam_select_words(2 ** 20, 64, 2 ** 20) == -1

    import ctypes

    def reorder(row=8, layers=1, n=1, pool=4, G=1, B=2, at=64):
        return lib.da_state_reorder((ctypes.c_long * 3)(at, row, layers), n, pool, 8, 8, G, B, None)
    for bad in (dict(B=0), dict(B=65), dict(G=65536), dict(pool=-1), dict(n=-1)):
        refused(reorder(**bad), "bad sizes")
    for bad in (dict(row=3), dict(row=0), dict(row=2 ** 31), dict(at=65), dict(layers=-1)):
        refused(reorder(**bad), "whole 2-byte units")
    assert reorder(n=0) == 0 and reorder(G=0) == 0 and reorder(B=1) == 0 and reorder(pool=0) == 0

    def attend(q=16, q_ld=64, cache=16, dtype=ops.BF16, blocks=4, G=1, B=2, Hq=2, Hkv=1, D=32, page=16, window=0, splits=1, ws=None, floats=0):
        return lib.da_attn_beams(q, q_ld, cache, dtype, 8, blocks, 8, 8, G, B, Hq, Hkv, D, page, 1.0, window, 8, 64, splits, ws, floats, None)
    for bad in (dict(B=0), dict(B=65), dict(G=-1), dict(G=1025, B=64), dict(Hq=3, Hkv=2), dict(Hq=2 ** 15), dict(Hkv=0), dict(blocks=0), dict(window=-1)):
        refused(attend(**bad), "bad sizes")
    for bad in (dict(D=24), dict(D=272), dict(page=8), dict(page=48)):
        refused(attend(**bad), "head size")
    refused(attend(dtype=7), "dtype")
    for bad in (dict(q=8), dict(q_ld=65), dict(cache=8)):
        refused(attend(**bad), "16 bytes")
    refused(attend(blocks=2 ** 28), "too large")
    for n in (0, 65):
        refused(attend(splits=n), "shares")
    refused(attend(splits=2), "workspace")
    refused(attend(splits=2, ws=64, floats=2 * 2 * 2 * 34 - 1), "workspace")
    assert attend(G=0) == 0


def test_a_beams_score_goes_to_the_device_in_two_parts():
    import torch
    from deliverance_amd.engine.beams import BeamSearch
    from deliverance_amd.engine.step import BeamStep, StepRunner
    scores = [-12345.678901234, -math.inf, -1.0 / 3.0, 0.0]
    step = BeamStep(2, 4, scores, [[32, 16]])
    high = np.array(StepRunner._beam_words(step, 3)[:6], dtype=np.int32).view(np.float32).astype(np.float64)
    low = np.array(StepRunner._beam_low_words(step, 3), dtype=np.int32).view(np.float32).astype(np.float64)
    assert low.shape == (6,) and low[[1, 3, 4, 5]].tolist() == [0.0] * 4 and high[1] == high[4] == -math.inf
    assert all(abs(high[i] + low[i] - scores[i]) <= 2.0 ** -48 * abs(scores[i]) for i in (0, 2, 3))
    # and back: int32 [4, requests, candidates], score, parent, token, what the score leaves
    chosen = torch.tensor([np.float32(high[[0, 2, 1]]).view(np.int32).tolist(), [1, 0, -1], [7, 3, -1],
                           np.float32(low[[0, 2, 1]]).view(np.int32).tolist()], dtype=torch.int32).view(4, 1, 3)
    (a, b, none), = BeamSearch._candidates(chosen)
    assert a[1:] == (1, 7) and b[1:] == (0, 3) and none == (-math.inf, -1, -1)
    assert abs(a[0] - scores[0]) <= 2.0 ** -48 * abs(scores[0]) and abs(b[0] - scores[2]) <= 2.0 ** -48


def test_a_step_of_beams_is_padded_to_no_more_than_the_engine_takes():
    from types import SimpleNamespace as N
    from deliverance_amd.engine.step import StepRunner
    runner = N(max_graph_batch=64, _bucket=StepRunner._bucket)
    pad = lambda n, b: StepRunner._beam_bucket(runner, n * b, b)  # noqa: E731
    assert [pad(n, 7) for n in (1, 2, 3, 5, 9)] == [7, 14, 28, 56, 63]         # (nine requests of seven beams: 63 rows, not 112)
    assert [pad(n, 1) for n in (1, 3, 64)] == [1, 4, 64] and pad(1, 64) == 64 and pad(2, 33) == 66
    assert [StepRunner._bucket(n) for n in (1, 2, 3, 4, 5, 64, 65)] == [1, 2, 4, 4, 8, 64, 128]


def test_recordings_of_steps_of_beams_do_not_pile_up(monkeypatch):
    from types import SimpleNamespace as N
    import torch
    from deliverance_amd.engine.step import StepRunner
    waits = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: waits.append(1))
    runner = N(MAX_BEAM_RECORDINGS=2, _graphs={8: "sampled"})
    for key in ((4, 4), (8, 4), (4, 4), (6, 3), (4, 4)):
        StepRunner._keep_recording(runner, key)
        runner._graphs.setdefault(key, "recording")
    assert list(runner._graphs) == [8, (6, 3), (4, 4)] and waits == [1]
    assert StepRunner.MAX_BEAM_RECORDINGS >= 8


# Both kernels' times on the card, us: (dtype, requests, beams, heads, key heads, head size, page, positions of the table, window, positions, shared ones) ->
# (the kernel that takes a sequence by itself, the one that reads shared pages once).
MEASURED = [
    (("bfloat16", 2, 3, 4, 4, 16, 64, 2048, 0, 23, 0), (6.5, 7.5)),
    (("bfloat16", 8, 4, 4, 4, 16, 32, 1024, 0, 40, 0), (4.1, 7.4)),
    (("bfloat16", 1, 3, 32, 8, 128, 16, 1024, 0, 102, 32), (5.0, 9.4)),
    (("bfloat16", 8, 5, 8, 1, 64, 16, 4096, 0, 23, 0), (4.7, 9.0)),
    (("bfloat16", 1, 4, 12, 12, 64, 16, 1024, 0, 531, 512), (5.4, 7.8)),
    (("bfloat16", 2, 3, 28, 4, 128, 64, 1024, 64, 76, 0), (5.4, 10.4)),
    (("bfloat16", 4, 32, 25, 25, 64, 64, 512, 0, 393, 304), (37.8, 23.3)),
    (("bfloat16", 8, 8, 25, 25, 64, 16, 1024, 0, 1000, 976), (53.8, 17.7)),
    (("bfloat16", 1, 32, 32, 32, 128, 16, 13568, 0, 13566, 13552), (382.1, 59.1)),
    (("bfloat16", 16, 2, 28, 4, 128, 16, 2048, 0, 601, 590), (33.9, 12.5)),
    (("float32", 1, 32, 4, 4, 32, 32, 1024, 0, 24, 0), (5.0, 7.9)),
    (("float32", 1, 4, 2, 2, 48, 64, 1024, 0, 33, 0), (5.1, 10.4)),
    (("float32", 1, 8, 8, 8, 128, 16, 2048, 64, 1256, 624), (7.9, 14.8)),
    (("float32", 2, 32, 6, 3, 64, 16, 8192, 0, 33, 24), (7.5, 11.7)),
    (("float32", 2, 4, 28, 4, 128, 16, 2048, 0, 843, 400), (30.9, 19.1)),
    (("float32", 1, 16, 32, 32, 128, 32, 32768, 0, 3785, 3712), (206.0, 41.4)),
]


@pytest.fixture
def beams_library():
    from deliverance_amd.kernels import build
    try:
        build.build(only=["attn_beams", "attn_f32", "run_step"], verbose=False)
    except build.KernelLibraryError as e:
        pytest.skip(str(e))


@pytest.mark.parametrize("case,times", MEASURED)
def test_steps_of_beams_go_to_the_faster_kernel(case, times, beams_library):
    import torch
    from deliverance_amd.kernels import ops
    dtype, groups, beams, heads, kv_heads, dim, page, width, window, length, shared = case
    gone = max(0, length - window) if window else 0
    here = ops.attention_beams_pays(groups, beams, heads, kv_heads, dim, page, width // page, getattr(torch, dtype), length - gone, max(0, shared - gone))
    assert here == (times[1] < times[0])


def test_what_a_step_of_beams_is_judged_by(beams_library, monkeypatch):
    """Positions that a window has left behind are neither seen nor shared; a step that would leave the calls issued from C++ has to be worth it."""
    from types import SimpleNamespace as N
    import torch
    from deliverance_amd.engine.step import BeamStep, StepRunner
    from deliverance_amd.kernels import ops
    layers = [N(mixer=N(paged_attention=lambda w=w: ((0, 4, 2, 64, w),))) for w in (0, 50)]
    runner = N(model=N(blocks=layers, dtype=torch.bfloat16, config=N(schedule=[N(cache=0, layer=0), N(cache=1, layer=1), N(cache=0, layer=0)])),
               cache=N(group_of_slot={0: 0, 1: 1}, page_size=16), native=object(), debug_hook=None, _beam_layers=None, _beam_choices={}, PART_BY_PART_US=46.0)
    asked = []
    monkeypatch.setattr(ops, "attention_beams_pays", lambda *a, host_us=0.0: (asked.append((a[-2:], host_us)), a[-1] > 0)[1])
    step = BeamStep(2, 4, [0.0] * 4, [[64, 96], [64, 96]])
    attend = StepRunner._beams_attend(runner, step, [70, 110], 8, 16, recorded=True)
    both = {(0, 4, 2, 64, 0), (1, 4, 2, 64, 50)}             # 90 and 50 positions, 80 and 40 of them shared, by steps of 16
    assert asked == [((95, 80), 0.0), ((63, 32), 0.0)] and attend == both
    assert StepRunner._beams_attend(runner, step, [71, 111], 8, 16, recorded=True) == both and len(asked) == 2
    assert StepRunner._beams_attend(runner, step, [79, 119], 8, 16, recorded=True) == both and asked[2:] == [((111, 80), 0.0), ((63, 16), 0.0)]
    asked.clear()
    attend = StepRunner._beams_attend(runner, BeamStep(2, 4, [0.0] * 4, [[0, 0], [16, 16]]), [70, 110], 4, 16, recorded=False)
    assert asked == [((95, 0), 46.0), ((63, 0), 46.0)] and attend == frozenset()
    assert StepRunner._beams_attend(runner, BeamStep(1, 4, [0.0] * 2, [[64, 64], [64, 64]]), [70, 70], 2, 16, recorded=True) == frozenset()
    runner.model.blocks[:] = [N(mixer=N()), layers[1]]        # (a mixer of a user's own that says nothing of its attention)
    runner._beam_layers, runner._beam_choices = None, {}
    assert StepRunner._beams_attend(runner, step, [70, 110], 8, 16, recorded=True) == {(1, 4, 2, 64, 50)}


def test_the_estimate_of_unusual_steps(beams_library):
    """Whatever the sizes, an answer; what cannot be is behind."""
    from deliverance_amd.kernels import ops
    ahead = ops._lib().da_attn_beams_ahead_ns
    big = ahead(1023, 64, 32, 32, 256, ops.BF16, 2 ** 20, 16, 1, 1, 2 ** 24, 2 ** 24)
    assert big == 10 ** 9
    for bad in ((0, 4, 4, 4, 64, ops.BF16, 8, 16, 1, 1, 10, 0), (1, 4, 4, 0, 64, ops.BF16, 8, 16, 1, 1, 10, 0), (1, 4, 4, 4, 60, ops.BF16, 8, 16, 1, 1, 10, 0),
                (1, 4, 4, 4, 64, ops.BF16, 8, 16, 1, 0, 10, 0), (1, 4, 4, 4, 64, ops.BF16, 8, 16, 1, 1, 0, 0)):
        assert ahead(*bad) == -1
    assert abs(ahead(1, 4, 4, 4, 64, ops.BF16, 8, 16, 1, 1, 10, -5)) < 10 ** 5 and abs(ahead(1, 4, 4, 4, 64, ops.F32, 8, 16, 1, 1, 10, 50)) < 10 ** 5
