"""The operators of beam search against plain 64-bit implementations: the choice among beams and vocabulary, the reordering of what
beams keep, attention over pages that beams share."""
import math

import pytest
import torch

from deliverance_amd.kernels import ops
from deliverance_amd.kernels.ops import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda:0" if torch.cuda.is_available() else "cpu"
INF = math.inf
quick = pytest.mark.simt_quick


# ------------------------------------------------------------------------------- the choice
def plain_select(logits, scores, B, K):
    """Keys in 64 bits; returns (scores float64, parents, tokens) as lists of rows, and the gaps between keys that follow each other."""
    R, V = logits.shape
    z = logits.double().cpu()
    z = torch.where(torch.isnan(z), -INF, z)
    top = z.amax(1, keepdim=True)
    x = torch.where(z == top, 0.0, z - top)
    x = torch.where(z == -INF, -INF, x)
    s = scores.double().cpu()
    s = torch.where(torch.isnan(s), -INF, s)
    keys = s[:, None] + (x - torch.log(torch.exp(x).sum(1, keepdim=True)))
    keys = torch.where(torch.isnan(keys), -INF, keys).view(R // B, B * V)
    value, place = torch.sort(keys, dim=1, descending=True, stable=True)
    short = max(0, K + 1 - B * V)
    value = torch.nn.functional.pad(value, (0, short), value=-INF)
    place = torch.nn.functional.pad(place, (0, short))
    none = value[:, :K] == -INF
    gaps = value[:, :K] - value[:, 1:K + 1]
    return (value[:, :K], torch.where(none, -1, place[:, :K] // V), torch.where(none, -1, place[:, :K] % V),
            torch.where(torch.isnan(gaps), 1.0, gaps))


def select(logits, scores, B, K):
    G = logits.shape[0] // B
    ws = torch.full((ops.beam_select_floats(logits.shape[0], B, logits.shape[1]),), math.nan, device=DEV)
    out = (torch.full((G, K), math.nan, device=DEV), torch.full((G, K), -7, dtype=torch.int32, device=DEV),
           torch.full((G, K), -7, dtype=torch.int32, device=DEV))
    got = ops.beam_select(logits, scores, B, *out, ws)
    return tuple(t.cpu() for t in got)


def check_select(logits, scores, B, K):
    want = plain_select(logits, scores, B, K)
    # The kernel's sum of exponentials is off by the 32-bit exponentials (two units in the last place: 2^-22), by the two roundings that add
    # four of them (2^-23) and by the operands' rounding (2^-24 of a difference d, weighed with its term e^-d: below 2^-24), together below
    # 2^-21; so keys of two beams compare as the 64-bit ones do where they are 1e-6 apart, or equal.
    gaps = want[3]
    assert bool(((gaps == 0.0) | (gaps > 1e-6)).all()), "the inputs do not keep the keys apart"
    got = select(logits, scores, B, K)
    assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2].long(), want[2])
    there = want[1] >= 0
    assert bool((got[0][~there] == -INF).all())
    off = (got[0].double() - want[0])[there].abs()
    near = 2.0 ** -24 * want[0][there].abs() + 2.0 ** -21
    inf = want[0][there].isinf()
    assert bool((off <= near)[~inf].all()) and bool((got[0].double()[there] == want[0][there])[inf].all())


SELECT = [pytest.param(1, 1, 1, 1, marks=quick), pytest.param(1, 1, 5, 9, marks=quick), pytest.param(2, 3, 255, 6, marks=quick),
          pytest.param(1, 4, 257, 8, marks=quick), (3, 8, 2049, 16), (1, 64, 300, 128), (2, 5, 4097, 10), (1, 17, 1023, 34), (5, 1, 50257, 12),
          (2, 4, 50257, 8), (1, 2, 262144, 128), (64, 8, 777, 16)]


@pytest.mark.parametrize("groups,beams,vocab,keep", SELECT)
@pytest.mark.parametrize("banned", [0.0, 0.7])
def test_the_choice_is_the_plain_one(groups, beams, vocab, keep, banned):
    g = torch.Generator().manual_seed(groups * 1000 + beams * 10 + vocab)
    logits = torch.randn(groups * beams, vocab, generator=g) * 3
    logits[torch.rand(groups * beams, vocab, generator=g) < banned] = -INF
    scores = -20 * torch.rand(groups * beams, generator=g)
    if beams > 2:
        scores[beams - 1::beams] = -INF
    check_select(logits.to(DEV), scores.to(DEV), beams, keep)


@pytest.mark.parametrize("vocab", [pytest.param(700, marks=quick), 5000])
def test_the_first_of_equal_entries(vocab):
    """All logits equal, and two beams with one score: far more equal keys than candidates, taken in the order of beams and tokens."""
    for beams, keep in ((1, 7), (3, 20), (2, 128)):
        logits = torch.full((2 * beams, vocab), 1.25)
        logits[beams:, 1::2] = 2.5                          # (second group: every other one is better)
        scores = torch.full((2 * beams,), -3.0)
        check_select(logits.to(DEV), scores.to(DEV), beams, keep)
    logits = torch.full((1, vocab), -INF)                   # one token is allowed
    logits[0, vocab - 3] = 4.0
    check_select(logits.to(DEV), torch.zeros(1, device=DEV), 1, 4)


@quick
def test_a_choice_with_masked_and_odd_numbers():
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(8, 600, generator=g)
    logits[0, 3] = math.nan                                 # counts as forbidden
    logits[1] = -INF                                        # a beam without a token
    logits[2, [4, 590]] = INF                               # these two share the probability
    logits[3] = math.nan
    logits[4] = torch.finfo(torch.float32).min              # a mask of the type's lowest value, everywhere: all the same
    logits[5, 10:] = torch.finfo(torch.float32).min
    logits[6, 7] = 3e38
    scores = torch.tensor([-1.0, -2.0, -7.5, 0.0, -9.0, -3.3, -5.7, math.nan])
    check_select(logits.to(DEV), scores.to(DEV), 8, 20)
    check_select(logits.to(DEV), torch.full((8,), -INF, device=DEV), 4, 5)
    check_select(logits.to(DEV), scores.to(DEV), 2, 16)


@quick
def test_a_choice_in_rows_of_a_wider_matrix():
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(6, 1031, generator=g).to(DEV)
    check_select(wide[:, 3:1004], torch.tensor([-4.0, -5.0, -6.0, -1.0, -2.0, -3.5], device=DEV), 3, 9)


@quick
def test_a_large_score_does_not_make_neighbouring_logits_equal():
    """At -60,000 a 32-bit sum has steps of 2^-8: the order is the logits' all the same."""
    logits = torch.zeros(2, 300)
    logits[:, 100:140] = 5 + torch.arange(40) * 2.0 ** -12
    scores = torch.tensor([-60000.0, -60000.00390625])
    check_select(logits.to(DEV), scores.to(DEV), 2, 30)


def test_a_choice_among_more_segments_and_entries_than_the_lists_hold():
    """Segments in stripes, so that the groups in front are better than the others with everything they have, and entries that are all
    near their segment's best: the bounds are searched bit by bit."""
    V = 262144
    v = torch.arange(V)
    row = -(v // 256 % 256).double() - (v % 256).double() * 2.0 ** -10
    logits = torch.stack([row, row]).float()
    check_select(logits.to(DEV), torch.tensor([-1.0, -1.30078125], device=DEV), 2, 128)
    # 128 best entries in each of many segments
    flat = torch.zeros(2, V)
    flat[:, 1000:200000] = 3.0
    check_select(flat.to(DEV), torch.tensor([-1.0, -1.0], device=DEV), 2, 128)


def test_refusals_of_the_choice():
    logits, scores = torch.zeros(6, 40, device=DEV), torch.zeros(6, device=DEV)
    out = (torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    ws = torch.zeros(ops.beam_select_floats(6, 3, 40), device=DEV)
    ops.beam_select(logits, scores, 3, *out, ws)
    for bad in (dict(logits=logits.bfloat16()), dict(logits=logits.t()), dict(scores=scores[:5]), dict(n_beams=4), dict(n_beams=0), dict(n_beams=65),
                dict(out_scores=out[0].double()), dict(out_parents=out[1].long()), dict(out_tokens=out[2][:1]), dict(out_scores=out[0].t()),
                dict(workspace=ws[:-1]), dict(workspace=ws.int()), dict(scores=scores.bfloat16()),
                dict(out_scores=torch.zeros(2, 129, device=DEV))):
        with pytest.raises(KernelError):
            args = dict(logits=logits, scores=scores, n_beams=3, out_scores=out[0], out_parents=out[1], out_tokens=out[2], workspace=ws)
            ops.beam_select(**{**args, **bad})
    empty = ops.beam_select(logits[:0], scores[:0], 3, out[0][:0], out[1][:0], out[2][:0], ws)
    assert empty[0].shape == (0, 4)


# ------------------------------------------------------------------------------- reordering
def plain_reorder(tensors, slots, parents, dim):
    out = [t.clone() for t in tensors]
    for t, new in zip(tensors, out):
        rows, to = t.transpose(0, dim), new.transpose(0, dim)
        for s, p in zip(slots.tolist(), parents.tolist()):
            for b in range(len(s)):
                if 0 <= p[b] < len(s) and 0 <= s[b] < rows.shape[0] and 0 <= s[p[b]] < rows.shape[0]:
                    to[s[b]] = rows[s[p[b]]]
    return out


def bits(t):
    return t.contiguous().view(torch.uint8)


def check_reorder(tensors, slots, parents, dim=0):
    want = plain_reorder([t.cpu() for t in tensors], slots, parents, dim)
    got = ops.state_reorder(tensors, slots.to(DEV), parents.to(DEV), dim=dim)
    for a, b in zip(got, want):
        assert torch.equal(bits(a.cpu()), bits(b))


@pytest.mark.parametrize("groups,beams", [pytest.param(1, 1, marks=quick), pytest.param(1, 2, marks=quick), pytest.param(2, 5, marks=quick),
                                          (1, 16), pytest.param(1, 17, marks=quick), (2, 64), (9, 8), (3, 4)])
@pytest.mark.parametrize("row", [1, 3, 4, 1025, 4096])
def test_rows_follow_their_parents(groups, beams, row):
    g = torch.Generator().manual_seed(groups * 100 + beams + row)
    pool = groups * beams + 3
    tensors = [torch.randint(-2 ** 31, 2 ** 31 - 1, (pool, row), generator=g, dtype=torch.int32).to(DEV),       # any bits, also of no numbers
               torch.randn(pool, row, generator=g).to(torch.bfloat16).to(DEV)]
    for kind in ("any", "permutation", "one", "none"):
        slots = torch.randperm(pool, generator=g)[:groups * beams].view(groups, beams).int()
        if kind == "any":
            parents = torch.randint(0, beams, (groups, beams), generator=g)
        elif kind == "permutation":
            parents = torch.stack([torch.randperm(beams, generator=g) for _ in range(groups)])
        else:
            parents = torch.full((groups, beams), beams - 1) if kind == "one" else torch.arange(beams).repeat(groups, 1)
        check_reorder(tensors, slots, parents.int())


@quick
def test_places_without_a_row_or_a_parent_stay():
    g = torch.Generator().manual_seed(3)
    t = [torch.randn(7, 12, generator=g).to(DEV)]
    slots = torch.tensor([[0, -1, 5, 2], [3, 7, 1, 6]], dtype=torch.int32)
    parents = torch.tensor([[2, 0, 1, -1], [2, 0, 4, 1]], dtype=torch.int32)
    check_reorder(t, slots, parents)


@pytest.mark.parametrize("layers", [pytest.param(3, marks=quick), 100])
def test_layers_of_one_tensor_and_many_tensors(layers):
    g = torch.Generator().manual_seed(layers)
    slots = torch.tensor([[4, 0, 6], [1, 5, 2]], dtype=torch.int32)
    parents = torch.tensor([[1, 1, 0], [2, 0, 1]], dtype=torch.int32)
    check_reorder([torch.randn(layers, 8, 2, 10, generator=g).to(DEV), torch.randn(2, 8, 33, generator=g).to(DEV)], slots, parents, dim=1)
    check_reorder([torch.randn(8, 1 + i % 7, generator=g).to(DEV) for i in range(layers)], slots, parents)


def test_refusals_of_reordering():
    t, i = torch.zeros(6, 4, device=DEV), torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    ops.state_reorder([t], i, i)
    ops.state_reorder([], i, i)
    ops.state_reorder([torch.zeros(6, 0, device=DEV)], i, i)
    wide = torch.zeros(1, 65, dtype=torch.int32, device=DEV)
    for args in (([t], i.long(), i.long()), ([t], i, i[:1]), ([t], i.view(-1), i.view(-1)), ([t.t()], i, i), ([t, t[:5]], i, i), ([t, t], i, i),
                 ([t, t.view(-1)[4:].view(5, 4)], i, i), ([torch.zeros(6, 3, dtype=torch.uint8, device=DEV)], i, i), ([t], i, i, 2),
                 ([t], wide, wide), ([t], i.t(), i.t())):
        with pytest.raises(KernelError):
            ops.state_reorder(*args)


# ------------------------------------------------------------------------------- attention
def beams_case(groups, beams, heads, kv_heads, dim, page, dtype, lengths, shared, seed, wide=0):
    """Lengths: of every sequence; shared: positions in pages that a group shares.  Rows that no sequence has written are no numbers."""
    g = torch.Generator().manual_seed(seed)
    blocks = max(1, -(-max(lengths) // page))
    need = [[max(0, -(-lengths[i * beams + b] // page) - shared[i] // page) for b in range(beams)] for i in range(groups)]
    n = sum(s // page for s in shared) + sum(map(sum, need)) + 2
    ids = torch.randperm(n, generator=g)
    cache = torch.randn(n, 2, kv_heads, page, dim, generator=g).to(dtype)
    table = torch.full((groups * beams, blocks), -1, dtype=torch.int32)
    at = 0
    for i in range(groups):
        k = shared[i] // page
        table[i * beams:(i + 1) * beams, :k] = ids[at:at + k].int()
        at += k
        for b in range(beams):
            s, m = i * beams + b, need[i][b]
            table[s, k:k + m] = ids[at:at + m].int()
            at += m
            if lengths[s] == 0:
                table[s] = -1
            elif m and lengths[s] % page:
                last = int(table[s, k + m - 1])
                cache[last, 0, :, lengths[s] % page:] = math.nan
                cache[last, 1].view(kv_heads, dim, page)[:, :, lengths[s] % page:] = math.nan
    cache[ids[at:]] = math.nan
    rows = (torch.randn(groups * beams, heads * dim + wide, generator=g) * 1.5).to(dtype).to(DEV)
    return dict(q=rows[:, :heads * dim], cache=cache.to(DEV), table=table.to(DEV), lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                shared=torch.tensor(shared, dtype=torch.int32, device=DEV), beams=beams, heads=heads)


def plain_attention(c, window=None):
    cache, table, lens, q = c["cache"].cpu().double(), c["table"].cpu(), c["lens"].cpu(), c["q"].cpu().double()
    n, _, Hkv, page, D = cache.shape
    Hq = c["heads"]
    out = torch.zeros(q.shape[0], Hq, D, dtype=torch.float64)
    for s in range(q.shape[0]):
        n = int(lens[s])
        if n <= 0:
            continue
        lo = max(0, n - window) if window else 0
        pos = torch.arange(lo, n)
        ids = table[s].long()[pos // page]
        k = cache[ids, 0, :, pos % page]                                                   # [keys, Hkv, D]
        v = cache[:, 1].reshape(-1, Hkv, D, page)[ids, :, :, pos % page]
        for h in range(Hq):
            p = torch.softmax(k[:, h // (Hq // Hkv)] @ q[s, h * D:(h + 1) * D] / math.sqrt(D), 0)
            out[s, h] = p @ v[:, h // (Hq // Hkv)]
    return out.view(q.shape[0], Hq * D)


def attend(c, window=None, splits=1):
    dtype, D = c["q"].dtype, c["cache"].shape[4]
    S = c["q"].shape[0]
    out = torch.full((S, c["heads"] * D), math.nan, dtype=dtype, device=DEV)
    ws = torch.full((max(1, ops.beam_workspace_floats(S, c["heads"], D, splits)),), math.nan, device=DEV)
    return ops.attention_beams(c["q"], c["cache"], c["table"], c["lens"], c["shared"], c["beams"], c["heads"], 1 / math.sqrt(D), window, out,
                               splits, ws)


def check_attention(c, window=None, splits=1):
    """A score of these inputs is below 60 and sums up to 256 products in 32-bit (error below 256 * 2^-24 * sum |q k| < 1e-4, in practice
    its root); e^x by a 32-bit product with log2 e (60 * 1.45 * 2^-24 = 5e-6); a bfloat16 weight in two parts keeps 2^-17.  A weight is
    thus off by less than 1e-4 of itself and the result by less than 2e-4 of the largest value; then it is rounded (half a step)."""
    got, want = attend(c, window, splits).cpu().double(), plain_attention(c, window)
    big = 6.0
    near = torch.finfo(c["q"].dtype).eps / 2 * want.abs() + 2e-4 * big * (1.0 if c["q"].dtype == torch.bfloat16 else 0.05)
    off = (got - want).abs()
    assert bool((off <= near).all()), f"off by {float(off.max())}, {float((off / near).max())} of what is allowed"


ATTEND = [  # groups, beams, heads, kv heads, head size, page, lengths, shared
    pytest.param(1, 1, 1, 1, 16, 16, [1], [0], marks=quick),
    pytest.param(1, 4, 2, 2, 64, 16, [147] * 4, [128], marks=quick),
    pytest.param(2, 3, 4, 2, 32, 32, [65, 65, 65, 200, 199, 198], [64, 160], marks=quick),
    pytest.param(2, 2, 3, 3, 48, 16, [0, 0, 70, 0], [0, 0], marks=quick),
    pytest.param(1, 3, 2, 1, 80, 64, [130, 0, 129], [128], marks=quick),
    (2, 8, 8, 2, 128, 16, [530] * 8 + [64] * 8, [512, 48]),
    (1, 5, 40, 2, 64, 16, [300] * 5, [240]),
    (1, 2, 32, 1, 16, 32, [77, 77], [64]),
    (1, 3, 2, 2, 256, 16, [400, 390, 410], [384]),
    (3, 4, 3, 3, 64, 64, [640] * 4 + [1] * 4 + [127] * 4, [640, 0, 64]),
    (1, 16, 2, 2, 64, 16, [1100 + i for i in range(16)], [0]),
    (1, 64, 2, 1, 32, 16, [210] * 64, [192]),
    (1, 2, 1, 1, 64, 16, [5000, 4999], [4096]),
    (9, 5, 60, 15, 32, 16, [40 + i % 7 for i in range(45)], [32] * 9),       # more workgroups than compute units: two tiles of rows a workgroup
    (13, 9, 40, 20, 48, 32, [97 if i % 9 else 0 for i in range(117)], [64] * 13),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("groups,beams,heads,kv_heads,dim,page,lengths,shared", ATTEND)
def test_attention_of_beams(groups, beams, heads, kv_heads, dim, page, lengths, shared, dtype):
    c = beams_case(groups, beams, heads, kv_heads, dim, page, dtype, lengths, shared, seed=dim + beams, wide=16)
    blocks = c["table"].shape[1]
    for splits in sorted({1, 3, ops.beam_splits(groups, beams, heads, kv_heads, dim, blocks, page, dtype)}):
        check_attention(c, splits=splits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [1, pytest.param(50, marks=quick), 64, 200])
def test_attention_of_beams_over_a_window(window, dtype):
    c = beams_case(2, 3, 4, 2, 64, 16, dtype, [300, 300, 300, 250, 240, 256], [288, 192], seed=window)
    for s, n in enumerate(c["lens"].tolist()):                # pages that the window has passed are gone
        gone = max(0, n - window) // 16
        if s < 3:                                             # (the group's tables agree on what they share)
            c["table"][s, :gone] = -1
    for splits in (1, 4):
        check_attention(c, window=window, splits=splits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@quick
def test_what_one_beam_alone_sees_does_not_reach_the_others(dtype):
    """Infinite and missing numbers in the first beam's own page; the other beams' rows are as if they were not there."""
    c = beams_case(1, 3, 2, 2, 48, 16, dtype, [140] * 3, [128], seed=9)
    want = plain_attention(c)
    own = int(c["table"][0, 8])
    c["cache"][own, 1].view(2, 48, 16)[:, :, 3] = INF
    c["cache"][own, 0, :, 5] = math.nan
    got = attend(c, splits=2).cpu().double()
    assert bool(got[0].isnan().any())
    assert float((got[1:] - want[1:]).abs().max()) <= 2.0 ** -8 * 4 + 1.2e-3


@quick
def test_sharing_does_not_change_what_is_attended():
    """The same tables, declared as shared or not."""
    c = beams_case(2, 4, 4, 2, 64, 16, torch.bfloat16, [200] * 4 + [333] * 4, [192, 320], seed=12)
    want = plain_attention(c)
    for shared in ([192, 320], [0, 0], [64, 100], [16, 10 ** 6]):
        c["shared"] = torch.tensor(shared, dtype=torch.int32, device=DEV)
        if shared[1] > 333:
            c["shared"][1] = 320
        got = attend(c, splits=2).cpu().double()
        assert float((got - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1.2e-3


def test_refusals_of_attention():
    c = beams_case(2, 2, 4, 2, 32, 16, torch.bfloat16, [40] * 4, [32, 32], seed=1)
    out = torch.zeros(4, 128, dtype=torch.bfloat16, device=DEV)
    ws = torch.zeros(ops.beam_workspace_floats(4, 4, 32, 3), device=DEV)
    good = dict(q=c["q"], cache_slot=c["cache"], block_table=c["table"], seq_lens=c["lens"], shared=c["shared"], n_beams=2, n_heads=4, scale=1.0,
                window=None, out=out, n_splits=3, workspace=ws)
    ops.attention_beams(**good)
    wide = torch.zeros(4, 129, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=c["q"].float()), dict(out=out.float()), dict(q=c["q"].half(), cache_slot=c["cache"].half(), out=out.half()),
                dict(q=wide[:, 1:]), dict(n_heads=3), dict(n_beams=3), dict(n_beams=0), dict(block_table=c["table"].long()),
                dict(block_table=c["table"][:3]), dict(seq_lens=c["lens"].long()), dict(shared=c["shared"][:1]), dict(workspace=ws[:-1]),
                dict(workspace=None), dict(cache_slot=c["cache"][:, :, :, :8].contiguous()), dict(window=-1),
                dict(q=c["q"][:, :32], out=out[:, :32], n_heads=4, cache_slot=c["cache"][..., :8].contiguous())):
        with pytest.raises(KernelError):
            ops.attention_beams(**{**good, **bad})


# ------------------------------------------------------------------------------- as programs use them
def recorded(f):
    """``f`` once eagerly, then recorded; a function that replays it."""
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    return graph.replay


@pytest.mark.needs_device
def test_recorded_calls_follow_their_inputs():
    """Two recordings that share a workspace, replayed in turn with other work between them, on inputs that change."""
    g = torch.Generator().manual_seed(31)
    logits, scores = torch.randn(8, 3001, device=DEV), -torch.rand(8, device=DEV)
    out = (torch.zeros(2, 8, device=DEV), torch.zeros(2, 8, dtype=torch.int32, device=DEV), torch.zeros(2, 8, dtype=torch.int32, device=DEV))
    c = beams_case(2, 4, 4, 4, 64, 16, torch.bfloat16, [700] * 8, [640, 656], seed=4)
    D, splits = 64, 3
    o = torch.zeros(8, 256, dtype=torch.bfloat16, device=DEV)
    ws = torch.zeros(max(ops.beam_select_floats(8, 4, 3001), ops.beam_workspace_floats(8, 4, D, splits)), device=DEV)
    state = torch.randn(12, 1000, device=DEV)
    slots = torch.tensor([[3, 1, 7, 0], [2, 11, 5, 6]], dtype=torch.int32, device=DEV)
    parents = torch.zeros(2, 4, dtype=torch.int32, device=DEV)

    def choose():
        ops.beam_select(logits, scores, 4, *out, ws)

    def rest():
        ops.attention_beams(c["q"], c["cache"], c["table"], c["lens"], c["shared"], 4, 4, 0.125, None, o, splits, ws)
        ops.state_reorder([state], slots, parents)

    first, second = recorded(choose), recorded(rest)
    for turn in range(4):
        logits.copy_(torch.randn(8, 3001, generator=g) * 2)
        scores.copy_(-torch.rand(8, generator=g) * 5)
        c["q"].copy_(torch.randn(8, 256, generator=g).bfloat16())
        state.copy_(torch.randn(12, 1000, generator=g))
        parents.copy_(torch.randint(0, 4, (2, 4), generator=g))
        first()
        want_state = plain_reorder([state.cpu()], slots.cpu(), parents.cpu(), 0)[0]
        second()
        want = plain_select(logits, scores, 4, 8)
        assert torch.equal(out[1].cpu().long(), want[1]) and torch.equal(out[2].cpu().long(), want[2])
        assert torch.equal(state.cpu(), want_state)
        eager = torch.zeros_like(o)
        ops.attention_beams(c["q"], c["cache"], c["table"], c["lens"], c["shared"], 4, 4, 0.125, None, eager, splits, torch.zeros_like(ws))
        assert torch.equal(eager, o)
        near = 2.0 ** -8 * plain_attention(c).abs() + 1.2e-3
        assert bool(((o.cpu().double() - plain_attention(c)).abs() <= near).all())


@pytest.mark.needs_device
def test_a_chain_of_steps_on_a_stream_of_its_own():
    """The three operators together, as a step uses them: attention, a choice, and what is kept follows it, all without the host."""
    stream = torch.cuda.Stream()
    g = torch.Generator().manual_seed(8)
    G, B, D, V = 2, 3, 32, 500
    c = beams_case(G, B, 2, 2, D, 16, torch.float32, [200] * 6, [192] * 2, seed=2)
    head = torch.randn(2 * D, V, generator=g)
    state = torch.randn(10, 77, generator=g)
    slots = torch.tensor([[9, 2, 4], [0, 7, 3]], dtype=torch.int32)
    scores = -torch.rand(G * B, generator=g)
    o = plain_attention(c)
    want = plain_select((o.float() @ head), scores, B, B)
    want_state = plain_reorder([state], slots, want[1].int(), 0)[0]
    dev = [t.to(DEV) for t in (head, state, slots, scores)]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = attend(c, splits=2)
        logits = got @ dev[0]
        out = (torch.empty(G, B, device=DEV), torch.empty(G, B, dtype=torch.int32, device=DEV), torch.empty(G, B, dtype=torch.int32, device=DEV))
        ops.beam_select(logits, dev[3], B, *out, torch.empty(ops.beam_select_floats(G * B, B, V), device=DEV))
        ops.state_reorder([dev[1]], dev[2], out[1])
    stream.synchronize()
    assert float(want[3].min()) > 1e-4                      # (32-bit logits of this size are off by about 1e-5)
    assert torch.equal(out[1].cpu().long(), want[1]) and torch.equal(out[2].cpu().long(), want[2])
    assert torch.equal(dev[1].cpu(), want_state)


@pytest.mark.needs_device
def test_places_beyond_32_bits():
    """A cache, states and logits whose last rows lie more than 2^32 bytes behind the first ones."""
    Hkv, page, D, n = 8, 64, 128, 24000                      # 6.3 GB
    big = torch.empty(n, 2, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    c = beams_case(1, 2, 8, Hkv, D, page, torch.bfloat16, [150, 140], [128], seed=3)
    few = c["cache"].shape[0]
    big[n - few:] = c["cache"]
    far = dict(c, cache=big, table=torch.where(c["table"] >= 0, c["table"] + (n - few), -1).int())
    assert torch.equal(attend(far), attend(c))
    del big, far
    row = 1 << 28                                            # 1 GiB a row
    t = torch.empty(6, row, dtype=torch.float32, device=DEV)
    for i in range(6):
        t[i, -3:] = i
        t[i, :3] = 10 + i
    ops.state_reorder([t], torch.tensor([[5, 0, 4]], dtype=torch.int32, device=DEV), torch.tensor([[1, 0, 0]], dtype=torch.int32, device=DEV))
    assert t[:, -1].tolist() == [5, 1, 2, 3, 5, 0] and t[:, 0].tolist() == [15, 11, 12, 13, 15, 10]
    del t
    wide = torch.empty(6, 1 << 29, dtype=torch.float32, device=DEV)
    part = wide[:, 7:1007]
    part.copy_(torch.randn(6, 1000, generator=torch.Generator().manual_seed(9)))
    check_select(part, torch.tensor([-1.0, -1.5, -2.5] * 2, device=DEV), 3, 6)
