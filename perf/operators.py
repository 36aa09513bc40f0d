"""The operators of beam search, as they are timed: the choice among beams and vocabulary, the reordering of what the beams keep,
and attention of one new token a beam over a paged cache whose first pages the beams of a request share.

With ``own`` false ``run`` computes them from elementary tensor operations; with ``own`` true by the engine's kernels
(``deliverance_amd.kernels.ops``: ``beam_select``, ``state_reorder``, ``attention_beams``).

* select: logits [groups * beams, vocab] (32-bit) and the beams' summed log-probabilities; the ``keep`` best (beam, token) pairs of every
  group by summed log-probability, the lowest beam * vocab + token first among equals.  A place without a beam has a score of -inf, a
  forbidden token a logit of -inf; candidates that do not exist are (-inf, -1, -1).
* reorder: tensors [pool, ...] (or [layers, pool, ...]) of which every beam holds one row (a page of keys and values, a recurrent state):
  the row of beam b becomes what the row of its parent was.
* attention: softmax(scale q K^T) V for one query row a beam.  A page of the cache holds, head by head, its keys row by row and its values
  dimension by dimension.  Rows that nobody has written are no numbers.
"""
import math

import torch

own = False
DEV = "cuda:0"
VOCAB = 50257
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    def select(name, groups, beams, vocab, keep, live=None, banned=0.0):
        return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab, "keep": keep, "live": live or beams,
                "banned": banned}

    def reorder(name, layers, row, pool, groups, beams, moved, dtype="bfloat16", row2=0, stacked=True):
        return {"name": name, "op": "reorder", "layers": layers, "row": row, "row2": row2, "pool": pool, "groups": groups, "beams": beams,
                "moved": moved, "dtype": dtype, "stacked": stacked}

    def attention(name, groups, beams, heads, kv_heads, dim, length, behind, page=16, dtype="bfloat16"):
        return {"name": name, "op": "attention", "groups": groups, "beams": beams, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "length": length, "behind": behind, "page": page, "dtype": dtype}

    return [
        # one request of four beams, GPT-2's vocabulary: what one user's step waits for
        select("select-1x4", 1, 4, VOCAB, 8),
        # the first choice behind the prompts: one row a request
        select("select-first-24x1", 24, 1, VOCAB, 12),
        # a full server: eight requests of eight beams, a fifth of the vocabulary forbidden
        select("select-8x8", 8, 8, VOCAB, 16, banned=0.2),
        # many requests, a large vocabulary, places without a beam
        select("select-32x8-large", 32, 8, 131071, 16, live=7),
        # the pages that four beams of one request are writing: 12 layers, 12 heads of 64, pages of 16
        reorder("reorder-pages-124m-1x4", 12, 2 * 12 * 16 * 64, 64, 1, 4, 2),
        # the same for eight requests of eight beams on 48 layers of 25 heads
        reorder("reorder-pages-1.5b-8x8", 48, 2 * 25 * 16 * 64, 160, 8, 8, 4),
        # recurrent layers: a short filter's inputs and a 32-bit matrix a head
        reorder("reorder-states-4x8", 16, 16 * 128 * 128, 32, 4, 8, 5, dtype="float32", row2=3 * 1025, stacked=False),
        # one request of four beams behind a prompt of 512 tokens
        attention("attention-1x4-512", 1, 4, 12, 12, 64, 531, 19),
        # eight requests of eight beams at GPT-2's longest contexts
        attention("attention-8x8-1000", 8, 8, 25, 25, 64, 1003, 60),
        # long contexts, four query heads a key head
        attention("attention-4x4-32k", 4, 4, 32, 8, 128, 32701, 200, page=64),
        # the 32-bit path: odd numbers of beams and positions
        attention("attention-f32-2x5-777", 2, 5, 12, 12, 64, 777, 33, dtype="float32"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("select", "reorder", "attention"))
    if op == "select":
        groups, beams = log(1, 32), log(1, 24)
        vocab = min(log(300, 160000), 32 * 8 * 131071 // (groups * beams))
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "keep": 2 * beams if rng.random() < 0.7 else rng.randint(1, 2 * beams),
                "live": rng.randint(max(1, beams - 2), beams), "banned": rng.choice((0.0, 0.0, 0.1, 0.9))}
    if op == "reorder":
        layers, groups, beams = log(1, 60), log(1, 12), log(2, 16)
        dtype = rng.choice(("bfloat16", "float32"))
        row, stacked = min(log(500, 300000), 600_000_000 // (layers * groups * beams * 4)) // 2 * 2, rng.random() < 0.6
        return {"op": op, "layers": layers, "row": row, "row2": 0 if stacked else rng.choice((0, rng.randint(1, 6000))), "stacked": stacked, "pool": groups * beams + rng.randint(0, 20), "groups": groups, "beams": beams, "moved": rng.randint(1, beams - 1), "dtype": dtype}
    groups, beams, kv_heads = log(1, 16), log(2, 16), log(1, 25)
    heads = kv_heads * rng.choice((1, 1, 2, 4, 5))
    dim, dtype = rng.choice((32, 48, 64, 64, 80, 128)), rng.choice(("bfloat16", "bfloat16", "float32"))
    length = log(1, min(32000, max(64, 4 * 8 * 32701 * 128 // (groups * beams * kv_heads * dim))))
    return {"op": op, "groups": groups, "beams": beams, "heads": heads, "kv_heads": kv_heads, "dim": dim, "length": length,
            "behind": min(length, log(1, 300)), "page": rng.choice((16, 32, 64)), "dtype": dtype}


def _lengths(case):
    """Per group: (positions, of which so many lie in pages that the group's beams share)."""
    n, page = case["length"], case["page"]
    totals = [n - (37 * g) % (n // 4 + 1) for g in range(case["groups"])]
    return [(t, max(0, t - case["behind"]) // page * page) for t in totals]


def work(case):
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": 4 * rows * (case["vocab"] + 1) + 12 * case["groups"] * case["keep"], "flops": 4 * rows * case["vocab"]}
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "reorder":
        read = min(case["moved"], case["beams"] - case["moved"])
        rows = case["groups"] * (read + case["moved"])
        return {"bytes": case["layers"] * rows * (case["row"] * size + case["row2"] * 4), "flops": 0}
    B, Hq, Hkv, D = case["beams"], case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    keys = sum(shared + B * (n - shared) for n, shared in lengths)
    return {"bytes": size * (keys * 2 * Hkv * D + 2 * case["groups"] * B * Hq * D), "flops": 4 * D * Hq * B * sum(n for n, _ in lengths)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    G, B = case["groups"], case["beams"]
    if case["op"] == "select":
        V, K = case["vocab"], case["keep"]
        logits = torch.randn(G * B, V, device=DEV, generator=g) * 2.5
        if case["banned"]:
            logits[torch.rand(G * B, V, device=DEV, generator=g) < case["banned"]] = -math.inf
        scores = -30.0 * torch.rand(G, B, device=DEV, generator=g)
        scores[:, case["live"]:] = -math.inf
        state = {"logits": logits, "scores": scores.view(-1).contiguous(),
                 "out": (torch.empty(G, K, device=DEV), torch.empty(G, K, dtype=torch.int32, device=DEV), torch.empty(G, K, dtype=torch.int32, device=DEV)),
                 "scratch": torch.empty(1 << 22, device=DEV)}
    elif case["op"] == "reorder":
        dtype, pool = TYPES[case["dtype"]], case["pool"]
        if case["stacked"]:
            tensors = [torch.randn(case["layers"], pool, case["row"], device=DEV, generator=g).to(dtype)]
        else:
            tensors = [torch.randn(pool, case["row"], device=DEV, generator=g).to(dtype) for _ in range(case["layers"])]
        if case["row2"]:
            tensors += [torch.randn(pool, case["row2"], device=DEV, generator=g) for _ in range(case["layers"])]
        slots = torch.randperm(pool, generator=h)[:G * B].view(G, B).to(torch.int32)
        parents = torch.arange(B, dtype=torch.int32).repeat(G, 1)
        for i in range(G):                                # who stays keeps its place; the others continue one of those
            order = torch.randperm(B, generator=h)
            gone, stay = order[:case["moved"]], order[case["moved"]:]
            parents[i, gone] = stay[torch.arange(len(gone)) % len(stay)].to(torch.int32)
        state = {"tensors": tensors, "slots": slots.to(DEV), "parents": parents.to(DEV)}
    else:
        dtype, page, D = TYPES[case["dtype"]], case["page"], case["dim"]
        Hq, Hkv = case["heads"], case["kv_heads"]
        lengths = _lengths(case)
        blocks = -(-max(n for n, _ in lengths) // page)
        need = sum(s // page + B * (-(-n // page) - s // page) for n, s in lengths)
        ids = torch.randperm(need, generator=h).to(torch.int32)
        table = torch.full((G * B, blocks), -1, dtype=torch.int32)
        at = 0
        cache = torch.randn(need, 2, Hkv, page, D, device=DEV, generator=g).to(dtype)
        for i, (n, s) in enumerate(lengths):
            m, k = -(-n // page), s // page
            table[i * B:(i + 1) * B, :k] = ids[at:at + k]
            at += k
            for b in range(B):
                table[i * B + b, k:m] = ids[at:at + m - k]
                at += m - k
                if n % page:                              # nobody has written the rest of the last page
                    last = int(table[i * B + b, m - 1])
                    cache[last, 0, :, n % page:] = math.nan
                    cache[last, 1].view(Hkv, D, page)[:, :, n % page:] = math.nan
        state = {"q": (torch.randn(G * B, Hq * D, device=DEV, generator=g) * 1.5).to(dtype), "cache": cache, "table": table.to(DEV),
                 "lens": torch.tensor([n for n, _ in lengths for _ in range(B)], dtype=torch.int32, device=DEV),
                 "shared": torch.tensor([s for _, s in lengths], dtype=torch.int32, device=DEV),
                 "out": torch.empty(G * B, Hq * D, dtype=dtype, device=DEV), "scratch": torch.empty(1 << 24, device=DEV)}
    state["case"] = case
    return state


# ------------------------------------------------------------------------------- the plain forms
def _select(state):
    case = state["case"]
    G, B, V, K = case["groups"], case["beams"], case["vocab"], case["keep"]
    z = torch.where(torch.isnan(state["logits"]), -math.inf, state["logits"]).double()
    top = z.amax(1, keepdim=True)
    x = torch.where(z == top, 0.0, z - top)               # (also where the largest is infinite)
    x = torch.where(z == -math.inf, -math.inf, x)
    keys = state["scores"].double()[:, None] + (x - torch.log(torch.exp(x).sum(1, keepdim=True)))
    keys = torch.where(torch.isnan(keys), -math.inf, keys).view(G, B * V)
    if K > B * V:
        keys = torch.nn.functional.pad(keys, (0, K - B * V), value=-math.inf)
    # the K largest, the lowest places among equals: first the K-th key, then the places by (above it, equal to it)
    least = torch.topk(keys, K).values[:, -1:]
    place = torch.arange(keys.shape[1], device=keys.device)
    rank = torch.where(keys > least, place, torch.where(keys == least, place + keys.shape[1], place + 2 * keys.shape[1]))
    places = torch.sort(torch.topk(rank, K, largest=False).values % keys.shape[1]).values
    found, order = torch.sort(keys.gather(1, places), dim=1, descending=True, stable=True)
    places, none = places.gather(1, order), found == -math.inf
    return {"scores": found.float(), "parents": torch.where(none, -1, places // V).int(), "tokens": torch.where(none, -1, places % V).int()}


def _reorder(state):
    from_rows = torch.gather(state["slots"].long(), 1, state["parents"].long()).view(-1)
    to_rows = state["slots"].long().view(-1)
    dim = 1 if state["case"]["stacked"] else 0
    return [t.index_copy_(dim, to_rows, t.index_select(dim, from_rows)) for t in state["tensors"]]


def _attention(state):
    case = state["case"]
    S, Hq, Hkv, D, page = case["groups"] * case["beams"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    pages, table = state["cache"], state["table"].long().clamp(min=0)
    n = table.shape[1] * page
    k = pages[:, 0][table].float().permute(0, 2, 1, 3, 4).reshape(S, Hkv, n, D)
    v = pages[:, 1].reshape(-1, Hkv, D, page)[table].float().permute(0, 2, 1, 4, 3).reshape(S, Hkv, n, D)
    seen = (torch.arange(n, device=DEV) < state["lens"][:, None])[:, None, :, None]
    k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
    scores = torch.matmul(state["q"].float().view(S, Hkv, Hq // Hkv, D), k.transpose(2, 3)) * (D ** -0.5)
    scores = torch.where(seen.transpose(2, 3), scores, -math.inf)
    w = torch.exp(scores - scores.amax(3, keepdim=True))
    return torch.matmul(w / w.sum(3, keepdim=True), v).reshape(S, Hq * D).to(state["out"].dtype)


def run(state):
    case = state["case"]
    if own:
        from deliverance_amd.kernels import ops
        if case["op"] == "select":
            scores, parents, tokens = ops.beam_select(state["logits"], state["scores"], case["beams"], *state["out"], workspace=state["scratch"])
            return {"scores": scores, "parents": parents, "tokens": tokens}
        if case["op"] == "reorder":
            return ops.state_reorder(state["tensors"], state["slots"], state["parents"], dim=1 if case["stacked"] else 0)
        splits = ops.beam_splits(case["groups"], case["beams"], case["heads"], case["kv_heads"], case["dim"], state["table"].shape[1], case["page"],
                                 TYPES[case["dtype"]])
        return ops.attention_beams(state["q"], state["cache"], state["table"], state["lens"], state["shared"], case["beams"], case["heads"],
                                   case["dim"] ** -0.5, None, state["out"], splits, state["scratch"])
    return {"select": _select, "reorder": _reorder, "attention": _attention}[case["op"]](state)


# ------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "select":
        G, B, V, K = case["groups"], case["beams"], case["vocab"], case["keep"]
        scores, parents, tokens = [], [], []
        for g in range(G):
            logp = torch.log_softmax(state["logits"][g * B:(g + 1) * B].double(), 1) + state["scores"][g * B:(g + 1) * B].double()[:, None]
            flat = torch.nan_to_num(logp, nan=-math.inf, neginf=-math.inf).view(-1)
            value, place = torch.sort(flat, descending=True, stable=True)
            value, place = value[:K].cpu(), place[:K].cpu()
            short = K - len(value)
            value = torch.cat([value, torch.full((short,), -math.inf, dtype=torch.float64)])
            place = torch.cat([place, torch.zeros(short, dtype=torch.long)])
            there = value > -math.inf
            scores.append(value)
            parents.append(torch.where(there, place // V, -1).int())
            tokens.append(torch.where(there, place % V, -1).int())
        return {"scores": torch.stack(scores), "parents": torch.stack(parents), "tokens": torch.stack(tokens)}
    if case["op"] == "reorder":
        moves = [(int(s[b]), int(s[p[b]])) for s, p in zip(state["slots"].cpu(), state["parents"].cpu()) for b in range(case["beams"]) if int(p[b]) != b]
        out = []
        for t in state["tensors"]:
            before = t.double()
            rows = before.transpose(0, 1) if case["stacked"] else before
            for to, came in moves:                        # (who is continued stays where it was)
                rows[to] = rows[came]
            out.append(before)
        return out
    S, Hq, Hkv, D, page = case["groups"] * case["beams"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(S, Hq, D, dtype=torch.float64, device=DEV)
    for s in range(S):
        n = int(state["lens"][s])
        ids = state["table"][s, :-(-n // page)].long()
        keys = state["cache"][ids, 0].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        values = state["cache"][ids, 1].double().reshape(len(ids), Hkv, D, page).permute(1, 2, 0, 3).reshape(Hkv, D, -1)[:, :, :n]
        q = state["q"][s].double().view(Hkv, Hq // Hkv, D)
        for h in range(Hkv):
            p = torch.softmax(q[h] @ keys[h].T / math.sqrt(D), 1)
            out[s, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)] = p @ values[h].T
    return out.view(S, Hq * D)
