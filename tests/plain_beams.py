"""Beam search written plainly: every beam's logits from the whole sequence, in numpy."""
import math

import numpy as np


def beam_search(logits_of, prompt, n_beams, max_new, ends=(), length_penalty=1.0, early_stopping=False):
    """``logits_of(ids)``: the last position's logits.  Returns (hypotheses [(rank, score, tokens)], best first; the smallest gap between two
    numbers whose order decides what is returned: the last candidate that goes on and the one behind it, with end tokens the last
    that may end a hypothesis and the one behind it, and the hypotheses' ranks)."""
    beams, finished, gap = [(0.0, [])], [], math.inf
    keep = n_beams * (1 + len(ends))
    for step in range(max_new):
        found = []
        for i, (score, tokens) in enumerate(beams):
            z = np.asarray(logits_of(list(prompt) + tokens), dtype=np.float64)
            z = z - z.max()
            z = z - math.log(np.exp(z).sum())
            found += [(score + z[v], i, v) for v in np.argsort(-z, kind="stable")[:keep + 1].tolist()]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        edges = {n_beams - 1} if ends else set()
        old, beams = beams, []
        for rank, (score, i, v) in enumerate(found[:keep]):
            if len(beams) == n_beams:
                break
            if v in ends:
                if rank < n_beams:
                    tokens = old[i][1] + [v]
                    finished.append((score / len(tokens) ** length_penalty, score, tokens))
            else:
                beams.append((score, old[i][1] + [v]))
                if len(beams) == n_beams:
                    edges.add(rank)
        gap = min([gap] + [found[e][0] - found[e + 1][0] for e in edges if e + 1 < len(found)])
        finished = sorted(finished, key=lambda h: -h[0])[:n_beams]
        if step == max_new - 1:
            finished += [(s / len(t) ** length_penalty, s, t) for s, t in beams]
            break
        if len(finished) == n_beams and (early_stopping or finished[-1][0] >= beams[0][0] / (step + 1) ** length_penalty):
            break
    finished = sorted(finished, key=lambda h: -h[0])
    gap = min([gap] + [a[0] - b[0] for a, b in zip(finished[:n_beams], finished[1:])])
    return finished[:n_beams], gap
