"""A plain search over beams: whole-sequence log probabilities in 64 bits, one sequence at a time."""

from __future__ import annotations

import math

import torch


def search(logits_of, prompt, width, max_new, stops=(), length_penalty=1.0, early_stopping=False):
    """``[(tokens, sum of log probabilities, ended)]`` best first, and the smallest difference between the keys of
    neighbours in the ranked continuations that decided something.  ``logits_of(tokens)`` gives the last token's logits."""
    beams, ended, gap = [([], 0.0)], [], math.inf
    for step in range(max_new):
        ranked = []
        for b, (tokens, score) in enumerate(beams):
            logp = torch.log_softmax(logits_of(list(prompt) + tokens).double(), -1)
            top = torch.topk(logp, min(width * (1 + len(stops)) + 1, logp.numel()))
            ranked += [(score + float(v), b, int(t)) for v, t in zip(top.values, top.indices)]
        ranked.sort(key=lambda x: -x[0])
        new = []
        for i, (score, b, token) in enumerate(ranked):
            if i + 1 < len(ranked):
                gap = min(gap, score - ranked[i + 1][0])
            if len(new) == width:
                break
            if token in stops:
                ended.append((beams[b][0] + [token], score, True))
            else:
                new.append((beams[b][0] + [token], score))
        beams = new
        key = lambda h: -h[1] / len(h[0]) ** length_penalty
        ended = sorted(ended, key=key)[:width]
        if len(ended) == width:
            if early_stopping or max(s for _, s in beams) / (step + 1) ** length_penalty <= -key(ended[-1]):
                break
    if len(ended) < width or len(beams[0][0]) >= max_new:
        ended = ended + [(t, s, False) for t, s in beams]
    return sorted(ended, key=key)[:width], gap
