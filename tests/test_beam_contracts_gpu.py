"""What the operators of a search over beams say of themselves, held to the last place that they promise."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_beam_kernels_gpu import BF16_HALF, DEV, F32_HALF, Shared, err_word, i32
from tokamak_b200.csrc import ops

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ attention

def check_one_rounding(c):
    """Of a bfloat16 result only its own rounding may be seen: a probability is two bfloat16, so what is left of its rounding is the
    second's, a half step of a half step; scores and sums are floats."""
    want, weight, size = c.oracle()
    score = (c.d + 4) * F32_HALF * size + 2.0 ** -22 + (1e-6 * c.softcap if c.softcap else 0.0)
    keys = int(c.positions.max()) + 1
    tol = (2 * score + keys ** 0.5 * F32_HALF * 4 + BF16_HALF * BF16_HALF) * weight
    off = (c.out.cpu().double() - want).abs()
    beyond = off - (tol + BF16_HALF * (want.abs() + tol))
    assert beyond.max() <= 0, f"{int((beyond > 0).sum())} of {beyond.numel()} elements are off by more than their rounding"
    assert c.err.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("form", [
    dict(members=[4], prefixes=[700], own=1),                                         # shared positions, groups of lanes in turns
    dict(members=[40, 33], prefixes=[300, 200], own=1, hq=8),                         # two tiles of query rows
    dict(members=[6], prefixes=[130], own=90, history=True, common=80),               # a common past
    dict(members=[3], prefixes=[0], own=150, hq=8),                                   # own positions alone
    dict(members=[5], prefixes=[40], own=200, history=True),                          # own positions of several writers
    dict(members=[2], prefixes=[70], own=600),                                        # cut into parts
    dict(members=[4], prefixes=[500], own=60, history=True, window=256, softcap=30.0, sinks=True)])
def test_shared_attention_is_off_by_its_own_rounding_only(form, d):
    c = Shared(**form, d=d, dtype=torch.bfloat16, seed=31).device()
    c.call()
    check_one_rounding(c)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 32)])
@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("window", [None, 50])
def test_a_row_with_a_position_that_is_none_sees_nothing(window, history, dtype, d):
    """Not the shared positions either; the other members of its group are what they are without it."""
    c = Shared([3, 2], [140, 50], 20, d=d, dtype=dtype, history=history, window=window, seed=12).device()
    c.call()
    c.check()
    whole = c.out.clone()
    place = c.table.shape[1] * c.page                    # the first position that the block table has no place for
    for bad in (place, 10 ** 6, -1, -10 ** 6):
        positions = c.positions.copy()
        positions[[1, 4]] = bad
        c.out.fill_(float("nan"))
        c.err.zero_()
        ops.attention_shared(c.dq, c.out, c.dk, c.dv_, c.shared(), i32(positions), *c.args[1:], **c.kw)
        assert c.err.tolist()[0] == 3
        assert bool((c.out[[1, 4]] == 0).all()), bad
        # (parts may be cut elsewhere without a common past: floats are added in another order)
        half = BF16_HALF if dtype == torch.bfloat16 else F32_HALF
        torch.testing.assert_close(c.out[[0, 2, 3]].float(), whole[[0, 2, 3]].float(), rtol=2 * half, atol=2.0 ** -12)


# ------------------------------------------------------------------------------------------------ selection

def ranked(x: np.ndarray, scores: np.ndarray, k: int):
    """``(keys, parents, tokens)`` as ``ops.beam_select`` describes them, in 64 bits: by key, then the lower beam, then the larger
    logit, then the lower token.  Finite logits and scores."""
    groups, beams = scores.shape
    vocab = x.shape[1]
    wide = x.astype(np.float64)
    d = wide - wide.max(axis=1, keepdims=True)
    keys = scores.astype(np.float64).reshape(-1, 1) + (d - np.log(np.exp(d).sum(axis=1, keepdims=True)))
    beam, token = np.divmod(np.arange(beams * vocab), vocab)
    out = []
    for g in range(groups):
        rows = slice(g * beams, (g + 1) * beams)
        order = np.lexsort((token, -wide[rows].reshape(-1), beam, -keys[rows].reshape(-1)))[:k]
        out.append((keys[rows].reshape(-1)[order], beam[order], token[order]))
    return tuple(np.stack(a) for a in zip(*out))


@pytest.mark.parametrize("beams,vocab,k", [(2, 2, 4), (3, 50, 40), (8, 9001, 64), (64, 4099, 256), (4, 50001, 16)])
def test_equal_scores_of_beams_whose_logits_differ_by_a_constant(beams, vocab, k):
    """Rows of whole numbers that differ by a whole number have the same keys to the last bit: the lower beam comes first, whatever
    its logits are."""
    rng = np.random.default_rng(vocab)
    base = rng.integers(-9, 6, (2, 1, vocab))
    x = (base + rng.permutation(np.arange(beams) * 5 - beams)[None, :, None]).reshape(2 * beams, vocab).astype(np.float32)
    s = np.full((2, beams), -3.0, dtype=np.float32)
    got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), k)
    keys, parents, tokens = ranked(x, s, k)
    assert (keys[:, 1:] == keys[:, :-1]).any()
    np.testing.assert_array_equal(got[1].cpu().numpy(), parents)
    np.testing.assert_array_equal(got[2].cpu().numpy(), tokens)


def test_equal_scores_of_one_beam_go_by_the_logit():
    """Logits so small beside the row's largest that their keys are the same in 64 bits."""
    x = np.zeros((4, 40), dtype=np.float32)
    x[:, 7] = 12.0
    x[:, 8:40] = np.float32(1e-30) * np.arange(1, 33, dtype=np.float32)
    s = np.full((1, 4), -1.0, dtype=np.float32)
    got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), 60)
    keys, parents, tokens = ranked(x, s, 60)
    assert tokens[0, 4:8].tolist() == [39, 38, 37, 36] and parents[0, 4:36].tolist() == [0] * 32
    np.testing.assert_array_equal(got[1].cpu().numpy(), parents)
    np.testing.assert_array_equal(got[2].cpu().numpy(), tokens)


def nearly_equal(kind, beams, vocab, seed):
    """Rows of logits, and scores with which the best continuations of all beams have keys within a score's last place."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((beams, vocab)) * 2.5).astype(np.float32)
    if kind == "low_start":                    # what a row begins with is far below the rest
        x[:, :vocab // 3] -= np.float32(20.0) + np.arange(beams, dtype=np.float32)[:, None] * np.float32(0.37)
    elif kind == "high":                       # a few tokens well above the rest, anywhere
        x[np.arange(beams)[:, None], rng.integers(0, vocab, (beams, 24))] += (rng.random((beams, 24)) * 9.0).astype(np.float32)
    elif kind == "flat":                       # many tokens that weigh alike, rows at different heights
        x = x * np.float32(0.2) + np.arange(beams, dtype=np.float32)[:, None] * np.float32(1.7)
    wide = x.astype(np.float64)
    top = wide.max(axis=1)
    logp = -np.log(np.exp(wide - top[:, None]).sum(axis=1))
    return x, (logp[0] - logp).astype(np.float32)[None, :]


@pytest.mark.parametrize("kind,beams,vocab,seed", [("normal", 64, 20011, 1), ("normal", 24, 151936, 2), ("low_start", 64, 20011, 3),
                                                   ("low_start", 24, 100003, 4), ("high", 64, 50001, 5), ("flat", 64, 20011, 6)])
def test_scores_that_nearly_are_equal_come_in_their_order(kind, beams, vocab, seed):
    x, s = nearly_equal(kind, beams, vocab, seed)
    keys, parents, tokens = ranked(x, s, beams)
    gaps = -np.diff(keys[0])
    # a row's logarithm is off by up to 1.5e-13 for the series of its exponentials and, sums of some hundred additions a thread and a tree
    # over the threads, by 100 * 2^-53 = 1.2e-14 for each side's sums; a key near 10 by 2^-50: two rows by 3.5e-13 in all
    assert gaps.min() > 4e-13 and np.median(gaps) < 2e-8
    for k in (beams, 1, 5, beams // 2):              # the last that is wanted, and the one behind it, are as close
        got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), k)
        np.testing.assert_array_equal(got[1].cpu().numpy(), parents[:, :k])
        np.testing.assert_array_equal(got[2].cpu().numpy(), tokens[:, :k])
