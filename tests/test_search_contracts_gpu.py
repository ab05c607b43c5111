"""What the operators of a search over beams say of themselves, held to the last place that they promise."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_beam_kernels_gpu import BF16_HALF, DEV, F32_HALF, Shared, err_word, i32, select_inputs, select_oracle
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


def test_sums_that_go_on_for_hundreds_of_steps():
    """Selections and what follows from them, a step on the other, against the same in 64 bits on the host: which beams go on, with which
    tokens, and their sums, as far as a row's logarithm is off (2e-13 a step) and a place of 64 bits near 4,000 (2^-41) a step."""
    groups, beams, vocab, k, steps, stops = 3, 6, 2003, 18, 500, [5, 77]
    rng = np.random.default_rng(8)
    slots = i32(np.arange(groups * beams).reshape(groups, beams))
    scores = torch.zeros(groups, beams, dtype=torch.float64, device=DEV)
    scores[:, 1:] = -float("inf")
    parents, tokens = torch.zeros_like(slots), torch.zeros_like(slots)
    want = scores.cpu().numpy().copy()
    stop_tokens, err = i32(stops), err_word()
    for step in range(steps):
        x = (rng.standard_normal((groups * beams, vocab)) * 2.0).astype(np.float32)
        cand = ops.beam_select(torch.from_numpy(x).to(DEV), scores, k, score_dtype=torch.float64)
        assert cand[0].dtype == torch.float64
        ops.beam_advance(cand, stop_tokens, slots, scores, parents, tokens, err)
        live = np.where(np.isfinite(want), want, -1e30)
        keys, by, tok = ranked(x, live, k)
        got = tuple(t.cpu().numpy() for t in cand)
        np.testing.assert_array_equal(got[1], by)
        np.testing.assert_array_equal(got[2], tok)
        assert np.abs(got[0] - keys).max() <= (step + 1) * (2e-13 + 2.0 ** -41)
        new = np.empty_like(want)
        for g in range(groups):
            seats, late = [None] * beams, []
            for c in [c for c in range(k) if tok[g, c] not in stops][:beams]:
                if seats[by[g, c]] is None:
                    seats[by[g, c]] = c
                else:
                    late.append(c)
            for c in late:
                seats[seats.index(None)] = c
            new[g] = keys[g][seats]
            assert parents[g].tolist() == by[g][seats].tolist() and tokens[g].tolist() == tok[g][seats].tolist()
        want = new
        assert np.abs(scores.cpu().numpy() - want).max() <= (step + 1) * (2e-13 + 2.0 ** -41)
    assert err.tolist()[0] == 0


@pytest.mark.parametrize("kind", ["normal", "rising", "few_values", "masked", "nothing", "infinite", "dead", "far", "equal"])
@pytest.mark.parametrize("groups,beams,vocab,k", [(2, 4, 30001, 8), (1, 1, 6, 6), (1, 64, 4099, 256), (145, 4, 9001, 8)])
def test_selection_with_sums_in_64_bits(groups, beams, vocab, k, kind):
    x, s = select_inputs(kind, groups, beams, vocab, seed=4)
    s = s.astype(np.float64) + (0.0 if kind in ("equal", "few_values") else np.random.default_rng(1).random(s.shape) * 1e-9)
    got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), k, score_dtype=torch.float64)
    for part in (slice(0, 2), slice(max(0, groups - 1), groups)):
        rows = slice(part.start * beams, min(part.stop, groups) * beams)
        keys, parents, tokens = select_oracle(x[rows], s[part], k)
        scores = got[0][part].cpu().numpy()
        finite = np.isfinite(keys)
        assert np.array_equal(np.isneginf(scores), np.isneginf(keys))
        # 1.5e-13 of a row's sum for the series, places of 64 bits (of keys up to some hundred) for the rest
        assert np.abs(scores[finite] - keys[finite]).max(initial=0.0) <= 2e-13 + 2.0 ** -51 * np.abs(keys[finite]).max(initial=0.0)
        np.testing.assert_array_equal(got[1][part].cpu().numpy(), parents)
        np.testing.assert_array_equal(got[2][part].cpu().numpy(), tokens)


def test_sums_of_another_type_are_refused():
    x, s = torch.zeros(6, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)
    wide = (s.double()[:, :1].contiguous(), ints(2, 1), ints(2, 1))
    for bad in (lambda: ops.beam_select(x, s, 4, score_dtype=torch.float64), lambda: ops.beam_select(x, s.double(), 4),
                lambda: ops.beam_select(x, s.half(), 4, score_dtype=torch.float16),
                lambda: ops.beam_select(x, s.double(), 4, score_dtype=torch.float64, out=(torch.zeros(2, 4, device=DEV), ints(2, 4), ints(2, 4))),
                lambda: ops.beam_advance(wide, None, ints(2, 3), s, ints(2, 3), ints(2, 3), err_word()),
                lambda: ops.beam_advance((wide[0].float(),) + wide[1:], None, ints(2, 3), s.double(), ints(2, 3), ints(2, 3), err_word()),
                lambda: ops.beam_advance((wide[0].half(),) + wide[1:], None, ints(2, 3), s.half(), ints(2, 3), ints(2, 3), err_word())):
        with pytest.raises(ops.KernelError):
            bad()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 32)])
def test_scales_and_caps_that_are_none_are_refused(dtype, d):
    """The maximum of the scores is taken before they are scaled."""
    c = Shared([3], [90], 20, d=d, dtype=dtype, seed=3).device()
    for bad in (dict(scale=0.0), dict(scale=-0.125), dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-5.0),
                dict(softcap=float("nan")), dict(softcap=float("inf"))):
        with pytest.raises(ops.KernelError):
            ops.attention_shared(c.dq, c.out, c.dk, c.dv_, c.shared(), *c.args, **{**c.kw, **bad})
    assert bool(torch.isnan(c.out).all())
    c.kw["softcap"] = 0.0                      # no cap
    c.call()
    c.check()


def in_float32(c):
    """The oracle's sums in float32, one request after the other."""
    starts, outs = np.cumsum([0] + list(c.members)), []
    for r, g in enumerate(c.group_of):
        pos, p = int(c.positions[r]), c.prefixes[g]
        slots = [c.prefix_slot[g] if t < p else c.slots[r] if c.history is None or t == pos else c.slots[starts[g] + c.history[c.slots[r], t - p]]
                 for t in range(pos + 1)]
        at = [c.table[s, t // c.page] for t, s in enumerate(slots)]
        k = torch.stack([c.k[a, :, t % c.page] for t, a in enumerate(at)])
        v = torch.stack([c.v[a, :, t % c.page] for t, a in enumerate(at)])
        x = torch.einsum("hpd,khd->hpk", c.q[r].view(c.hkv, -1, c.d), k) * c.scale
        if c.softcap:
            x = c.softcap * torch.tanh(x / c.softcap)
        outs.append(torch.einsum("hpk,khd->hpd", torch.softmax(x, -1), v).reshape(c.hq, c.dv))
    return torch.stack(outs).double()


@pytest.mark.parametrize("softcap", [None, 5.0, 30.0, 50.0])
@pytest.mark.parametrize("history", [False, True])
def test_float32_shared_attention_is_as_good_as_float32(softcap, history):
    """Its error, as a root mean square, beside that of the same sums in elementary float32 operations: half as much again for another
    order of the additions."""
    c = Shared([4, 3], [300, 130], 60, hq=8, hkv=2, d=64, dtype=torch.float32, history=history, softcap=softcap, seed=41).device()
    c.call()
    c.check()
    want = c.oracle()[0]
    rms = lambda x: float((x - want).pow(2).mean().sqrt())
    assert rms(c.out.cpu().double()) <= 1.5 * rms(in_float32(c))


def test_nearly_equal_scores_in_one_group_of_several_and_in_a_graph():
    """Rows that lie apart at any address; what one replay found in doubt is nothing to the next."""
    groups, beams, vocab, k = 3, 8, 20011, 12
    cases = []
    for seed in (11, 12):
        x, s = select_inputs("normal", groups, beams, vocab, seed=seed)
        x[beams:2 * beams], s[1:2] = nearly_equal("normal", beams, vocab, seed)
        cases.append((x, s) + ranked(x, s, k))
        gaps = np.abs(np.diff(cases[-1][2], axis=1))
        assert gaps.min() > 4e-13 and gaps[1].min() < 1e-8 < 1e-5 < gaps[[0, 2]].min()
    memory = torch.full((3 + groups * beams * (vocab + 5),), float("nan"), device=DEV)
    logits = memory[3:].view(groups * beams, vocab + 5)[:, :vocab]
    scores = torch.zeros(groups, beams, device=DEV)
    graph, out = torch.cuda.CUDAGraph(), None
    ops.beam_select(logits, scores, k)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.beam_select(logits, scores, k)
    for x, s, _, parents, tokens in cases + cases[:1]:
        logits.copy_(torch.from_numpy(x))
        scores.copy_(torch.from_numpy(s))
        graph.replay()
        np.testing.assert_array_equal(out[1].cpu().numpy(), parents)
        np.testing.assert_array_equal(out[2].cpu().numpy(), tokens)
