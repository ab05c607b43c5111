"""Selection over beams, the beams that go on, records that follow them, and attention over shared prefixes, against their
definitions in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tokamak_b200.csrc import ops
from tokamak_b200.csrc.ops import KernelError, SharedPrefix

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32_HALF = 2.0 ** -24
BF16_HALF = 2.0 ** -8


def err_word():
    return torch.zeros(4, dtype=torch.int32, device=DEV)


def i32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).to(DEV)


# ------------------------------------------------------------------------------------------------ selection

def select_oracle(logits: np.ndarray, scores: np.ndarray, k: int):
    """``(keys, parents, tokens)`` by the definition in 64 bits: keys, then (within a beam) logits, then places."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    x = logits.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    keys = np.full_like(x, -np.inf)
    flat_scores = scores.astype(np.float64).reshape(-1)
    for r in range(x.shape[0]):
        s = flat_scores[r]
        top = x[r].max()
        if not s > -np.inf or top == -np.inf:
            continue
        if top == np.inf:
            keys[r][x[r] == np.inf] = s - math.log(int((x[r] == np.inf).sum()))
            continue
        d = x[r] - top
        keys[r] = s + (d - math.log(np.exp(d).sum()))
    logit = np.where(np.isneginf(keys), -np.inf, x)
    keys, logit = keys.reshape(groups, -1), logit.reshape(groups, -1)
    out = []
    for g in range(groups):
        order = np.lexsort((np.arange(beams * vocab), -logit[g], -keys[g]))[:k]
        out.append((keys[g][order], order // vocab, order % vocab))
    return tuple(np.stack(a) for a in zip(*out))


def select_inputs(kind, groups, beams, vocab, seed=0):
    rng = np.random.default_rng(seed)
    rows = groups * beams
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    s = (-20.0 - 3.0 * rng.random((groups, beams))).astype(np.float32)
    if kind == "peaked":
        x[np.arange(rows), rng.integers(0, vocab, rows)] += 40.0
    elif kind == "rising":
        x = np.sort(x, axis=1)
    elif kind == "falling":
        x = -np.sort(-x, axis=1)
    elif kind == "equal":                    # every logit the same, beams with the same score too
        x[:] = 1.25
        s[:] = -7.0
    elif kind == "few_values":               # long ties at the border
        x = np.round(x).astype(np.float32)
        s = np.repeat(s[:, :1], beams, axis=1)
    elif kind == "masked":                   # a mask of -inf, one of the type's lowest value, and NaN
        x[:, ::3] = -np.inf
        x[:, 1::5] = np.finfo(np.float32).min
        x[:, 2::7] = np.nan
    elif kind == "nothing":                  # rows that leave nothing
        x[::2] = -np.inf
    elif kind == "all_lowest":
        x[0] = np.finfo(np.float32).min
    elif kind == "infinite":
        x[0, [0, vocab // 2]] = np.inf
        if rows > 1:
            x[1, vocab - 1] = np.inf
    elif kind == "dead":                     # beams that cannot go on; the group's first only may
        s[:, 1:] = -np.inf
        if beams > 2:
            s[:, 2] = np.nan
        x[1:] = np.nan
    elif kind == "far":                      # logits that a sum with a fixed reference would lose
        x += np.where(np.arange(vocab) > vocab // 2, 500.0, -500.0).astype(np.float32)
    return x, s


def check_selection(x, s, k, got):
    keys, parents, tokens = select_oracle(x, s, k)
    scores = got[0].cpu().numpy().astype(np.float64)
    finite = np.isfinite(keys)
    assert np.array_equal(np.isneginf(scores), np.isneginf(keys))
    # rounded once to float32; the sum of the exponentials: 2^-23 of an exponential's own error, 2^-23 of two additions of
    # floats, 2^-24 |x - ref| of the difference's rounding, which weighs at most ln(vocab) + 1 on average over a softmax
    slack = 2.0 ** -22 + F32_HALF * (math.log(x.shape[1]) + 1.0)
    off = np.abs(scores - np.where(finite, keys, 0.0))
    assert np.all(off[finite] <= F32_HALF * np.abs(keys[finite]) + slack), off[finite].max()
    np.testing.assert_array_equal(got[1].cpu().numpy(), parents)
    np.testing.assert_array_equal(got[2].cpu().numpy(), tokens)


SELECT = [(1, 1, 7, 7, "normal"), (1, 1, 1, 1, "normal"), (2, 3, 5, 15, "normal"), (1, 1, 151936, 8, "normal"),
          (2, 4, 317, 8, "normal"), (3, 5, 50001, 17, "normal"), (1, 64, 4099, 256, "normal"), (5, 2, 8192, 1, "peaked"),
          (2, 4, 151936, 8, "rising"), (1, 2, 65536, 33, "falling"), (1, 4, 20000, 64, "equal"), (1, 64, 4096, 256, "equal"),
          (2, 8, 9001, 16, "few_values"), (2, 3, 12289, 12, "masked"), (2, 4, 1000, 8, "nothing"), (1, 1, 6, 6, "nothing"),
          (1, 2, 4097, 10, "all_lowest"), (1, 3, 30001, 6, "infinite"), (3, 4, 5000, 8, "dead"), (1, 4, 3, 12, "dead"),
          (1, 2, 40000, 9, "far"), (40, 16, 1001, 32, "normal"), (300, 1, 8200, 4, "normal")]


@pytest.mark.parametrize("groups,beams,vocab,k,kind", SELECT)
def test_selection(groups, beams, vocab, k, kind):
    x, s = select_inputs(kind, groups, beams, vocab)
    got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), k)
    check_selection(x, s, k, got)


@pytest.mark.parametrize("kind", ["normal", "rising", "few_values", "far"])
@pytest.mark.parametrize("k", [8, 256])
def test_selection_in_long_segments(k, kind):
    """Rows enough for one segment each: many tiles between the first threshold and the last."""
    x, s = select_inputs(kind, 145, 4, 60007, seed=3)
    got = ops.beam_select(torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV), k)
    some = slice(0, 2)                           # the oracle sorts every group: the first two and the last
    check_selection(x[:8], s[some], k, tuple(t[some] for t in got))
    check_selection(x[-4:], s[-1:], k, tuple(t[-1:] for t in got))


@pytest.mark.parametrize("offset,extra", [(0, 1), (1, 0), (2, 5), (3, 2)])
def test_selection_of_rows_that_start_on_any_four_bytes(offset, extra):
    groups, beams, vocab, k = 2, 3, 9973, 12
    x, s = select_inputs("normal", groups, beams, vocab, seed=3)
    rows, ld = groups * beams, vocab + extra
    memory = torch.full((offset + rows * ld + 8,), float("inf"), device=DEV)          # what lies around the rows is not read
    view = memory[offset:offset + rows * ld].view(rows, ld)[:, :vocab]
    view.copy_(torch.from_numpy(x))
    check_selection(x, s, k, ops.beam_select(view, torch.from_numpy(s).to(DEV), k))


def test_selection_captured_twice_and_on_two_streams():
    cases = []
    for seed in (1, 2):
        x, s = select_inputs("normal", 2, 4, 30000, seed=seed)
        cases.append((x, s, torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV)))
    ops.beam_select(cases[0][2], cases[0][3], 8)
    graphs, outs = [], []
    for _, _, tx, ts in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.beam_select(tx, ts, 8))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (x, s, _, _), out in zip(cases, outs):
        check_selection(x, s, 8, out)
    # other logits through the same graph
    cases[0][2].copy_(cases[1][2]); cases[0][3].copy_(cases[1][3])
    graphs[0].replay()
    torch.cuda.synchronize()
    check_selection(cases[1][0], cases[1][1], 8, outs[0])


def test_selection_refuses():
    x, s = torch.zeros(6, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    for bad in (lambda: ops.beam_select(x.cpu(), s, 4), lambda: ops.beam_select(x.bfloat16(), s, 4),
                lambda: ops.beam_select(x.t(), s, 4), lambda: ops.beam_select(x, s.view(-1), 4),
                lambda: ops.beam_select(x[:5], s, 4), lambda: ops.beam_select(x, s, 0), lambda: ops.beam_select(x, s, 151),
                lambda: ops.beam_select(torch.zeros(65, 300, device=DEV), torch.zeros(1, 65, device=DEV), 4),
                lambda: ops.beam_select(torch.zeros(6, 500, device=DEV), s, 257),
                lambda: ops.beam_select(x, s.double(), 4),
                lambda: ops.beam_select(x[:1].expand(6, 50), s, 4),
                lambda: ops.beam_select(x, s, 4, out=(torch.empty(2, 4, device=DEV),) * 3),
                lambda: ops.beam_select(x, s, 4, out=(torch.empty(2, 5, device=DEV), torch.empty(2, 5, dtype=torch.int32, device=DEV),
                                                      torch.empty(2, 5, dtype=torch.int32, device=DEV)))):
        with pytest.raises(KernelError):
            bad()
    empty = ops.beam_select(torch.zeros(0, 50, device=DEV), torch.zeros(0, 3, device=DEV), 4)
    assert empty[0].shape == (0, 4)


# ------------------------------------------------------------------------------------------------ the beams that go on

def advance_oracle(cand, stops, beams, begin):
    scores, parents, tokens = [], [], []
    for cs, cp, ct in zip(*[c.tolist() for c in cand]):
        picked = []
        for a, b, c in zip(cs, cp, ct):
            if not a > -math.inf:
                break
            if c not in stops and len(picked) < beams:
                picked.append((a, b, c))
        seats, late = [None] * beams, []
        for i, (a, b, c) in enumerate(picked):
            want = i if begin else b
            if seats[want] is None:
                seats[want] = (a, want if begin else b, c)
            else:
                late.append((a, b, c))
        for x in late:
            seats[seats.index(None)] = x
        seats = [(-math.inf, i, 0) if x is None else x for i, x in enumerate(seats)]
        scores.append([x[0] for x in seats]); parents.append([x[1] for x in seats]); tokens.append([x[2] for x in seats])
    return scores, parents, tokens


@pytest.mark.parametrize("groups,beams,k,n_stop,begin", [(1, 1, 1, 0, False), (3, 4, 8, 1, False), (2, 4, 8, 0, True),
                                                         (2, 8, 9, 3, False), (1, 64, 256, 2, False), (4, 3, 4, 2, True)])
def test_beams_that_go_on(groups, beams, k, n_stop, begin):
    rng = np.random.default_rng(5)
    vocab = 6 if beams < 64 else 40
    scores = -np.sort(rng.random((groups, k))).astype(np.float32)
    scores[-1, k // 2 + 1:] = -np.inf                                    # fewer than beams may be left
    parents = rng.integers(0, 1 if begin else beams, (groups, k))
    tokens = rng.integers(0, vocab, (groups, k))
    stops = list(range(n_stop))
    cand = (torch.from_numpy(scores).to(DEV), i32(parents), i32(tokens))
    max_slots = groups * beams + 3
    slots = rng.permutation(max_slots)[:groups * beams].reshape(groups, beams)
    records = torch.full((max_slots, 8), -5, dtype=torch.int32, device=DEV)
    history = torch.full((max_slots, 32), 99, dtype=torch.uint8, device=DEV)
    prefix = i32(np.arange(groups) * 3 + 7)
    step = 5
    positions = i32(np.repeat(np.arange(groups) * 3 + 7 + step, beams))
    new = (torch.zeros(groups, beams, device=DEV), torch.zeros(groups, beams, dtype=torch.int32, device=DEV),
           torch.zeros(groups, beams, dtype=torch.int32, device=DEV))
    err = err_word()
    ops.beam_advance(cand, i32(stops) if n_stop else None, i32(slots), *new, err, records=records, history=history,
                     positions=positions, prefix_len=prefix, begin=begin)
    want = advance_oracle((torch.from_numpy(scores), torch.from_numpy(parents), torch.from_numpy(tokens)), stops, beams, begin)
    for got, w in zip(new, want):
        assert got.tolist() == torch.tensor(w, dtype=got.dtype).tolist()
    want_records = np.full((max_slots, 8), -5)
    want_records[slots.reshape(-1), 7] = np.array(want[2]).reshape(-1)
    np.testing.assert_array_equal(records.cpu().numpy(), want_records)
    want_history = np.full((max_slots, 32), 99)
    if not begin:
        want_history[slots, step] = np.arange(beams)[None, :]
    np.testing.assert_array_equal(history.cpu().numpy(), want_history)
    assert err.tolist() == [0, 0, 0, 0]


def test_beams_that_go_on_refuse_and_report():
    cand = (torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    slots = i32([[0, 1], [2, 3]])
    new = lambda: (torch.zeros(2, 2, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV))
    err = err_word()
    history = torch.zeros(4, 8, dtype=torch.uint8, device=DEV)
    for bad in (lambda: ops.beam_advance(cand, None, slots[:1], *new(), err), lambda: ops.beam_advance(cand[:2] + (cand[0],), None, slots, *new(), err),
                lambda: ops.beam_advance(cand, None, slots, *new(), err, history=history),
                lambda: ops.beam_advance(cand, None, slots, *new(), err, records=torch.zeros(4, 7, dtype=torch.int32, device=DEV)),
                lambda: ops.beam_advance(cand, torch.zeros(1, dtype=torch.int64, device=DEV), slots, *new(), err)):
        with pytest.raises(KernelError):
            bad()
    # a slot outside the records, and a position outside the history
    ops.beam_advance(cand, None, i32([[0, 1], [2, 9]]), *new(), err, records=torch.zeros(4, 8, dtype=torch.int32, device=DEV))
    assert err.tolist()[0] == 4
    err.zero_()
    ops.beam_advance(cand, None, slots, *new(), err, history=history, positions=i32([20, 20, 20, 20]), prefix_len=i32([2, 15]))
    assert err.tolist()[0] == 3 and int(history[:2].sum()) == 0 and history[3, 5] == 1


# ------------------------------------------------------------------------------------------------ records

def reorder_oracle(t, slots, parents):
    new = t.clone()
    for row, frm in zip(slots.tolist(), parents.tolist()):
        for s, p in zip(row, frm):
            new[:, s] = t[:, row[p]]
    return new


RECORDS = {"state": (torch.float32, (3, 2, 5)), "tail": (torch.bfloat16, (3, 1365)), "token": (torch.int32, (1,)),
           "history": (torch.uint8, (1031,)), "one_byte": (torch.uint8, (1,)), "odd_pair": (torch.bfloat16, (1,)), "eight": (torch.float32, (6,)),
           "large": (torch.float32, (4, 64, 64)), "none": (torch.float32, (0,))}


@pytest.mark.parametrize("groups,seats", [(1, 1), (1, 2), (3, 4), (2, 7), (2, 16), (1, 33), (2, 64)])
@pytest.mark.parametrize("kind", ["identity", "shift", "random", "all_from_one"])
def test_records_follow(groups, seats, kind):
    rng = np.random.default_rng(11)
    max_slots = groups * seats + 5
    slots = rng.permutation(max_slots)[:groups * seats].reshape(groups, seats)
    parents = {"identity": np.tile(np.arange(seats), (groups, 1)), "shift": np.tile(np.roll(np.arange(seats), 1), (groups, 1)),
               "random": rng.integers(0, seats, (groups, seats)), "all_from_one": np.full((groups, seats), seats - 1)}[kind]
    gen = torch.Generator().manual_seed(0)
    tensors = []
    for dtype, shape in RECORDS.values():
        t = torch.randint(0, 255, (2, max_slots) + shape, generator=gen)
        tensors.append(t.to(dtype).to(DEV))
    want = [reorder_oracle(t.cpu(), slots, parents) for t in tensors]
    err = err_word()
    ops.reorder_slots(tensors, i32(slots), i32(parents), err)
    for name, got, w in zip(RECORDS, tensors, want):
        assert torch.equal(got.cpu(), w), name
    assert err.tolist()[0] == 0


@pytest.mark.parametrize("kind", ["identity", "shift", "random", "all_from_one", "in_two"])
@pytest.mark.parametrize("groups,seats,sizes", [(3, 8, [(2, 400004), (1, 4), (3, 3076)]), (1, 24, [(5, 700000)]), (60, 16, [(2, 20488), (1, 12)]),
                                                (200, 2, [(1, 16384)])])
def test_long_records_follow(groups, seats, sizes, kind):
    """Records of many bytes (sizes: keys, and floats of a record), among short ones."""
    rng = np.random.default_rng(13)
    max_slots = groups * seats + 3
    slots = rng.permutation(max_slots)[:groups * seats].reshape(groups, seats)
    parents = {"identity": np.tile(np.arange(seats), (groups, 1)), "shift": np.tile(np.roll(np.arange(seats), 1), (groups, 1)),
               "random": rng.integers(0, seats, (groups, seats)), "all_from_one": np.full((groups, seats), seats - 1),
               "in_two": np.where(rng.random((groups, 1)) < 0.5, np.arange(seats), np.arange(seats) // 2 * 2)}[kind]
    gen = torch.Generator(device=DEV).manual_seed(3)
    tensors = [torch.randn(keys, max_slots, n, device=DEV, generator=gen) for keys, n in sizes]
    at, source = torch.from_numpy(slots).to(DEV), torch.from_numpy(np.take_along_axis(slots, parents, axis=1)).to(DEV)
    want = []
    for t in tensors:
        w = t.clone()
        w[:, at.reshape(-1)] = t[:, source.reshape(-1)]
        want.append(w)
    err = err_word()
    ops.reorder_slots(tensors, i32(slots), i32(parents), err)
    assert all(torch.equal(a, b) for a, b in zip(tensors, want)) and err.tolist()[0] == 0
    # a seat with a slot or a parent that there is not stays as it is, and so does what would go on from it
    before = [t.clone() for t in tensors]
    bad_slots, bad_parents = slots.copy(), np.tile(np.arange(seats), (groups, 1))
    bad_slots[0, 0], bad_parents[0, 1], bad_parents[-1, 0] = max_slots, 0, seats
    ops.reorder_slots(tensors, i32(bad_slots), i32(bad_parents), err)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before)) and err.tolist()[0] == 4


def test_records_at_addresses_on_any_boundary_and_many_tensors():
    memory = torch.arange(0, 4096, dtype=torch.int32, device=DEV).to(torch.uint8)
    err = err_word()
    slots, parents = i32([[0, 2, 3]]), i32([[1, 0, 0]])
    for offset in (1, 2, 4, 8):
        t = memory[offset:offset + 4 * 48].view(1, 4, 48)
        before, want = memory.clone(), reorder_oracle(t.cpu(), slots.cpu(), parents.cpu())
        ops.reorder_slots([t], slots, parents, err)
        assert torch.equal(t.cpu(), want)
        assert torch.equal(memory[:offset], before[:offset]) and torch.equal(memory[offset + 192:], before[offset + 192:])
    many = [torch.randn(1, 4, 3 + i, device=DEV) for i in range(60)]
    want = [reorder_oracle(t.cpu(), slots.cpu(), parents.cpu()) for t in many]
    ops.reorder_slots(many, slots, parents, err)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(many, want)) and err.tolist()[0] == 0


def test_records_refuse_and_report():
    t, err = torch.arange(12.0, device=DEV).view(1, 4, 3), err_word()
    slots, parents = i32([[0, 1, 2]]), i32([[0, 0, 1]])
    for bad in (lambda: ops.reorder_slots([t.cpu()], slots, parents, err), lambda: ops.reorder_slots([t.transpose(1, 2)], slots, parents, err),
                lambda: ops.reorder_slots([t, torch.zeros(1, 5, 3, device=DEV)], slots, parents, err),
                lambda: ops.reorder_slots([t], slots, parents[:, :2], err), lambda: ops.reorder_slots([t], slots.long(), parents, err),
                lambda: ops.reorder_slots([t], i32([list(range(65))]), i32([[0] * 65]), err), lambda: ops.reorder_slots([t[0, 0]], slots, parents, err)):
        with pytest.raises(KernelError):
            bad()
    ops.reorder_slots([], slots, parents, err)
    ops.reorder_slots([t], slots[:0], parents[:0], err)
    assert t.flatten().tolist() == list(range(12)) and err.tolist()[0] == 0
    # a parent that is none and a slot that is none leave their seats as they are; the others move
    ops.reorder_slots([t], i32([[0, 1, 2]]), i32([[0, 5, 1]]), err)
    assert err.tolist()[0] == 4 and t[0, 1].tolist() == [3, 4, 5] and t[0, 2].tolist() == [3, 4, 5]
    err.zero_()
    ops.reorder_slots([t], i32([[0, 7, 3]]), i32([[0, 0, 0]]), err)
    assert err.tolist()[0] == 4 and t[0, 3].tolist() == [0, 1, 2]


# ------------------------------------------------------------------------------------------------ attention

class Shared:
    """Inputs of one call: groups of members with prefixes and own positions, pages in no order, everything that no
    request may see filled with NaN."""

    def __init__(self, members, prefixes, own, *, hq=4, hkv=2, d=64, dv=None, page=16, dtype=torch.bfloat16, history=False, seed=0,
                 window=None, softcap=None, sinks=False, common=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.dv, self.page, self.dtype = hq, hkv, d, dv or d, page, dtype
        self.members, self.prefixes = members, prefixes
        groups, rows = len(members), sum(members)
        self.rows = rows
        self.group_of = np.repeat(np.arange(groups), members)
        own = np.array(own).reshape(-1) if np.size(own) == rows else np.repeat(np.broadcast_to(own, groups), members)
        self.positions = np.array(prefixes)[self.group_of] + own - 1
        self.max_own = int(own.max())
        n_slots = groups + rows + 2
        slots = rng.permutation(n_slots)
        self.prefix_slot, self.slots = slots[:groups], slots[groups:groups + rows]
        max_pages = int(max(self.positions.max(), max(prefixes))) // page + 1
        need = sum(-(-p // page) for p in prefixes) + sum(int(self.positions[r]) // page - prefixes[g] // page + 1
                                                          for r, g in enumerate(self.group_of) if self.positions[r] >= prefixes[g])
        ids = iter(rng.permutation(need + 3).tolist())
        self.table = np.full((n_slots, max_pages), -1, dtype=np.int32)
        k = torch.full((need + 3, hkv, page, d), float("nan"))
        v = torch.full((need + 3, hkv, page, self.dv), float("nan"))

        def fill(slot, lo, hi):
            for i in range(lo // page, (hi - 1) // page + 1) if hi > lo else ():
                if self.table[slot, i] < 0:
                    self.table[slot, i] = next(ids)
            for t in range(lo, hi):
                at = self.table[slot, t // page]
                k[at, :, t % page] = torch.randn(hkv, d, generator=gen)
                v[at, :, t % page] = torch.randn(hkv, self.dv, generator=gen)

        for g, p in enumerate(prefixes):
            fill(self.prefix_slot[g], 0, p)
        for r, g in enumerate(self.group_of):
            fill(self.slots[r], prefixes[g], int(self.positions[r]) + 1)
        self.history = None
        if history:
            self.history = rng.integers(200, 256, (n_slots, self.max_own + 3)).astype(np.uint8)      # nobody's, where nothing was written
            for r, g in enumerate(self.group_of):
                start = int(np.cumsum([0] + list(members))[g])
                for t in range(int(own[r]) - 1):
                    if t < common:                       # the same writer for all members
                        self.history[self.slots[r], t] = (7 * t + 3) % members[g]
                        continue
                    able = [m for m in range(members[g]) if own[start + m] > t]
                    self.history[self.slots[r], t] = able[rng.integers(len(able))]
        self.k, self.v = k.to(dtype), v.to(dtype)
        self.q = (torch.randn(rows, hq, d, generator=gen) * 1.5).to(dtype)
        self.window, self.softcap = window, softcap
        self.sinks = torch.randn(hq, generator=gen) if sinks else None
        self.scale = d ** -0.5
        self.err = err_word()

    def shared(self, **kw):
        args = dict(max_members=max(self.members), max_prefix=max(self.prefixes), max_own=self.max_own,
                    history=None if self.history is None else torch.from_numpy(self.history).to(DEV))
        args.update(kw)
        return SharedPrefix(i32(np.cumsum([0] + list(self.members))), i32(self.prefix_slot), i32(self.prefixes), **args)

    def device(self):
        self.dq, self.dk, self.dv_ = self.q.to(DEV), self.k.to(DEV), self.v.to(DEV)
        self.out = torch.full((self.rows, self.hq, self.dv), float("nan"), dtype=self.dtype, device=DEV)
        self.args = (i32(self.positions), i32(self.slots), i32(self.table), self.err)
        self.kw = dict(scale=self.scale, window=self.window, softcap=self.softcap, sinks=None if self.sinks is None else self.sinks.to(DEV))
        return self

    def call(self, shared=None):
        ops.attention_shared(self.dq, self.out, self.dk, self.dv_, shared or self.shared(), *self.args, **self.kw)
        return self.out

    def oracle(self):
        """``(output, sum of p |v|, a bound on a score's rounding)`` in 64 bits, request by request."""
        outs, weights, rounding = [], [], 0.0
        starts = np.cumsum([0] + list(self.members))
        for r, g in enumerate(self.group_of):
            pos, p = int(self.positions[r]), self.prefixes[g]
            lo = max(0, pos - self.window + 1) if self.window else 0
            ks, vs = [], []
            for t in range(lo, pos + 1):
                slot = self.slots[r]
                if t < p:
                    slot = self.prefix_slot[g]
                elif self.history is not None and t < pos:
                    slot = self.slots[starts[g] + self.history[self.slots[r], t - p]]
                at = self.table[slot, t // self.page]
                ks.append(self.k[at, :, t % self.page]); vs.append(self.v[at, :, t % self.page])
            k, v = torch.stack(ks).double(), torch.stack(vs).double()                   # [keys, hkv, .]
            q = self.q[r].double().view(self.hkv, -1, self.d)
            s = torch.einsum("hpd,khd->hpk", q, k) * self.scale
            rounding = max(rounding, float(torch.einsum("hpd,khd->hpk", q.abs(), k.abs()).max()) * self.scale)
            if self.softcap:
                s = self.softcap * torch.tanh(s / self.softcap)
            if self.sinks is not None:
                s = torch.cat((s, self.sinks.double().view(self.hkv, -1, 1)), dim=-1)
            w = torch.softmax(s, dim=-1)[..., :len(ks)]
            outs.append(torch.einsum("hpk,khd->hpd", w, v).reshape(self.hq, self.dv))
            weights.append(torch.einsum("hpk,khd->hpd", w, v.abs()).reshape(self.hq, self.dv))
        return torch.stack(outs), torch.stack(weights), rounding

    def check(self, out=None):
        out = (self.out if out is None else out).cpu().double()
        want, weight, size = self.oracle()
        # a score: d products and as many additions of floats, a fast tanh of 1e-6 of the cap, 2^-22 of an exponential; twice,
        # for the numerator and the denominator
        score = (self.d + 4) * F32_HALF * size + 2.0 ** -22 + (1e-6 * self.softcap if self.softcap else 0.0)
        keys = int(self.positions.max()) + 1
        tol = (2 * score + keys ** 0.5 * F32_HALF * 4) * weight
        if self.dtype == torch.bfloat16:
            # probabilities in front of the second product and the output are rounded to bfloat16
            tol = tol + BF16_HALF * weight + BF16_HALF * (want.abs() + tol + BF16_HALF * weight)
        else:
            tol = tol + F32_HALF * want.abs()
        assert torch.isfinite(out).all()
        worst = ((out - want).abs() - tol).max()
        assert worst <= 0, f"off by {float((out - want).abs().max()):.3g}, {float(worst):.3g} beyond the bound"
        assert self.err.tolist() == [0, 0, 0, 0]


SHAPES = {
    "one": dict(members=[1], prefixes=[0], own=1),
    "one_key_shared": dict(members=[2], prefixes=[1], own=1),
    "no_prefix": dict(members=[3], prefixes=[0], own=40),
    "page_end": dict(members=[4], prefixes=[64], own=16),
    "mid_page": dict(members=[4, 4], prefixes=[61, 200], own=[5, 35]),
    "ragged": dict(members=[1, 5, 2], prefixes=[0, 130, 33], own=[9, 1, 2, 3, 70, 17, 64, 65]),
    "tile": dict(members=[9], prefixes=[129], own=33),
    "many": dict(members=[40, 3], prefixes=[300, 70], own=20),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_shared_attention(shape, history, dtype):
    c = Shared(**SHAPES[shape], dtype=dtype, history=history).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,dv,page", [(8, 1, 128, 128, 16), (5, 1, 64, 64, 32), (4, 4, 128, 128, 64), (16, 1, 128, 128, 128), (6, 2, 16, 16, 8),
                                              (6, 1, 32, 32, 8), (4, 2, 30, 18, 5), (2, 1, 256, 256, 16), (2, 2, 6, 250, 1),
                                              (33, 1, 64, 64, 16), (4, 2, 128, 64, 16), (10, 2, 128, 128, 24)])
def test_shared_attention_sizes(hq, hkv, d, dv, page, dtype):
    c = Shared([3, 6], [70, 145], 37, hq=hq, hkv=hkv, d=d, dv=dv, page=page, dtype=dtype, history=True, seed=2).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 32)])
@pytest.mark.parametrize("window", [1, 20, 37, 64, 100, 5000])
def test_shared_attention_windows(window, dtype, d):
    """Windows that end in the own positions, at their first, and inside the shared ones; requests of several lengths."""
    c = Shared([4, 2], [150, 40], [37, 37, 30, 2, 50, 1], window=window, dtype=dtype, d=d, seed=4, softcap=20.0, sinks=True).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_attention_options(dtype):
    for kw in (dict(softcap=5.0), dict(sinks=True), dict(softcap=30.0, sinks=True)):
        c = Shared([5], [100], 30, dtype=dtype, history=True, d=128, seed=6, **kw).device()
        c.call()
        c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_attention_long(dtype):
    c = Shared([6], [1500], 300, hq=8, hkv=1, d=128, dtype=dtype, history=True, seed=7).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("members", [[8], [9], [16, 3], [20, 17, 1], [33]])
def test_shared_attention_of_many_query_heads(members, dtype, d):
    """More (query head, member) pairs over a key head than a tile of rows, or two, hold."""
    c = Shared(members, [150, 70, 200][:len(members)], 21, hq=16, hkv=1, d=d, dtype=dtype, history=True, seed=14).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype,d,hq", [(torch.float32, 64, 4), (torch.bfloat16, 64, 4), (torch.bfloat16, 128, 4), (torch.bfloat16, 128, 32)])
@pytest.mark.parametrize("members,prefixes,own,common,window", [
    ([4], [100], 60, 59, None), ([4], [100], 60, 58, None), ([8, 3], [64, 130], 200, 150, None), ([5], [0], 90, 80, None), ([2], [1], 66, 64, None),
    ([6], [200], 300, 290, 64), ([6], [200], 300, 290, 310), ([6], [200], 150, 140, 152), ([20], [300], 129, 127, None), ([4, 4], [33, 70], 2, 1, None),
    ([3], [150], [140, 90, 120], 89, None)])
def test_shared_attention_of_beams_with_a_common_past(members, prefixes, own, common, window, dtype, d, hq):
    c = Shared(members, prefixes, own, hq=hq, hkv=2, d=d, dtype=dtype, history=True, common=common, window=window, seed=15).device()
    c.call()
    c.check()


@pytest.mark.parametrize("d,hq,members,own", [(128, 16, [12], 400), (64, 16, [16, 2], 200), (128, 16, [40], [70 * (i % 5) + 1 for i in range(40)]),
                                              (128, 2, [70], 40), (64, 32, [9], [1, 700, 1, 1, 65, 64, 63, 300, 2]), (128, 8, [3], 900)])
def test_shared_attention_of_single_members_keys(d, hq, members, own):
    c = Shared(members, [150, 90][:len(members)], own, hq=hq, hkv=1, d=d, dtype=torch.bfloat16, seed=17).device()
    c.call()
    c.check()


def test_shared_attention_of_very_many_small_groups():
    """More pieces than a block lists at a time."""
    n = 1700
    c = Shared([1] * n, [5 + i % 3 for i in range(n)], [1 + i % 4 for i in range(n)], hq=4, hkv=4, d=64, dtype=torch.bfloat16, seed=16).device()
    c.call()
    c.check()


@pytest.mark.parametrize("d,hkv", [(64, 2), (128, 2), (128, 8)])
def test_shared_attention_of_groups_of_all_sizes(d, hkv):
    """One tile of query rows and two, long sequences of keys and single tiles in turn."""
    members, prefixes = [40, 1, 70, 3, 33, 2, 64, 1, 5], [700, 3, 310, 64, 129, 1, 500, 65, 260]
    x = Shared(members, prefixes, own=24, hq=4 * hkv, hkv=hkv, d=d, history=True, common=20, seed=9).device()
    first = x.call().clone()
    x.check(first)
    cold = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    for i in range(12):
        cold.fill_(i)
        assert torch.equal(x.call(), first), f"call {i}"


@pytest.mark.parametrize("d", [64, 128])
def test_shared_attention_of_keys_that_come_late(d):
    """Long sequences of key tiles in every block, read from memory that no cache holds: what a tile waits for arrives late."""
    x = Shared([2] * 12, [1180 + 49 * i for i in range(12)], own=40, hq=16, hkv=8, d=d, history=True, common=30, seed=5).device()
    first = x.call().clone()
    x.check(first)
    cold = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    for i in range(24):
        cold.fill_(i)
        x.out.fill_(float("nan"))
        assert torch.equal(x.call(), first), f"call {i}"
    x.check()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("prefixes,window", [([70, 0], None), ([0, 0], None), ([300, 33], 700)])
def test_shared_attention_of_long_own_positions(prefixes, window, dtype, d):
    """Few rows with many positions of their own, which several blocks share out."""
    c = Shared([2, 1], prefixes, [900, 530, 257], hq=8, hkv=2, d=d, dtype=dtype, window=window, sinks=True, seed=21).device()
    c.call()
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("history", [False, True])
def test_shared_attention_of_groups_without_members(history, dtype):
    c = Shared([0, 2, 0, 0, 3, 0], [40, 70, 0, 130, 200, 65], 30, d=64, dtype=dtype, history=history, seed=22).device()
    c.call()
    c.check()


def test_shared_attention_at_addresses_on_any_boundary():
    for dtype in (torch.float32, torch.bfloat16):
        c = Shared([3], [70], 20, d=64, dtype=dtype, seed=13).device()
        def moved(t):
            memory = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
            memory[1:] = t.reshape(-1)
            return memory[1:].view(t.shape)
        c.dq, c.dk, c.dv_, c.out = (moved(t) for t in (c.dq, c.dk, c.dv_, c.out))
        c.call()
        c.check()


def test_shared_attention_queries_inside_the_prefix():
    """A row whose position lies inside the shared ones sees those up to its own."""
    c = Shared([3], [90], 1, d=64, seed=8).device()
    pos = np.array([89, 40, 0])
    ops.attention_shared(c.dq, c.out, c.dk, c.dv_, c.shared(), i32(pos), *c.args[1:], **c.kw)
    c.positions = pos
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_attention_twice_gives_the_same_bits_and_leaves_the_rest(dtype):
    c = Shared([4, 7], [333, 20], 90, dtype=dtype, d=128, history=True, seed=9).device()
    first = c.call().clone()
    for _ in range(3):
        c.out.fill_(float("nan"))
        assert torch.equal(c.call(), first)
    # the rows of a larger buffer behind the last request stay as they are
    big = torch.full((c.rows + 4, c.hq, c.dv), 7.0, dtype=dtype, device=DEV)
    ops.attention_shared(c.dq, big[:c.rows], c.dk, c.dv_, c.shared(), *c.args, **c.kw)
    assert torch.equal(big[:c.rows], first) and bool((big[c.rows:] == 7.0).all())


def test_shared_attention_captured_and_on_two_streams():
    cs = [Shared([4], [200 + 40 * i], 50, d=128, history=True, seed=10 + i).device() for i in range(2)]
    for c in cs:
        c.call()
    graphs, shareds = [], [c.shared() for c in cs]
    torch.cuda.synchronize()
    for c, sh in zip(cs, shareds):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.call(sh)
        graphs.append(g)
        c.out.fill_(float("nan"))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for c in cs:
        c.check()
    # shorter prefixes and positions than those that the capture was planned for
    c, sh = cs[1], shareds[1]
    sh.prefix_len.fill_(100)
    c.args[0].fill_(99)
    graphs[1].replay()
    torch.cuda.synchronize()
    c.prefixes, c.positions = [100], np.full(4, 99)
    c.check()


def test_shared_attention_refuses():
    c = Shared([3], [40], 5, d=64).device()
    call = lambda q=None, out=None, k=None, v=None, shared=None, args=None, **kw: ops.attention_shared(
        c.dq if q is None else q, c.out if out is None else out, c.dk if k is None else k, c.dv_ if v is None else v,
        shared or c.shared(), *(args or c.args), **{**c.kw, **kw})
    sh = c.shared()
    bad_starts = SharedPrefix(sh.group_start[:1], sh.prefix_slot, sh.prefix_len, 3, 40, 5)
    for bad in (lambda: call(q=c.dq.float()), lambda: call(q=c.dq.cpu()), lambda: call(out=c.out[:, :, :32]), lambda: call(k=c.dk.transpose(0, 1)),
                lambda: call(q=c.dq.half(), out=c.out.half(), k=c.dk.half(), v=c.dv_.half()),
                lambda: call(q=c.dq[:, :3].contiguous(), out=c.out[:, :3].contiguous()), lambda: call(shared=bad_starts), lambda: call(window=0),
                lambda: call(sinks=torch.zeros(3, device=DEV)), lambda: call(args=(c.args[0][:2],) + c.args[1:]),
                lambda: call(args=(c.args[0].long(),) + c.args[1:]), lambda: call(shared=c.shared(max_members=0)), lambda: call(shared=c.shared(max_own=0)),
                lambda: call(shared=c.shared(history=torch.zeros(2, 5, dtype=torch.uint8, device=DEV))),
                lambda: call(shared=c.shared(history=torch.zeros(c.table.shape[0], 5, dtype=torch.int32, device=DEV)))):
        with pytest.raises(KernelError):
            bad()
    assert bool(torch.isnan(c.out).all())


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 32)])
def test_shared_attention_reports(dtype, d):
    """Faults in what the device reads are reported and followed nowhere."""
    c = Shared([3, 2], [40, 50], 20, dtype=dtype, d=d, history=True, seed=12).device()

    def code(shared=None, positions=None, slots=None, table=None):
        c.err.zero_()
        ops.attention_shared(c.dq, c.out, c.dk, c.dv_, shared or c.shared(), i32(c.positions if positions is None else positions),
                             i32(c.slots if slots is None else slots), i32(c.table if table is None else table), c.err, **c.kw)
        return c.err.tolist()[0]

    assert code() == 0
    table = c.table.copy(); table[c.prefix_slot[0], 1] = -1
    assert code(table=table) == 2
    table = c.table.copy(); table[c.slots[1], 50 // c.page] = 10 ** 6
    assert code(table=table) == 2
    assert code(positions=[59, -1, 59, 69, 69]) == 3
    assert code(positions=[59, 59, 59, 69, 10 ** 6]) in (2, 3)
    slots = c.slots.copy(); slots[4] = c.table.shape[0]
    assert code(slots=slots) == 4
    sh = c.shared(); sh.prefix_slot[1] = -3
    assert code(shared=sh) == 4
    sh = c.shared(); sh.history[c.slots[0], 3] = 200
    assert code(shared=sh) == 4
    assert code(shared=c.shared(max_members=2)) == 4           # a group with more members than the call was planned for
    assert code(shared=c.shared(max_prefix=0)) == 4
    assert code() == 0
    c.check()
