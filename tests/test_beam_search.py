"""Search over beams, what needs no device: parameters, the host's bookkeeping, forked requests in the cache manager."""

from __future__ import annotations

import math
import random
import types

import pytest

from tokamak_b200 import BeamSearchParams
from tokamak_b200.cache.manager import CacheManager, KVGroup, KVPagesNeed, OutOfSlotsError, StateGroup, StateNeed
from tokamak_b200.cli import build_parser


def test_parameters_are_checked():
    for bad in (dict(beam_width=0), dict(beam_width=33), dict(max_new_tokens=0), dict(length_penalty=-1.0), dict(length_penalty=math.nan)):
        with pytest.raises(ValueError):
            BeamSearchParams(**bad)
    p = BeamSearchParams()
    assert (p.beam_width, p.max_new_tokens, p.length_penalty, p.early_stopping, p.ignore_eos) == (4, 128, 1.0, False, False)


def test_command_line_options():
    args = build_parser().parse_args(["--model", "m", "--beam-width", "5", "--length-penalty", "0.6"])
    assert args.beam_width == 5 and args.length_penalty == 0.6 and build_parser().parse_args(["--model", "m"]).beam_width == 0


def manager(pages=12, page=4, slots=6, window=None):
    return CacheManager([KVGroup(KVPagesNeed(1, 8, window), pages, page, ["a"])], [StateGroup(StateNeed((2,)), ["s"])], slots)


@pytest.mark.parametrize("length", [1, 4, 7, 8])
def test_a_forked_request_holds_pages_behind_its_parents_positions_only(length):
    m = manager()
    m.admit("p"); m.grow("p", length); m.advance("p", length)
    m.fresh_slots.clear()
    held = set(m.kv_groups[0].held_pages("p"))
    slots = [m.fork("p", i) for i in range(3)]
    assert len(set(slots)) == 3 and not m.fresh_slots and all(m.length(i) == length for i in range(3))
    assert all(m.kv_groups[0].held_pages(i) == [] for i in range(3))
    m.table_writes.clear()
    for i in range(3):
        m.grow(i, length + 5)
        own = m.kv_groups[0].held_pages(i)
        # its pages begin with the one that its first position falls into, and cover the last
        assert len(own) == (length + 4) // 4 - length // 4 + 1 and not held & set(own)
        held |= set(own)
        m.advance(i, 5)
    assert sorted({w[2] for w in m.table_writes}) == list(range(length // 4, (length + 4) // 4 + 1))
    m.check_invariants()
    for i in range(3):
        m.free(i)
    m.free("p")
    m.check_invariants()
    assert m.kv_groups[0].num_free == 12 and m.num_free_slots == 6


def test_forks_that_cannot_be():
    m = manager(slots=2)
    with pytest.raises(KeyError):
        m.fork("p", 0)
    m.admit("p"); m.grow("p", 6); m.advance("p", 6)
    m.fork("p", 0)
    with pytest.raises(ValueError):
        m.fork("p", 0)
    with pytest.raises(OutOfSlotsError):
        m.fork("p", 1)
    m.check_invariants()


def test_a_window_gives_the_pages_of_forked_requests_back():
    m = manager(pages=12, window=5)
    m.admit("p"); m.grow("p", 6); m.advance("p", 6)
    m.fork("p", 0)
    for n in range(7, 20):
        m.grow(0, n); m.advance(0, 1)
        m.check_invariants()
    assert len(m.kv_groups[0].held_pages(0)) <= 3
    m.free(0); m.free("p")
    assert m.kv_groups[0].num_free == 12


def test_the_hosts_side_of_a_search():
    from tokamak_b200.engine.beam import Search
    params = BeamSearchParams(beam_width=2, max_new_tokens=9, length_penalty=1.0)
    s = Search(0, [1, 2], 9)
    stops = frozenset({7})
    s.take(params, stops, [(-1.0, 0, 4), (-1.5, 0, 7), (-2.0, 0, 5), (-3.0, 0, 6)], [(-1.0, 0, 4), (-2.0, 1, 5)])
    assert s.tokens == [[4], [5]] and [(h.tokens, h.sum_logprobs, h.ended) for h in s.ended] == [([7], -1.5, True)] and not s.done
    # both go on from seat 0: seat 1's beam ends here; the stop token behind the last beam that goes on counts for nothing
    s.take(params, stops, [(-1.2, 0, 3), (-1.4, 0, 8), (-1.5, 1, 7), (-9.0, 1, 1)], [(-1.2, 0, 3), (-1.4, 0, 8)])
    assert s.tokens == [[4, 3], [4, 8]] and len(s.ended) == 1 and not s.done
    s.take(params, stops, [(-1.3, 1, 7), (-6.0, 0, 2), (-6.5, 1, 2), (-7.0, 0, 1)], [(-6.0, 0, 2), (-6.5, 1, 2)])
    # two ended ones (-1.5 for one token, -1.3 for three), and no running beam better than the worse of them
    assert [h.tokens for h in s.ended] == [[4, 8, 7], [7]] and s.done
    found = s.hypotheses(params)
    assert [h.tokens for h in found] == [[4, 8, 7], [7]] and math.isclose(found[0].score(1.0), -1.3 / 3)
    # a search whose every beam is dead is over; one at its cap returns running beams
    d = Search(1, [1], 9)
    d.take(params, stops, [(-1.0, 0, 7), (-math.inf, 0, 0)], [(-math.inf, 0, 0), (-math.inf, 1, 0)])
    assert d.done and [h.tokens for h in d.hypotheses(params)] == [[7]]
    c = Search(2, [1], 1)
    c.take(params, frozenset(), [(-1.0, 0, 4), (-2.0, 0, 5)], [(-1.0, 0, 4), (-2.0, 1, 5)])
    assert c.done and [(h.tokens, h.ended) for h in c.hypotheses(params)] == [([4], False), ([5], False)]


def test_models_whose_attention_cannot_read_shared_keys_are_refused():
    from tokamak_b200.engine.beam import refuses_search
    block = lambda mixer, need: types.SimpleNamespace(mixer=mixer, cache_need=lambda: need)
    knows, other = types.SimpleNamespace(SHARED_PREFIX=True), types.SimpleNamespace()
    model = lambda **blocks: types.SimpleNamespace(blocks=blocks)
    assert refuses_search(model(a=block(knows, KVPagesNeed(1, 8)), b=block(other, StateNeed((3,))))) is None
    assert "'b'" in refuses_search(model(a=block(knows, KVPagesNeed(1, 8)), b=block(other, KVPagesNeed(1, 8))))
    assert refuses_search(model(a=block(other, {"mixer": {"pages": KVPagesNeed(1, 8)}}))) is not None


def test_segments_of_rows_of_logits():
    """Within what the kernels hold, and on the kernel with registers for three blocks an SM wherever that costs least."""
    from tokamak_b200.csrc import ops
    sms = 148
    for rows, beams, vocab, k in [(1, 1, 151936, 8), (1, 1, 1, 1), (32, 4, 151936, 8), (16, 4, 151936, 8), (24, 4, 151936, 8), (64, 64, 4096, 256),
                                  (512, 16, 100003, 32), (65535, 1, 5, 5), (8, 8, 2 ** 21, 64)]:
        n = ops.beam_segments(sms, rows, beams, vocab, k)
        assert 1 <= n <= max(1, -(-vocab // 3584)) and beams * n * k <= max(16384, beams * k)
    # 416 blocks of four tiles, three an SM, cost less than 480 of three, four an SM
    assert ops.beam_segments(sms, 32, 4, 151936, 8) == 13
    assert ops.beam_segments(sms, 512, 16, 100003, 32) == 1


def test_the_host_keeps_a_tree_of_tokens():
    """A step adds a node for every beam and copies none of what the beams have behind them."""
    from tokamak_b200.engine.beam import Search
    params, width, steps = BeamSearchParams(beam_width=4, max_new_tokens=4000), 4, 3000
    s, want = Search(0, [1], 4000), [[] for _ in range(width)]
    rng = random.Random(3)
    for n in range(steps):
        parents = [rng.randrange(width) if n else 0 for _ in range(width)]
        seats = [(-0.1 * n - 0.01 * i, p, 10 * n + i) for i, p in enumerate(parents)]
        before = s.heads
        s.take(params, frozenset(), seats, seats)
        if n:
            assert all(head[0] is before[p] for head, p in zip(s.heads, parents))
        want = [want[p] + [10 * n + i] for i, p in enumerate(parents)]
    assert s.tokens == want and s.length == steps
    assert [h.tokens for h in s.hypotheses(params)] == want
