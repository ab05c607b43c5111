"""``LLM.beam_search`` against a plain search in 64 bits over whole sequences."""

from __future__ import annotations

import functools
import json
import math
import tempfile
from pathlib import Path

import pytest
import torch

import ketalix_configs as kc
import tiny_configs
from helpers import random_tokens
from plain import beam_plain, ketalix_plain, qwen3_plain

pytestmark = pytest.mark.gpu

_TMP = []
QWEN = {tag: tiny_configs.ALL[tag] for tag in ("A", "B", "C", "D", "W")}


@functools.lru_cache(maxsize=None)
def folder_of(tag: str, dtype: str, eos: tuple = ()) -> Path:
    from tokamak_b200.weights import write_random_model
    raw, init, _ = QWEN[tag] if tag in QWEN else kc.ALL[tag]
    tmp = tempfile.TemporaryDirectory(prefix=f"tk_beam_{tag}_{dtype}_")
    _TMP.append(tmp)
    write_random_model(tmp.name, raw, dtype=dtype, **init)
    if eos:
        path = Path(tmp.name) / "config.json"
        path.write_text(json.dumps({**json.loads(path.read_text()), "eos_token_id": list(eos)}))
    return Path(tmp.name)


@functools.lru_cache(maxsize=None)
def _loaded(folder: str, tag: str):
    return (qwen3_plain if tag in QWEN else ketalix_plain).load_folder(folder)


@functools.lru_cache(maxsize=None)
def _last_logits(folder: str, tag: str, tokens: tuple) -> torch.Tensor:
    cfg, w = _loaded(folder, tag)
    if tag in QWEN:
        return qwen3_plain.forward_logits(cfg, w, list(tokens), torch.float64)[-1]
    return ketalix_plain.forward_logits(cfg, w, list(tokens))[-1].double()


def plain_search(tag, dtype, prompt, **kw):
    folder = str(folder_of(tag, dtype))
    return beam_plain.search(lambda t: _last_logits(folder, tag, tuple(t)), prompt, **kw)


def vocab_of(tag):
    raw = (QWEN[tag] if tag in QWEN else kc.ALL[tag])[0]
    return raw.get("vocab_size", raw.get("vocab"))


def page_of(tag):
    return (QWEN[tag] if tag in QWEN else kc.ALL[tag])[2]


def prompts_of(tag, lengths):
    return [random_tokens(vocab_of(tag), n, seed=31 * n + 5) for n in lengths]


# (model, prompt lengths, width, tokens, EOS tokens, length penalty, early stopping)
CASES = [("A", (5, 17, 33), 3, 8, (), 1.0, False), ("B", (1, 20), 4, 9, (), 0.0, False), ("B", (7, 31), 2, 12, (142, 203), 1.0, False),
         ("C", (16, 40), 4, 20, (), 1.0, False), ("D", (3, 70), 3, 12, (), 1.0, False), ("W", (30, 9), 3, 30, (), 1.0, False),
         ("C", (33,), 5, 10, (1, 2, 3, 71, 100, 101, 168), 2.0, True), ("A", (17,), 3, 8, (240,), 0.0, False)]


def llm_for(tag, dtype, width, groups, eos=(), **kw):
    from tokamak_b200 import LLM
    if tag not in QWEN:
        kw.setdefault("max_seq_len", 512)
    return LLM(folder_of(tag, dtype, eos), dtype=dtype, block_size=page_of(tag), max_batch_size=groups * (width + 1),
               kv_pool_tokens=8192, **kw)


@pytest.mark.parametrize("tag,lengths,width,tokens,eos,penalty,early", CASES)
def test_searches_match_the_plain_one(tag, lengths, width, tokens, eos, penalty, early):
    from tokamak_b200 import BeamSearchParams
    prompts = prompts_of(tag, lengths)
    llm = llm_for(tag, "float32", width, len(prompts), eos)
    params = BeamSearchParams(beam_width=width, max_new_tokens=tokens, length_penalty=penalty, early_stopping=early)
    outs = llm.beam_search(prompt_token_ids=prompts, params=params)
    for prompt, out in zip(prompts, outs):
        want, _ = plain_search(tag, "float32", prompt, width=width, max_new=tokens, stops=eos, length_penalty=penalty, early_stopping=early)
        assert out.prompt_token_ids == prompt and [h.output_token_ids for h in out.hypotheses] == [t for t, _, _ in want]
        for h, (t, total, ended) in zip(out.hypotheses, want):
            # logits of the float32 path are off by up to 2e-4 (1 + |x|) (tests/helpers.py); a token's log probability by twice that
            assert abs(h.cumulative_logprob - total) <= len(t) * 2 * 2e-4 * 2
            assert h.finish_reason.value == ("stop" if ended else "length")
            assert math.isclose(h.score, h.cumulative_logprob / len(t) ** penalty)
    llm.cache_manager.check_invariants()
    assert all(g.num_free == g.num_pages for g in llm.cache_manager.kv_groups)
    # again, step by step from the host, without graphs, and with prompts in small portions
    llm.plain_steps = True
    again = llm.beam_search(prompt_token_ids=prompts, params=params)
    assert [[h.output_token_ids for h in o.hypotheses] for o in again] == [[h.output_token_ids for h in o.hypotheses] for o in outs]


@pytest.mark.parametrize("tag,dtype", [("C", "bfloat16"), ("D", "bfloat16"), ("W", "bfloat16")])
def test_searches_in_bfloat16_return_what_they_say(tag, dtype):
    """Rounding may flip a near tie, so every hypothesis is held against the plain log probabilities of its own tokens."""
    from tokamak_b200 import BeamSearchParams
    prompts = prompts_of(tag, (20, 45))
    llm = llm_for(tag, dtype, 4, 2)
    outs = llm.beam_search(prompt_token_ids=prompts, params=BeamSearchParams(beam_width=4, max_new_tokens=12))
    folder = str(folder_of(tag, dtype))
    for prompt, out in zip(prompts, outs):
        assert len({tuple(h.output_token_ids) for h in out.hypotheses}) == 4
        for h in out.hypotheses:
            total, slack = 0.0, 0.0
            for i, token in enumerate(h.output_token_ids):
                logits = _last_logits(folder, tag, tuple(prompt + h.output_token_ids[:i]))
                total += float(torch.log_softmax(logits, -1)[token])
                slack += 2 * 0.1 * float(logits.std())          # a bfloat16 logit is off by up to 0.1 of its row's spread (tests/helpers.py)
            assert abs(h.cumulative_logprob - total) <= slack
        assert [h.score for h in out.hypotheses] == sorted((h.score for h in out.hypotheses), reverse=True)


@pytest.mark.parametrize("tag", [t for t in kc.ALL][:2])
def test_searches_over_recurrent_layers(tag):
    """The recurrent states follow their beams (windowed attention with caps and sinks beside them)."""
    from tokamak_b200 import BeamSearchParams
    prompts = prompts_of(tag, (6, 21))
    llm = llm_for(tag, "float32", 3, 2)
    outs = llm.beam_search(prompt_token_ids=prompts, params=BeamSearchParams(beam_width=3, max_new_tokens=10))
    for prompt, out in zip(prompts, outs):
        want, _ = plain_search(tag, "float32", prompt, width=3, max_new=10)
        assert [h.output_token_ids for h in out.hypotheses] == [t for t, _, _ in want]


def test_searches_run_in_waves_and_leave_nothing_behind():
    from tokamak_b200 import BeamSearchParams, SamplingParams
    prompts = prompts_of("C", (16, 40, 9, 27, 16))
    params = BeamSearchParams(beam_width=3, max_new_tokens=14)
    wide, narrow = llm_for("C", "float32", 3, 5), llm_for("C", "float32", 3, 2, max_num_batched_tokens=16)
    want = [[h.output_token_ids for h in o.hypotheses] for o in wide.beam_search(prompt_token_ids=prompts, params=params)]
    assert wide.last_stats["waves"] == 1 and wide.last_stats["graph_replays"] > 0
    greedy = narrow.generate(prompt_token_ids=prompts[:2], sampling_params=SamplingParams(temperature=0.0, max_new_tokens=6))
    for _ in range(2):
        narrow.core.cache.poison_free_pages()
        got = [[h.output_token_ids for h in o.hypotheses] for o in narrow.beam_search(prompt_token_ids=prompts, params=params)]
        assert got == want and narrow.last_stats["waves"] == 3
    assert all(g.num_free == g.num_pages for g in narrow.cache_manager.kv_groups)
    # generation before and after a search gives the same tokens; a width of one is greedy generation
    again = narrow.generate(prompt_token_ids=prompts[:2], sampling_params=SamplingParams(temperature=0.0, max_new_tokens=6))
    assert [o.output_token_ids for o in again] == [o.output_token_ids for o in greedy]
    one = narrow.beam_search(prompt_token_ids=prompts[:2], params=BeamSearchParams(beam_width=1, max_new_tokens=6))
    assert [o.hypotheses[0].output_token_ids for o in one] == [o.output_token_ids for o in greedy]


def test_searches_that_are_refused():
    from tokamak_b200 import BeamSearchParams
    llm = llm_for("C", "float32", 3, 1)
    p = [[1, 2, 3]]
    with pytest.raises(ValueError, match="max_batch_size"):
        llm.beam_search(prompt_token_ids=p, params=BeamSearchParams(beam_width=4))
    with pytest.raises(ValueError, match="exactly one"):
        llm.beam_search(params=BeamSearchParams(beam_width=3))
    with pytest.raises(ValueError, match="vocabulary"):
        llm.beam_search(prompt_token_ids=[[10 ** 6]], params=BeamSearchParams(beam_width=3))
    with pytest.raises(ValueError):
        llm.beam_search(prompt_token_ids=[[]], params=BeamSearchParams(beam_width=3))
    assert llm.beam_search(prompt_token_ids=[], params=BeamSearchParams(beam_width=3)) == []
    small = llm_for("C", "float32", 3, 1, max_seq_len=256)
    small.cache_manager.kv_groups[0].allocator.num_pages = 20          # what the pool says it holds
    with pytest.raises(ValueError, match="kv_pool_tokens"):
        small.beam_search(prompt_token_ids=[[1] * 100], params=BeamSearchParams(beam_width=3, max_new_tokens=100))


def test_sums_are_carried_in_64_bits(monkeypatch):
    """What a step starts from is, to 2e-13, what the one before it returned plus a log probability in 64 bits, and so is what is reported."""
    from tokamak_b200 import BeamSearchParams
    from tokamak_b200.engine import beam
    prompt, width, tokens = prompts_of("C", (40,))[0], 3, 60
    llm = llm_for("C", "float32", width, 1)
    llm.plain_steps = True
    calls, select = [], beam.ops.beam_select

    def recorded(logits, scores, candidates, **kw):
        before = scores.clone()
        out = select(logits, scores, candidates, **kw)
        calls.append((logits.clone(), before, tuple(t.clone() for t in out)))
        return out

    monkeypatch.setattr(beam.ops, "beam_select", recorded)
    found = llm.beam_search(prompt_token_ids=[prompt], params=BeamSearchParams(beam_width=width, max_new_tokens=tokens, ignore_eos=True))[0].hypotheses
    assert len(calls) == tokens
    for i, (logits, before, (scores, parents, chosen)) in enumerate(calls):
        logp = torch.log_softmax(logits.double(), -1)
        want = before.double()[0, parents[0].long()] + logp[parents[0].long(), chosen[0].long()]
        assert float((scores[0].double() - want).abs().max()) <= 2e-13 + 2.0 ** -51 * float(want.abs().max())
        if i > 0:
            assert set(before[0].tolist()) <= set(calls[i - 1][2][0][0].tolist())
    assert [h.cumulative_logprob for h in found] == calls[-1][2][0][0][:width].tolist()


def run_order(monkeypatch):
    """What a search launches and reads, in order: ``"launch"`` and ``"collect"``, with the beams' tokens at each launch."""
    from tokamak_b200.engine.beam import BeamRunner
    order, launch, collect = [], BeamRunner.launch, BeamRunner.collect

    def launched(self, searches, done):
        order.append(("launch", [list(t) for s in searches for t in s.tokens]))
        return launch(self, searches, done)

    def collected(self, pending):
        order.append(("collect", None))
        return collect(self, pending)

    monkeypatch.setattr(BeamRunner, "launch", launched)
    monkeypatch.setattr(BeamRunner, "collect", collected)
    return order


@pytest.mark.parametrize("tag,dtype", [("C", "float32"), ("D", "bfloat16")])
def test_plain_steps_of_a_search(tag, dtype, monkeypatch):
    """With ``plain_steps`` a step is launched once the one before it has been read; the tokens do not depend on it, nor on how the
    prompts are cut."""
    from tokamak_b200 import BeamSearchParams
    prompts, params = prompts_of(tag, (33, 50)), BeamSearchParams(beam_width=3, max_new_tokens=16, ignore_eos=True)
    order = run_order(monkeypatch)
    llm = llm_for(tag, dtype, 3, 2)
    ahead = llm.beam_search(prompt_token_ids=prompts, params=params)
    assert llm.last_stats["graph_replays"] > 0
    kinds = [k for k, _ in order]
    assert any(a == b == "launch" for a, b in zip(kinds, kinds[1:]))
    order.clear()
    llm.plain_steps = True
    plain = llm.beam_search(prompt_token_ids=prompts, params=params)
    kinds = [k for k, _ in order]
    assert kinds[0] == "collect" and kinds[1:] == ["launch", "collect"] * 15 and llm.last_stats["graph_replays"] == 0
    assert [[h.output_token_ids for h in o.hypotheses] for o in plain] == [[h.output_token_ids for h in o.hypotheses] for o in ahead]
    if dtype == "float32":                      # (in bfloat16 other portions may round otherwise)
        cut = llm_for(tag, dtype, 3, 2, max_num_batched_tokens=16)
        cut.plain_steps = True
        small = cut.beam_search(prompt_token_ids=prompts, params=params)
        assert cut.last_stats["steps"] > llm.last_stats["steps"]
        assert [[h.output_token_ids for h in o.hypotheses] for o in small] == [[h.output_token_ids for h in o.hypotheses] for o in ahead]


@pytest.mark.parametrize("tag", ["C", "D"])
def test_searches_that_grow_into_the_next_bucket(tag):
    """Positions pass 256 in the middle of a search: the step is planned, and captured, anew."""
    from tokamak_b200 import BeamSearchParams
    prompts, params = prompts_of(tag, (247, 236)), BeamSearchParams(beam_width=3, max_new_tokens=40, ignore_eos=True)
    for dtype in ("float32", "bfloat16"):
        llm = llm_for(tag, dtype, 3, 2)
        first = llm.beam_search(prompt_token_ids=prompts, params=params)
        graphs = llm._beam_runner.graphs
        assert len({key[1] for key in graphs}) == 2 and llm.last_stats["graph_replays"] >= 30
        again = llm.beam_search(prompt_token_ids=prompts, params=params)
        llm.plain_steps = True
        plain = llm.beam_search(prompt_token_ids=prompts, params=params)
        for o in (again, plain):
            assert [[(h.output_token_ids, h.cumulative_logprob) for h in x.hypotheses] for x in o] == \
                   [[(h.output_token_ids, h.cumulative_logprob) for h in x.hypotheses] for x in first]


@pytest.mark.parametrize("tag", ["C", "D", "W"])
def test_every_beams_logits_in_bfloat16(tag, monkeypatch):
    """Step by step and beam by beam against the plain model on the beam's own tokens: a key of another beam's past would show."""
    from helpers import assert_logits_close
    from tokamak_b200 import BeamSearchParams
    from tokamak_b200.engine import beam
    prompts, width = prompts_of(tag, (20, 45)), 4
    order, select, logits = run_order(monkeypatch), beam.ops.beam_select, []

    def recorded(x, *args, **kw):
        logits.append(x.cpu())
        return select(x, *args, **kw)

    monkeypatch.setattr(beam.ops, "beam_select", recorded)
    llm = llm_for(tag, "bfloat16", width, 2)
    llm.plain_steps = True
    llm.beam_search(prompt_token_ids=prompts, params=BeamSearchParams(beam_width=width, max_new_tokens=10, ignore_eos=True))
    past = [tokens for kind, tokens in order if kind == "launch"]
    assert len(past) == 9 == len(logits) - 1
    folder = str(folder_of(tag, "bfloat16"))
    moved = 0
    for step, (tokens, rows) in enumerate(zip(past, logits[1:])):
        moved += sum(t[:-1] != past[step - 1][i] for i, t in enumerate(tokens)) if step else 0
        for i, t in enumerate(tokens):
            assert_logits_close(rows[i:i + 1], _last_logits(folder, tag, tuple(prompts[i // width] + t))[None], "bfloat16", f"step {step}, beam {i}")
    assert moved > 0                            # beams did change seats


def test_as_many_eos_tokens_as_there_are_candidates_for():
    from tokamak_b200 import BeamSearchParams
    eos = tuple(range(3, 43))                   # forty: 3 * 41 candidates, but not 32 * 41
    prompt = prompts_of("C", (20,))[0]
    llm = llm_for("C", "float32", 32, 1, eos)
    out = llm.beam_search(prompt_token_ids=[prompt], params=BeamSearchParams(beam_width=3, max_new_tokens=6))[0]
    want, _ = plain_search("C", "float32", prompt, width=3, max_new=6, stops=eos)
    assert [h.output_token_ids for h in out.hypotheses] == [t for t, _, _ in want]
    with pytest.raises(ValueError, match="EOS tokens"):
        llm.beam_search(prompt_token_ids=[prompt], params=BeamSearchParams(beam_width=32, max_new_tokens=6))
    assert llm.beam_search(prompt_token_ids=[prompt], params=BeamSearchParams(beam_width=32, max_new_tokens=6, ignore_eos=True))


def test_graphs_outlive_another_number_of_prompts():
    """Fewer prompts or tokens run on what is there; more make room for both."""
    from tokamak_b200 import BeamSearchParams
    prompts, found = prompts_of("C", (16, 40, 9, 33)), lambda outs: [[h.output_token_ids for h in o.hypotheses] for o in outs]
    params = lambda n: BeamSearchParams(beam_width=3, max_new_tokens=n, ignore_eos=True)
    llm = llm_for("C", "float32", 3, 4)
    runners, graphs = [], []
    for some, tokens in ((slice(0, 2), 12), (slice(0, 1), 12), (slice(1, 3), 7), (slice(0, 2), 12), (slice(0, 4), 5), (slice(2, 4), 12), (slice(0, 1), 20)):
        got = llm.beam_search(prompt_token_ids=prompts[some], params=params(tokens))
        fresh = llm_for("C", "float32", 3, 4)
        assert found(got) == found(fresh.beam_search(prompt_token_ids=prompts[some], params=params(tokens)))
        runners.append(llm._beam_runner)
        graphs.append(len(llm._beam_runner.graphs))
    first, wider, longer = runners[0], runners[4], runners[6]
    assert runners == [first] * 4 + [wider] * 2 + [longer] and len({id(r) for r in runners}) == 3
    assert (wider.buffers.groups, wider.longest, longer.buffers.groups, longer.longest) == (4, 12, 4, 20)
    assert graphs[1] >= graphs[0] and graphs[3] == graphs[2]             # the fourth call replays what the first has captured
    assert llm.beam_search(prompt_token_ids=prompts[:1], params=BeamSearchParams(beam_width=2, max_new_tokens=5)) and llm._beam_runner.width == 2
