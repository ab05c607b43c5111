"""The steps of ``LLM.beam_search``: what they carry, in which order they run, and what of them is kept between calls."""

from __future__ import annotations

import gc

import pytest
import torch

import tiny_configs
from test_beam_search_gpu import _last_logits, folder_of, llm_for, plain_search, prompts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def nothing_left_behind():
    """Engines, their graphs and the memory that held them are gone before the next test, of whichever file."""
    yield
    gc.collect()
    torch.cuda.empty_cache()


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


@pytest.mark.parametrize("width,tokens,eos", [(8, 4, ()), (6, 5, (2,)), (16, 3, (0, 4))])
def test_vocabularies_smaller_than_a_search_is_wide(width, tokens, eos, tmp_path):
    """One row has fewer continuations than there are beams; several have enough."""
    import json

    from plain import beam_plain, qwen3_plain
    from tokamak_b200 import LLM, BeamSearchParams
    from tokamak_b200.weights import write_random_model
    raw, init, page = tiny_configs.ALL["C"]
    write_random_model(str(tmp_path), {**raw, "vocab_size": 7}, dtype="float32", **init)
    if eos:
        path = tmp_path / "config.json"
        path.write_text(json.dumps({**json.loads(path.read_text()), "eos_token_id": list(eos)}))
    cfg, weights = qwen3_plain.load_folder(str(tmp_path))
    prompt = [1, 5, 3]
    llm = LLM(tmp_path, dtype="float32", block_size=page, max_batch_size=width + 1, kv_pool_tokens=4096)
    found = llm.beam_search(prompt_token_ids=[prompt], params=BeamSearchParams(beam_width=width, max_new_tokens=tokens))[0].hypotheses
    want, _ = beam_plain.search(lambda t: qwen3_plain.forward_logits(cfg, weights, list(t), torch.float64)[-1], prompt, width=width, max_new=tokens,
                                stops=eos)
    assert [h.output_token_ids for h in found] == [t for t, _, _ in want] and len(found) == width
