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
