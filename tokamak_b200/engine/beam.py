"""Search over beams: ``LLM.beam_search``.

A search holds a slot for its prompt, whose pages all of its beams read (``ops.attention_shared``), and one for every
beam, with pages of its own for the positions behind the prompt and the fixed-size records of the model's recurrent
layers.  A step brings the next token of every beam of all searches that run:

* the forward pass over the slot records, as a step of single next tokens is always opened;
* ``ops.beam_select`` ranks the continuations of every search, ``ops.beam_advance`` says which of them go on in which
  slots and writes their tokens into the slot records;
* ``ops.reorder_slots`` moves what the recurrent layers keep, and the beams' histories, to the slots that go on.

Keys and values never move: a beam's history names, position by position, the beam in whose pages they lie.  Nothing of
this needs the host, so a step is launched before the one before it has been read and, where every part of the model
allows it, replayed from a CUDA graph; the host reads the ranked continuations of every step and keeps the tree of tokens
and the hypotheses that have ended.

Searches that do not fit side by side (slots, pages) run one wave after the other.  Layers whose attention has options that
the shared-prefix kernel does not know are refused (a mixer declares ``SHARED_PREFIX``).
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

from ..cache.manager import KVPagesNeed
from ..csrc import ops
from ..models.decoder import flat_needs
from ..sampling.beam import BeamSearchParams
from .step import StepBatch, StepEntry, StepFunction, _bucket


def stops_max(width: int) -> int:
    """EOS tokens for which there are candidates enough: were all of them ranked first in every beam, ``width`` others must be left."""
    return ops.BEAM_MAX_CANDIDATES // width - 1


def refuses_search(model) -> str | None:
    """Why a model's layers cannot be searched over, or ``None``."""
    for name, block in model.blocks.items():
        pages = any(isinstance(need, KVPagesNeed) for _, need in flat_needs(name, block.cache_need()))
        if pages and not getattr(getattr(block, "mixer", None), "SHARED_PREFIX", False):
            mixer = type(getattr(block, "mixer", block)).__name__
            return f"the attention of block {name!r} ({mixer}) cannot read keys that beams share"
    return None


@dataclass
class Hypothesis:
    """An ended continuation: its tokens, the sum of their log probabilities, and whether an EOS token ended it."""

    tokens: list[int]
    sum_logprobs: float
    ended: bool

    def score(self, length_penalty: float) -> float:
        return self.sum_logprobs / len(self.tokens) ** length_penalty


def path(node) -> list[int]:
    """Tokens from the root of a tree to ``node``, which is ``(parent, token)``, or ``None`` for the root."""
    out = []
    while node is not None:
        node, token = node
        out.append(token)
    return out[::-1]


@dataclass
class Search:
    """One prompt's search as the host keeps it."""

    index: int
    prompt: list[int]
    budget: int                         # most tokens that may be generated
    beams: list = field(default_factory=list)        # request ids of the beams, seat by seat
    heads: list = field(default_factory=list)        # last node of every running beam in the tree of tokens, seat by seat
    length: int = 0                     # tokens of a running beam
    scores: list[float] = field(default_factory=list)
    ended: list[Hypothesis] = field(default_factory=list)
    done: bool = False

    @property
    def prompt_id(self):
        return ("prompt", self.index)

    @property
    def tokens(self) -> list[list[int]]:
        """Tokens of every running beam, seat by seat."""
        return [path(head) for head in self.heads]

    def take(self, params: BeamSearchParams, stops: frozenset, candidates, seats) -> None:
        """One step's ranked continuations and the beams that go on: ended ones become hypotheses."""
        width = params.beam_width
        running = 0
        for score, parent, token in candidates:
            if running == width or score == -math.inf:
                break                    # what ranks behind the last beam that goes on does not end a hypothesis either
            if token in stops:
                self.ended.append(Hypothesis(path((self.heads[parent] if self.heads else None, token)), score, True))
            else:
                running += 1
        past = self.heads or [None] * width
        self.heads = [(past[parent], token) for _, parent, token in seats]
        self.scores = [score for score, _, _ in seats]
        self.length = length = self.length + 1
        rank = lambda h: -h.score(params.length_penalty)
        self.ended = sorted(self.ended, key=rank)[:width]
        best = max(self.scores)
        if len(self.ended) == width:
            # sums only fall: at its present length no running beam will be ranked higher than it is now
            worst = self.ended[-1].score(params.length_penalty)
            self.done = params.early_stopping or best / length ** params.length_penalty <= worst
        self.done = self.done or best == -math.inf or length >= self.budget

    def hypotheses(self, params: BeamSearchParams) -> list[Hypothesis]:
        """The best hypotheses, ended or cut off at the cap on tokens, best first."""
        out = list(self.ended)
        if len(out) < params.beam_width or self.length >= self.budget:
            out += [Hypothesis(t, s, False) for t, s in zip(self.tokens, self.scores) if s > -math.inf]
        return sorted(out, key=lambda h: -h.score(params.length_penalty))[:params.beam_width]


class BeamBuffers:
    """Tensors at fixed addresses that describe the running searches, for at most ``groups`` of ``width`` beams."""

    def __init__(self, step: StepFunction, groups: int, width: int, candidates: int, longest: int):
        device = step.device
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)
        self.groups, self.width, self.candidates = groups, width, candidates
        self.parts = (("cand_scores", candidates, torch.float64), ("scores", width, torch.float64), ("cand_parents", candidates, torch.int32),
                      ("cand_tokens", candidates, torch.int32), ("parents", width, torch.int32), ("tokens", width, torch.int32))
        self.history = torch.zeros((step.manager.max_slots, -(-longest // 16) * 16), dtype=torch.uint8, device=device)
        self.group_start = torch.arange(groups + 1, dtype=torch.int32, device=device) * width
        self.prefix_slot, self.prefix_len = i32(groups), i32(groups)
        # what the host reads of a step: for every search the ranked continuations and the beams that go on, whose scores, in 64
        # bits, are what the next step starts from
        self.words = i32(groups * 4 * (candidates + width))
        self.hosts = [torch.zeros(4 + self.words.numel(), dtype=torch.int32).pin_memory() for _ in range(3)]
        self.turn = 0

    def views(self, n: int, words: torch.Tensor | None = None) -> dict:
        """The parts of ``words`` (the device's, or a copy of them) for ``n`` searches."""
        words = self.words if words is None else words
        at, out = 0, {}
        for name, size, dtype in self.parts:
            taken = n * size * dtype.itemsize // 4
            out[name] = words[at:at + taken].view(dtype).view(n, size)
            at += taken
        out["used"] = at
        return out


@dataclass
class _Pending:
    searches: list
    host: torch.Tensor
    event: torch.cuda.Event


class BeamRunner:
    """Runs searches of one width on an engine's step function, at most ``max_groups`` side by side and none longer than
    ``longest`` tokens."""

    def __init__(self, step: StepFunction, width: int, stops, max_groups: int, longest: int):
        self.step, self.width, self.longest = step, width, longest
        self.cache, self.manager, self.model = step.cache, step.manager, step.model
        self.stops = frozenset(stops)
        self.vocab = self.model.spec.head.vocab_size
        # were every EOS token ranked in front of the others in every beam, `width` others are left; a first step has one row's
        self.candidates = min(width * (1 + len(self.stops)), width * self.vocab)
        self.buffers = BeamBuffers(step, max_groups, width, self.candidates, longest)
        self.stop_tokens = (torch.tensor(sorted(self.stops), dtype=torch.int32, device=step.device) if self.stops else None)
        self.records = list(self.cache._states) + [self.buffers.history.unsqueeze(0)]
        self.graphs: dict = {}
        self.seen: dict = {}
        self.placed = 0                  # searches that the buffers hold

    def takes(self, width: int, stops, groups: int, longest: int) -> bool:
        """Whether its buffers, and the graphs that hold their addresses, do for searches of this kind."""
        return (width == self.width and frozenset(stops) == self.stops and groups <= self.buffers.groups and longest <= self.longest)

    def start(self, params: BeamSearchParams, max_step_tokens: int, plain: bool = False) -> None:
        """What one call asks for.  ``plain``: no step is launched before the one before it has been read, and none is replayed; the
        host writes every beam's position and token."""
        self.params, self.max_step_tokens, self.plain, self.steps = params, max_step_tokens, plain, 0

    # ---- prompts ---------------------------------------------------------------------------------------------------
    def prefill(self, searches: list[Search]) -> torch.Tensor:
        """Logits of every prompt's last token; prompts go through in steps of at most ``max_step_tokens`` tokens."""
        logits = torch.empty((len(searches), self.vocab), dtype=torch.float32, device=self.step.device)
        at = [0] * len(searches)
        while True:
            room, entries, last = self.max_step_tokens, [], []
            for i, s in enumerate(searches):
                n = min(room, len(s.prompt) - at[i])
                if n <= 0:
                    continue
                ends = at[i] + n == len(s.prompt)
                entries.append(StepEntry(s.prompt_id, s.prompt[at[i]:at[i] + n], [n - 1] if ends else []))
                if ends:
                    last.append(i)
                at[i] += n
                room -= n
            if not entries:
                return logits
            got = self.step.run(entries)
            self.steps += 1
            if last:
                logits[torch.tensor(last, device=logits.device)] = got

    @torch.inference_mode()
    def begin(self, searches: list[Search]) -> None:
        """Run the prompts, pick the first beams and give them slots that go on from their prompt's."""
        n, w, b = len(searches), self.width, self.buffers
        device = self.step.device
        logits = self.prefill(searches)
        v = b.views(n)
        cand = ops.beam_select(logits, torch.zeros((n, 1), dtype=torch.float64, device=device), min(self.candidates, self.vocab),
                               score_dtype=torch.float64)
        v["cand_scores"].fill_(-math.inf)
        for name, part in zip(("cand_scores", "cand_parents", "cand_tokens"), cand):
            v[name][:, :part.shape[1]] = part
        seats = []
        for s in searches:
            s.beams = [(s.index, i) for i in range(w)]
            for beam in s.beams:
                self.manager.fork(s.prompt_id, beam)
            seats.append([self.manager.slot(s.prompt_id)] + [self.manager.slot(beam) for beam in s.beams])
        slots = torch.tensor(seats, dtype=torch.int32, device=device)
        err = self.step.buffers.result[:4]
        ops.beam_advance((v["cand_scores"], v["cand_parents"], v["cand_tokens"]), self.stop_tokens, slots[:, 1:].contiguous(),
                         v["scores"], v["parents"], v["tokens"], err, begin=True)
        self.placed = n
        if self.cache._states:
            ops.reorder_slots(self.cache._states, slots, torch.zeros_like(slots), err)
        self.collect(self._read(searches, v["used"]))
        self.write_records(searches)

    def write_records(self, searches: list[Search]) -> None:
        """Where every beam is and its last token, for the next step."""
        for s in searches:
            for beam, (_, token) in zip(s.beams, s.heads):
                self.cache.write_record(self.manager.slot(beam), temperature=0.0, top_k=0, top_p=1.0, seed=0,
                                        computed=self.manager.length(beam), last_token=token)

    def place(self, searches: list[Search], order: list[int]) -> None:
        """Put what the device holds of the running searches in their order (``order``: where each was before)."""
        n, b = len(searches), self.buffers
        if len(order) != self.placed:
            b.views(n)["scores"].copy_(b.views(self.placed)["scores"][torch.tensor(order, device=self.step.device)])
            self.placed = n
        meta = torch.tensor([[self.manager.slot(s.prompt_id) for s in searches], [len(s.prompt) for s in searches]],
                            dtype=torch.int32, device=self.step.device)
        b.prefix_slot[:n].copy_(meta[0])
        b.prefix_len[:n].copy_(meta[1])

    # ---- steps of the beams -------------------------------------------------------------------------------------------
    def _launches(self, batch: StepBatch, n: int) -> None:
        st, b, w = self.step, self.buffers, self.width
        v = b.views(n)
        slots = st.buffers.dec_slots[:n * w].view(n, w)
        ops.decode_begin(st.buffers.updates, st.buffers.dec_slots, n * w, st.max_seq_len, st.buffers.dec_token_ids,
                         st.buffers.dec_positions, st.buffers.dec_kv_len, batch.err)
        logits = self.model.forward(batch)
        cand = ops.beam_select(logits, v["scores"], self.candidates, out=(v["cand_scores"], v["cand_parents"], v["cand_tokens"]),
                               score_dtype=torch.float64)
        ops.beam_advance(cand, self.stop_tokens, slots, v["scores"], v["parents"], v["tokens"], batch.err,
                         records=self.cache.slot_records, history=b.history, positions=batch.positions, prefix_len=b.prefix_len)
        ops.reorder_slots(self.records, slots, v["parents"], batch.err)

    @torch.inference_mode()
    def launch(self, searches: list[Search], done: int) -> _Pending:
        """Start the step that brings every beam's token number ``done`` (one is there) to its next."""
        st, n, w, b = self.step, len(searches), self.width, self.buffers
        entries = [StepEntry(beam, None, [0]) for s in searches for beam in s.beams]
        if self.plain:
            self.write_records(searches)
        batch = st._build_from_state(entries)
        # the bounds are buckets, so that what the kernels plan from them changes rarely
        prefix = _bucket(max(len(s.prompt) for s in searches))
        own = min(_bucket(done), max(self.longest, 1))
        batch.shared = ops.SharedPrefix(b.group_start[:n + 1], b.prefix_slot[:n], b.prefix_len[:n], max_members=w, max_prefix=prefix,
                                        max_own=own, history=b.history)
        key = (n, batch.max_kv_len, prefix, own)
        graph = self.graphs.get(key)
        if graph is None and st.use_graphs and st.graph_safe and not self.plain and self.seen.get(key, 0) >= 1:
            graph = self._capture(key, batch, n)
        if graph is not None and not self.plain:
            graph["graph"].replay()
            st.graph_launches += graph["kernels"]
            st.graph_replays += 1
        else:
            self.seen[key] = self.seen.get(key, 0) + 1
            self._launches(batch, n)
        st.finish(entries)
        self.steps += 1
        return self._read(searches, b.views(n)["used"])

    def _capture(self, key, batch: StepBatch, n: int) -> dict:
        st = self.step
        if st._graph_pool is None:
            st._graph_pool = torch.cuda.graph_pool_handle()
        graph = torch.cuda.CUDAGraph()
        before = ops.LAUNCHES
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, pool=st._graph_pool):
            self._launches(batch, n)
        self.graphs[key] = {"graph": graph, "kernels": ops.LAUNCHES - before}
        ops.LAUNCHES = before
        return self.graphs[key]

    def _read(self, searches: list[Search], used: int) -> _Pending:
        b, bufs = self.buffers, self.step.buffers
        host = b.hosts[b.turn]
        b.turn = (b.turn + 1) % len(b.hosts)
        host[:4].copy_(bufs.result[:4], non_blocking=True)
        host[4:4 + used].copy_(b.words[:used], non_blocking=True)
        bufs.d2h_bytes += 4 * (4 + used)
        event = torch.cuda.Event()
        event.record()
        return _Pending(list(searches), host, event)

    def collect(self, pending: _Pending) -> bool:
        """Read a step; whether a search ended with it."""
        pending.event.synchronize()
        self.step._raise_on_error(pending.host[:4].tolist())
        cols = {name: part.tolist() for name, part in self.buffers.views(len(pending.searches), pending.host[4:]).items() if name != "used"}
        ended = False
        for i, s in enumerate(pending.searches):
            if not s.done:
                s.take(self.params, self.stops, zip(*(cols[name][i] for name in ("cand_scores", "cand_parents", "cand_tokens"))),
                       list(zip(*(cols[name][i] for name in ("scores", "parents", "tokens")))))
                ended = ended or s.done
        return ended

    def free(self, s: Search) -> None:
        for beam in s.beams:
            self.manager.free(beam)
        self.manager.free(s.prompt_id)

    def run(self, searches: list[Search]) -> None:
        """All searches of one wave to their ends."""
        try:
            self.begin(searches)
            running, order = [s for s in searches if not s.done], [i for i, s in enumerate(searches) if not s.done]
            pending, done, fresh = None, 1, True
            while running or pending is not None:
                if pending is None:
                    if fresh:
                        self.place(running, order)
                        fresh = False
                    pending = self.launch(running, done)
                    done += 1
                ahead = None
                if not self.plain and all(s.budget > done for s in running):
                    # the next step needs nothing of this one that is not on the device
                    ahead = self.launch(running, done)
                    done += 1
                if self.collect(pending):
                    if ahead is not None:
                        self.collect(ahead)          # what it brings for the searches that have ended is not looked at
                        ahead = None
                    order = [i for i, s in enumerate(running) if not s.done]
                    for s in running:
                        if s.done:
                            self.free(s)
                    running, fresh = [running[i] for i in order], True
                pending = ahead
        finally:
            torch.cuda.current_stream(self.step.device).synchronize()      # nothing in flight reads pages that go back
            for s in searches:
                self.free(s)
