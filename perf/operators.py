"""What a search over beams costs: selection over beams and vocabulary, what a beam's slot keeps moving to another slot,
and attention of single next tokens that read a shared prefix once for all of its readers.

Head counts, head sizes, vocabularies and recurrent states are those of the models that the bench and ``perf/cases.py``
run (32 query heads over 8 of 128 elements and 151,936 tokens; 16 over 4 with caps, sinks and a window of 1,024 and
states of 8 x 128 x 256 beside them); beam counts, lengths and the rest are generic.

With ``own`` false every operator is computed in elementary torch operations, in 32 bits or (keys of the selection, which
lie next to one another) in 64; with ``own`` true by the framework's kernels.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases

def _select(name, groups, beams, vocab, candidates):
    return {"name": name, "op": "select", "groups": groups, "beams": beams, "vocab": vocab, "candidates": candidates}


def _reorder(name, groups, beams, layers, state, tail, history):
    return {"name": name, "op": "reorder", "groups": groups, "beams": beams, "layers": layers, "state": state, "tail": tail,
            "history": history}


def _attention(name, groups, members, heads, kv_heads, dim, prefix, own_len, *, dtype="bf16", history=True, page=16, window=0,
               softcap=0.0, sinks=False):
    return {"name": name, "op": "attention", "groups": groups, "members": members, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "prefix": prefix, "own": own_len, "dtype": dtype, "history": history, "page": page, "window": window,
            "softcap": softcap, "sinks": sinks}


def listed():
    return [
        # the first selection of a search: one row, the prompt's last
        _select("select-first", 1, 1, 151936, 8),
        # a step of a few searches
        _select("select-8x4", 8, 4, 151936, 8),
        # many wide searches over a vocabulary whose rows start on any four bytes
        _select("select-32x16", 32, 16, 100003, 32),
        # a model without recurrent layers: only the histories move
        _reorder("reorder-history", 4, 4, 0, 0, 0, 512),
        # a few searches with the recurrent states of four layers
        _reorder("reorder-8x4", 8, 4, 4, 8 * 128 * 256, 3 * 4096, 512),
        # wide searches; convolution tails of an odd number of elements beside the states
        _reorder("reorder-12x8", 12, 8, 8, 8 * 128 * 256, 3 * 1365, 1024),
        # one search, true 32-bit path, heads of 64, a prefix that ends inside a page
        _attention("attention-f32", 1, 4, 16, 8, 64, 1021, 61, dtype="f32"),
        # one search over a prompt of ordinary length
        _attention("attention-1x8", 1, 8, 32, 8, 128, 2048, 257),
        # searches over prompts of several lengths
        _attention("attention-16x4", 16, 4, 32, 8, 128, 4093, 129),
        # 48 requests behind one long instruction, each with its own dialogue (no search: no history)
        _attention("attention-1x48", 1, 48, 32, 8, 128, 8192, 700, history=False),
        # windowed layers with caps and sinks; the window begins inside the prefix
        _attention("attention-window", 8, 8, 16, 4, 128, 2500, 300, window=1024, softcap=30.0, sinks=True),
        # long documents, wide searches
        _attention("attention-4x16", 4, 16, 32, 8, 128, 32768, 1024),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("select", "reorder", "attention", "attention"))
    if op == "select":
        groups = _log_uniform(rng, 1, 64)
        beams = _log_uniform(rng, 1, max(1, min(16, 512 // groups)))
        vocab = rng.choice((151936, 65536, _log_uniform(rng, 257, 100003)))
        if groups * beams * vocab > 32 * 16 * 100003:
            vocab = 32 * 16 * 100003 // (groups * beams)
        return _select("", groups, beams, vocab, min(2 * beams + rng.choice((0, 0, 6)), vocab))
    if op == "reorder":
        groups = _log_uniform(rng, 1, 16)
        beams = _log_uniform(rng, 2, 16)
        layers = rng.randint(0, 8)
        state = rng.choice((8 * 128 * 256, 4 * 64 * 64, _log_uniform(rng, 1000, 8 * 128 * 256)))
        tail = rng.choice((0, 3 * 4096, _log_uniform(rng, 64, 16384)))
        while layers and groups * (beams + 1) * layers * state > 12 * 9 * 8 * 8 * 128 * 256:
            layers -= 1
        return _reorder("", groups, beams, layers, state if layers else 0, tail if layers else 0, 16 * _log_uniform(rng, 1, 64))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (16, 4, 128), (16, 8, 64), (40, 8, 128)))
    groups = _log_uniform(rng, 1, 16)
    members = _log_uniform(rng, 2, max(2, 64 // groups))
    most = 2048 if dtype == "f32" else 32768
    prefix = _log_uniform(rng, 16, min(most, 4 * 32768 // groups))
    own_len = _log_uniform(rng, 1, 1024 if dtype == "bf16" else 256)
    window = rng.choice((0, 0, 0, 1024))
    return _attention("", groups, members, heads, kv_heads, dim, prefix, own_len, dtype=dtype, history=rng.random() < 0.7,
                      page=rng.choice((16, 16, 32)), window=window, softcap=rng.choice((0.0, 0.0, 30.0)),
                      sinks=rng.random() < 0.25)


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _parents(rng, *shape):
    """Which seat each seat of a search goes on from after a step: some three in ten lose their beam to a better one's
    second continuation; a beam that goes on keeps its seat."""
    beams = shape[-1]
    dead = rng.random(shape) < 0.3
    dead[..., 0] = False                       # the best one goes on
    # a random seat that goes on, for every seat
    score = np.where(dead[..., None, :], -1.0, rng.random(shape + (beams,)))
    return np.where(dead, score.argmax(-1), np.arange(beams)).astype(np.int64)


def _history(case, rng):
    """Seat that wrote each generated position of every beam's past, ``[groups, beams, own - 1]``."""
    steps = case["own"] - 1
    parents = _parents(rng, steps, case["groups"], case["members"])
    out = np.zeros((case["groups"], case["members"], max(1, steps)), dtype=np.uint8)
    now = np.broadcast_to(np.arange(case["members"]), (case["groups"], case["members"])).copy()
    for n in range(steps - 1, -1, -1):
        now = np.take_along_axis(parents[n], now, axis=1)
        out[:, :, n] = now
    return out


def _lengths(case):
    """Shared positions of every group and own positions (the new token among them) of every request."""
    g, w = case["groups"], case["members"]
    prefix = np.array([case["prefix"] - i * (case["prefix"] // (2 * g)) for i in range(g)])
    if case["history"]:
        own_len = np.full(g * w, case["own"])
    else:
        own_len = np.array([case["own"] - i * (case["own"] // (2 * g * w)) for i in range(g * w)])
    return prefix, own_len


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "attention": _prepare_attention}[case["op"]](case, seed)


def _prepare_select(case, seed):
    """Logits as a head makes them: a spread of some two and a half, a few tokens well above the rest; scores of beams that
    have run for a while."""
    g, w, v, k = case["groups"], case["beams"], case["vocab"], case["candidates"]
    gen = _gen(seed)
    logits = torch.randn(g * w, v, device=DEVICE, generator=gen) * 2.5
    top = torch.randint(0, v, (g * w, min(v, 24)), device=DEVICE, generator=gen)
    logits.scatter_add_(1, top, torch.rand(top.shape, device=DEVICE, generator=gen) * 9.0)
    scores = -20.0 - 3.0 * torch.rand(g, w, device=DEVICE, generator=gen)
    out = (torch.empty(g, k, device=DEVICE), torch.empty(g, k, dtype=torch.int32, device=DEVICE),
           torch.empty(g, k, dtype=torch.int32, device=DEVICE))
    return {"case": case, "logits": logits, "scores": scores, "out": out}


def _prepare_reorder(case, seed):
    """The records of every slot (a search holds a slot for its prompt and one for every beam, in no order) and the seats
    that the beams go on from."""
    g, w = case["groups"], case["beams"]
    rng = np.random.default_rng(seed)
    gen = _gen(seed)
    n = g * (w + 1)
    slots = rng.permutation(n)[:g * w].reshape(g, w)
    parents = _parents(rng, g, w)
    records = [torch.randint(0, w, (1, n, case["history"]), dtype=torch.uint8, device=DEVICE, generator=gen)]
    if case["layers"]:
        records.append(torch.randn(case["layers"], n, case["state"], device=DEVICE, generator=gen))
        if case["tail"]:
            records.append(torch.randn(case["layers"], n, case["tail"], device=DEVICE, generator=gen).bfloat16())
    i32 = lambda a: torch.from_numpy(a.astype(np.int32)).to(DEVICE)
    return {"case": case, "records": records, "slots": i32(slots), "parents": i32(parents),
            "err": torch.zeros(4, dtype=torch.int32, device=DEVICE)}


def _prepare_attention(case, seed):
    """Pages in no order: a group's shared positions under its own row of the block table, every request's own ones under
    the request's."""
    g, w, page, hkv, d = case["groups"], case["members"], case["page"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    rng = np.random.default_rng(seed)
    gen = _gen(seed)
    prefix, own_len = _lengths(case)
    rows = g * w
    group_of = np.repeat(np.arange(g), w)
    positions = prefix[group_of] + own_len - 1
    last = positions // page
    first = prefix[group_of] // page
    prefix_pages = -(-prefix // page)
    n_pages = int(prefix_pages.sum() + (last - first + 1).sum())
    order = rng.permutation(n_pages)
    slots = rng.permutation(g + rows)
    table = np.full((g + rows, int(max(last.max() + 1, prefix_pages.max()))), -1, dtype=np.int32)
    at = 0
    for i in range(g):
        table[slots[i], :prefix_pages[i]] = order[at:at + prefix_pages[i]]
        at += prefix_pages[i]
    for r in range(rows):
        n = last[r] - first[r] + 1
        table[slots[g + r], first[r]:last[r] + 1] = order[at:at + n]
        at += n
    history = None
    if case["history"]:
        ld = -(-case["own"] // 16) * 16
        history = np.zeros((g + rows, ld), dtype=np.uint8)
        history[slots[g:], :max(1, case["own"] - 1)] = _history(case, rng).reshape(rows, -1)
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)
    pool = torch.randn(2, n_pages, hkv, page, d, device=DEVICE, generator=gen, dtype=torch.float32).to(dtype)
    q = (torch.randn(rows, case["heads"], d, device=DEVICE, generator=gen) * 1.5).to(dtype)
    sinks = torch.randn(case["heads"], device=DEVICE, generator=gen) if case["sinks"] else None
    return {"case": case, "q": q, "out": torch.empty_like(q), "k": pool[0], "v": pool[1], "table": i32(table),
            "positions": i32(positions), "req_slot": i32(slots[g:]), "group_start": i32(np.arange(g + 1) * w),
            "prefix_slot": i32(slots[:g]), "prefix_len": i32(prefix),
            "history": None if history is None else torch.from_numpy(history).to(DEVICE), "sinks": sinks,
            "max_prefix": int(prefix.max()), "max_own": int(own_len.max()), "scale": d ** -0.5,
            "err": torch.zeros(4, dtype=torch.int32, device=DEVICE)}


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"select": _own_select, "reorder": _own_reorder, "attention": _own_attention}[op](state)
    return {"select": _plain_select, "reorder": _plain_reorder, "attention": _plain_attention}[op](state)


def _own_select(s):
    from tokamak_b200.csrc import ops
    return ops.beam_select(s["logits"], s["scores"], s["case"]["candidates"], out=s["out"])


def _own_reorder(s):
    from tokamak_b200.csrc import ops
    ops.reorder_slots(s["records"], s["slots"], s["parents"], s["err"])
    return s["records"]


def _own_attention(s):
    from tokamak_b200.csrc import ops
    c = s["case"]
    shared = ops.SharedPrefix(s["group_start"], s["prefix_slot"], s["prefix_len"], max_members=c["members"],
                              max_prefix=s["max_prefix"], max_own=s["max_own"], history=s["history"])
    ops.attention_shared(s["q"], s["out"], s["k"], s["v"], shared, s["positions"], s["req_slot"], s["table"], s["err"],
                         scale=s["scale"], window=c["window"] or None, softcap=c["softcap"] or None, sinks=s["sinks"])
    return s["out"]


def _plain_select(s):
    """Keys in 64 bits: the K-th and the one behind it may differ in the last bits of 32."""
    c = s["case"]
    x = s["logits"].double()
    x = x - x.amax(dim=1, keepdim=True)
    x -= x.exp().sum(dim=1, keepdim=True).log()
    keys = (x.view(c["groups"], c["beams"], -1) + s["scores"].double()[:, :, None]).view(c["groups"], -1)
    # equal keys: the lowest place first, which a stable order keeps
    best, at = torch.sort(keys, dim=1, descending=True, stable=True)
    best, at = best[:, :c["candidates"]], at[:, :c["candidates"]]
    return best.float(), (at // c["vocab"]).int(), (at % c["vocab"]).int()


def _move(records, slots, source):
    records[:, slots] = records[:, source]
    return records


def _plain_reorder(s):
    slots = s["slots"].long()
    source = slots.gather(1, s["parents"].long())
    return [_move(t, slots, source) for t in s["records"]]


def _plain_attention(s):
    c = s["case"]
    g, w, hkv, d, page = c["groups"], c["members"], c["kv_heads"], c["dim"], c["page"]
    per = c["heads"] // hkv
    table, slot = s["table"].long(), s["req_slot"].long()
    prefix = s["prefix_len"].long()
    positions = s["positions"].long()
    group_of = torch.arange(g, device=DEVICE).repeat_interleave(w)
    q = s["q"].float().view(g, w, hkv, per, d)
    k, v = s["k"].permute(0, 2, 1, 3), s["v"].permute(0, 2, 1, 3)              # [page, offset, head, d]
    # the shared positions of every group
    t = torch.arange(s["max_prefix"], device=DEVICE)
    where = (s["prefix_slot"].long()[:, None], (t // page)[None, :])
    pages = table[where].clamp_min(0)
    off = (t % page)[None, :].expand_as(pages)
    kp, vp = k[pages, off].float(), v[pages, off].float()                      # [g, P, hkv, d]
    low = positions.view(g, w) - c["window"] + 1 if c["window"] else torch.zeros(g, w, dtype=torch.long, device=DEVICE)
    seen_p = (t < prefix[:, None, None]) & (t >= low[:, :, None])              # [g, w, P]
    sp = torch.einsum("gwhpd,gkhd->gwhpk", q, kp)
    # the positions behind them, in the pages of whoever wrote them
    n = torch.arange(s["max_own"], device=DEVICE)
    at = prefix[group_of][:, None] + n                                         # [rows, S]
    writer = slot[:, None].expand(-1, s["max_own"])
    if s["history"] is not None:
        seat = s["history"][slot][:, :s["max_own"]].long().clamp_max(w - 1)
        writer = torch.where(at < positions[:, None], slot.view(g, w)[group_of[:, None], seat], writer)
    pages = table[writer, (at // page).clamp_max(table.shape[1] - 1)].clamp_min(0)
    ko, vo = k[pages, at % page].float().view(g, w, -1, hkv, d), v[pages, at % page].float().view(g, w, -1, hkv, d)
    seen_o = ((at <= positions[:, None]) & (at >= low.reshape(-1)[:, None])).view(g, w, -1)
    so = torch.einsum("gwhpd,gwkhd->gwhpk", q, ko)
    score = torch.cat((sp, so), dim=-1) * s["scale"]
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    score = score.masked_fill(~torch.cat((seen_p, seen_o), dim=-1)[:, :, None, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    score = (score - top).exp_()
    total = score.sum(dim=-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (s["sinks"].view(1, 1, hkv, per, 1) - top).exp()
    score /= total
    np_ = sp.shape[-1]
    out = torch.einsum("gwhpk,gkhd->gwhpd", score[..., :np_], vp) + torch.einsum("gwhpk,gwkhd->gwhpd", score[..., np_:], vo)
    return out.reshape(g * w, c["heads"], d).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    return {"select": _work_select, "reorder": _work_reorder, "attention": _work_attention}[case["op"]](case)


def _work_select(c):
    rows = c["groups"] * c["beams"]
    # a subtraction, an exponential, a sum and a comparison for every logit
    return {"bytes": 4 * rows * c["vocab"] + 4 * rows + 12 * c["groups"] * c["candidates"], "flops": 4 * rows * c["vocab"]}


def _work_reorder(c):
    """Records that change are written, the different ones that they come from read."""
    rng = np.random.default_rng(0)
    g, w = c["groups"], c["beams"]
    rng.permutation(g * (w + 1))
    parents = _parents(rng, g, w)
    moved = parents != np.arange(w)
    sources = sum(len(set(parents[i][moved[i]])) for i in range(g))
    each = c["history"] + c["layers"] * (4 * c["state"] + 2 * c["tail"])
    return {"bytes": max(1, int(moved.sum()) + sources) * each + 8 * g * w, "flops": 0}


def _work_attention(c):
    prefix, own_len = _lengths(c)
    g, w = c["groups"], c["members"]
    size = torch.empty(0, dtype=DTYPES[c["dtype"]]).element_size()
    row = 2 * c["kv_heads"] * c["dim"] * size                # a position's keys and values
    positions = np.repeat(prefix, w) + own_len - 1
    low = np.maximum(0, positions - c["window"] + 1) if c["window"] else np.zeros_like(positions)
    shared = np.maximum(0, np.repeat(prefix, w) - low)       # shared positions that a request sees
    mine = positions + 1 - np.maximum(low, np.repeat(prefix, w))
    total = shared.reshape(g, w).max(axis=1).sum() * row
    if c["history"]:
        # positions that beams have in common lie in one place
        seats = _history(c, np.random.default_rng(0))
        skip = c["own"] - int(mine.max())
        past = np.sort(seats[:, :, skip:c["own"] - 1], axis=1)
        distinct = past.shape[0] * past.shape[2] + int((past[:, 1:] != past[:, :-1]).sum()) if c["own"] > 1 else 0
        total += (distinct + g * w) * row
    else:
        total += int(mine.sum()) * row
    total += 2 * g * w * c["heads"] * c["dim"] * size
    return {"bytes": int(total), "flops": int(4 * c["heads"] * c["dim"] * (shared + mine).sum())}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "attention": _exact_attention}[case["op"]](s)


def _exact_select(s):
    """Row by row in 64 bits: log probabilities, then the best of all rows of a group."""
    c = s["case"]
    picked = []
    for i in range(c["groups"]):
        rows = []
        for b in range(c["beams"]):
            x = s["logits"][i * c["beams"] + b].double()
            rows.append(s["scores"][i, b].double() + torch.log_softmax(x, 0))
        picked.append(torch.topk(torch.cat(rows), c["candidates"]).values)
    return torch.stack(picked), None, None


def _exact_reorder(s):
    """Record by record."""
    slots, parents = s["slots"].tolist(), s["parents"].tolist()
    out = []
    for t in s["records"]:
        new = t.clone()
        for row, frm in zip(slots, parents):
            for slot, p in zip(row, frm):
                new[:, slot] = t[:, row[p]]
        out.append(new.double() if new.is_floating_point() else new)
    return out


def _exact_attention(s):
    """Request by request: its visible positions one after the other, wherever they lie."""
    c = s["case"]
    w, page, per = c["members"], c["page"], c["heads"] // c["kv_heads"]
    prefix, positions = s["prefix_len"].tolist(), s["positions"].tolist()
    slots, prefix_slot = s["req_slot"].tolist(), s["prefix_slot"].tolist()
    table = s["table"].long()
    out = torch.empty(len(slots), c["heads"], c["dim"], dtype=torch.float64, device=DEVICE)
    for r, slot in enumerate(slots):
        g = r // w
        first = max(0, positions[r] - c["window"] + 1) if c["window"] else 0
        pos = torch.arange(first, positions[r] + 1, device=DEVICE)
        writer = torch.full_like(pos, slot)
        if s["history"] is not None:
            past = (pos >= prefix[g]) & (pos < positions[r])
            seats = s["history"][slot, (pos - prefix[g])[past]].long()
            writer[past] = s["req_slot"][g * w:(g + 1) * w].long()[seats]
        writer[pos < prefix[g]] = prefix_slot[g]
        at = table[writer, pos // page]
        k, v = s["k"][at, :, pos % page].double(), s["v"][at, :, pos % page].double()        # [keys, hkv, d]
        q = s["q"][r].double().view(c["kv_heads"], per, -1)
        x = torch.matmul(q, k.permute(1, 2, 0)) * s["scale"]
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        if s["sinks"] is not None:
            x = torch.cat((x, s["sinks"].double().view(c["kv_heads"], per, 1)), dim=-1)
        p = torch.softmax(x, dim=-1)[..., :pos.numel()]
        out[r] = torch.matmul(p, v.permute(1, 0, 2)).reshape(c["heads"], -1)
    return out
