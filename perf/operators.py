"""Serving a batch of requests over a paged KV cache, as measurable cases.

Four operators work together in a server's step: the plan lays out pages for
the new tokens of every request, the append rotates Q and K and writes K and
V to their slots, and attention runs either over the cached pages (decode,
chunks of a prompt) or over whole packed prompts.

``listed()`` holds named cases, ``draw(rng)`` gives more of the same ranges.
``prepare`` makes the device tensors a server has in hand before the call,
``run`` is one pass -- the plain torch form, or the framework's calls where
``own`` is true -- ``exact`` the same outputs in 64 bits from the operators'
definitions, and ``work`` the bytes and operations no implementation can do
without.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

NONE = -1  # no page, no slot: 0xFFFFFFFF of the library's u32, seen as int32
THETA = 10000.0

# (query heads, KV heads): the head groupings of the test suite and the benchmark.
HEADS = [(9, 3), (15, 5), (32, 8), (8, 8), (12, 3)]
DTYPES = {"f16": (torch.float16, 2), "f32": (torch.float32, 4)}


def listed() -> list[dict]:
    return [
        # One decode step's plan: every running request gets a slot, some a new page.
        {"name": "plan_decode", "op": "plan", "decodes": 48, "chunks": 0, "chunk": 1, "idle": 3,
         "longest": 4000, "page": 16, "padding": 13},
        # A full batch where prompts come in: thousands of new tokens, many new pages.
        {"name": "plan_prompts", "op": "plan", "decodes": 384, "chunks": 96, "chunk": 512, "idle": 32,
         "longest": 4000, "page": 64, "padding": 0},
        # The append of one decode step of the 360M model's heads, the batch padded to a fixed size.
        {"name": "append_decode_f16", "op": "append", "dtype": "f16", "heads": 15, "kv_heads": 5,
         "head_dim": 64, "decodes": 27, "chunks": 0, "chunk": 1, "idle": 0, "longest": 2000,
         "page": 16, "padding": 5},
        # The append of several prompt chunks and decodes, heads of 128.
        {"name": "append_chunks_f16", "op": "append", "dtype": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "decodes": 31, "chunks": 16, "chunk": 512, "idle": 1, "longest": 1000,
         "page": 32, "padding": 0},
        # A handful of short prompts at once: latency counts.
        {"name": "packed_short_f16", "op": "packed", "dtype": "f16", "heads": 15, "kv_heads": 5,
         "head_dim": 64, "prompts": 7, "longest": 200, "padding": 9},
        # A batch of long prompts of a model with heads of 128.
        {"name": "packed_long_f16", "op": "packed", "dtype": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "prompts": 8, "longest": 4096, "padding": 0},
        # The same in f32 (models loaded without conversion), ragged.
        {"name": "packed_f32", "op": "packed", "dtype": "f32", "heads": 9, "kv_heads": 3,
         "head_dim": 64, "prompts": 5, "longest": 1021, "padding": 0},
        # One user's decode step: the smallest call, all latency.
        {"name": "decode_one_f16", "op": "paged", "dtype": "f16", "heads": 15, "kv_heads": 5,
         "head_dim": 64, "decodes": 1, "chunks": 0, "chunk": 1, "idle": 0, "longest": 1535,
         "page": 16, "padding": 0},
        # A server's decode step over ragged contexts: bound by the bytes of the cache.
        {"name": "decode_batch_f16", "op": "paged", "dtype": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "decodes": 60, "chunks": 0, "chunk": 1, "idle": 4, "longest": 8000,
         "page": 16, "padding": 0},
        # One very long document: a single token over a hundred thousand cached ones.
        {"name": "decode_long_f16", "op": "paged", "dtype": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "decodes": 1, "chunks": 0, "chunk": 1, "idle": 0, "longest": 100003,
         "page": 64, "padding": 0},
        # Prompts taken in chunks while other requests decode, in one call.
        {"name": "chunks_and_decodes_f16", "op": "paged", "dtype": "f16", "heads": 15,
         "kv_heads": 5, "head_dim": 64, "decodes": 20, "chunks": 4, "chunk": 509, "idle": 0,
         "longest": 4000, "page": 32, "padding": 3},
        # A decode step in f32, two new tokens for some (a draft being checked).
        {"name": "decode_f32", "op": "paged", "dtype": "f32", "heads": 9, "kv_heads": 3,
         "head_dim": 64, "decodes": 13, "chunks": 3, "chunk": 2, "idle": 1, "longest": 3000,
         "page": 16, "padding": 0},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case: dict) -> float:
    """What bounds a case's pass: its bytes, operations, and the plain form's padded scores."""
    w = work(case)
    scores = 0
    if case["op"] in ("packed", "paged"):
        spans = _spans(case)
        scores = (len(spans) * case["heads"] * max(n for _, n in spans)
                  * max(c + n for c, n in spans))
    return max(w["bytes"], w["flops"] / 50, 4 * scores)


def draw(rng) -> dict:
    op = rng.choice(["plan", "append", "packed", "packed", "paged", "paged", "paged"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        case = {"op": op}
        if op != "plan":
            case["dtype"] = rng.choice(["f16", "f16", "f32"])
            case["heads"], case["kv_heads"] = rng.choice(HEADS)
            case["head_dim"] = rng.choice([64, 64, 128, 128, 96, 80, 32])
        if op == "packed":
            case.update(prompts=_log(rng, 1, 48), longest=_log(rng, 16, 4096),
                        padding=rng.choice([0, 0, rng.randrange(1, 40)]))
        else:
            chunked = rng.random() < 0.4
            case.update(decodes=_log(rng, 1, 400 if op == "plan" else 96),
                        chunks=_log(rng, 1, 96 if op == "plan" else 12) if chunked else 0,
                        chunk=_log(rng, 2, 600) if chunked else 1,
                        idle=rng.choice([0, 0, rng.randrange(1, 9)]),
                        longest=_log(rng, 16, 4000 if op != "paged" else 20000),
                        page=rng.choice([16, 16, 32, 64, 128]),
                        padding=rng.choice([0, 0, rng.randrange(1, 40)]))
        if _cost(case) <= most:
            return case


# ------------------------------------------------------------------ inputs


def _spans(case: dict) -> list[tuple[int, int]]:
    """(cached, new) tokens of every request, the same for every seed but for their order:
    lengths spread up to the longest, which is among them."""
    if case["op"] == "packed":
        rng = random.Random(1000 * case["prompts"] + case["longest"])
        return [(0, case["longest"])] + [(0, _log(rng, max(1, case["longest"] // 16),
                                                   case["longest"]))
                                         for _ in range(case["prompts"] - 1)]
    rng = random.Random(1000 * case["decodes"] + case["longest"])
    cached = [case["longest"]] + [rng.randint(0, case["longest"])
                                  for _ in range(case["decodes"] + case["chunks"] - 1)]
    new = [1] * case["decodes"] + [case["chunk"]] * case["chunks"]
    return list(zip(cached, new)) + [(0, 0)] * case["idle"]


def _int(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _layout(case: dict, seed: int) -> dict:
    """The requests of a step in the seed's order, and the pages that they hold."""
    rng = random.Random(seed)
    spans = _spans(case)
    rng.shuffle(spans)
    offsets = [0]
    for _, n in spans:
        offsets.append(offsets[-1] + n)
    tokens = offsets[-1] + case["padding"]
    t = {"offsets": _int(offsets), "tokens": tokens, "sequences": len(spans), "spans": spans,
         "max_queries": max(n for _, n in spans), "max_context": max(c + n for c, n in spans)}
    if case["op"] == "packed":
        return t
    page = case["page"]
    whole = [-(-(c + n) // page) for c, n in spans]
    had = [-(-c // page) for c, _ in spans]
    t["max_blocks"] = -(-(case["longest"] + case["chunk"]) // page)
    # the pages of the cache, in the order that a server's coming and going leaves
    t["pages"] = sum(whole) + 8
    ids = np.random.default_rng(seed).permutation(t["pages"])
    table = np.full((len(spans), t["max_blocks"]), NONE, np.int32)
    free, at = [], 0
    for i, n in enumerate(whole):
        table[i, :n] = ids[at:at + n]
        free += list(range(at + had[i], at + n))
        at += n
    t["free"] = _int(np.concatenate([ids[free], ids[at:]]).astype(np.int32))
    before = table.copy()
    for i, n in enumerate(had):
        before[i, n:] = NONE
    t["table_before"] = torch.from_numpy(before).cuda()
    t["table"] = torch.from_numpy(table).cuda()
    t["context"] = _int([c + n for c, n in spans])
    positions = np.zeros(tokens, np.int32)
    slots = np.full(tokens, NONE, np.int32)
    for i, (c, n) in enumerate(spans):
        pos = np.arange(c, c + n)
        positions[offsets[i]:offsets[i + 1]] = pos
        slots[offsets[i]:offsets[i + 1]] = table[i, pos // page] * page + pos % page
    t["positions"], t["slots"] = torch.from_numpy(positions).cuda(), torch.from_numpy(slots).cuda()
    return t


def _tables(rows: int, head_dim: int):
    inv = THETA ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv[None, :]
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def _inputs(case: dict, seed: int) -> dict:
    """The named inputs of a case and the buffers that its pass writes."""
    t = _layout(case, seed)
    if case["op"] == "plan":
        spans = t["spans"]
        return {"cached": _int([c for c, _ in spans]), "fresh": _int([n for _, n in spans]),
                "free": t["free"], "table": t["table_before"], "pages": t["pages"],
                "offsets": torch.zeros(len(spans) + 1, dtype=torch.int32, device="cuda"),
                "context": torch.zeros(len(spans), dtype=torch.int32, device="cuda"),
                "slots": torch.zeros(t["tokens"], dtype=torch.int32, device="cuda"),
                "positions": torch.zeros(t["tokens"], dtype=torch.int32, device="cuda"),
                "taken": torch.zeros(1, dtype=torch.int32, device="cuda")}
    rng = torch.Generator(device="cuda")
    rng.manual_seed(seed)
    dtype = DTYPES[case["dtype"]][0]
    qh, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=rng)

    t["out"] = torch.zeros((t["tokens"], qh, d), dtype=dtype, device="cuda")
    if case["op"] != "paged":
        # the rows of one projection: all query heads, then the key and the value heads
        t["rows"] = normal(t["tokens"], (qh + 2 * kvh) * d)
    else:
        t["q"] = normal(t["tokens"], qh, d)
    if case["op"] != "packed":
        t["k_pages"] = normal(t["pages"], kvh, case["page"], d)
        t["v_pages"] = normal(t["pages"], kvh, case["page"], d)
    if case["op"] == "append":
        t["cos"], t["sin"] = _tables(t["max_blocks"] * case["page"], d)
    return t


def prepare(case: dict, seed: int) -> dict:
    state = {"case": case, "t": _inputs(case, seed)}
    torch.cuda.synchronize()
    return state


def _split(case: dict, rows: torch.Tensor):
    """The [T, heads, D] views of projection rows: Q, K, V."""
    qh, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    heads = rows.view(rows.shape[0], qh + 2 * kvh, d)
    return heads[:, :qh], heads[:, qh:qh + kvh], heads[:, qh + kvh:]


# -------------------------------------------------------------- plain forms


def _owner(offsets: torch.Tensor, tokens: int):
    """Each token's request, its place within it, and whether it is one's at all."""
    at = torch.arange(tokens, device=offsets.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), at.int(), right=True)
    live = seq < offsets.numel() - 1
    seq = seq.clamp(max=offsets.numel() - 2)
    return seq, at - offsets[seq], live


def _plain_plan(case, t):
    page = case["page"]
    cached, fresh = t["cached"].long(), t["fresh"].long()
    blocks = t["table"].shape[1]
    have = ((cached + page - 1) // page).clamp(max=blocks)
    whole = ((cached + fresh + page - 1) // page).clamp(max=blocks)
    need = whole - have
    t["offsets"][1:] = torch.cumsum(fresh, 0)
    t["context"].copy_(cached + fresh)
    t["taken"].copy_(need.sum())
    column = torch.arange(blocks, device="cuda")[None]
    take = (torch.cumsum(need, 0) - need)[:, None] + column - have[:, None]
    new = (column >= have[:, None]) & (column < whole[:, None])
    given = t["free"][take.clamp(0, t["free"].numel() - 1)]
    given = torch.where(take < t["free"].numel(), given, NONE)
    t["table"].copy_(torch.where(new, given, t["table"]))
    seq, at, live = _owner(t["offsets"], t["slots"].numel())
    pos = cached[seq] + at
    entry = t["table"][seq, (pos // page).clamp(0, blocks - 1)].long()
    live = live & (pos // page < blocks) & (entry >= 0) & (entry < t["pages"])
    t["slots"].copy_(torch.where(live, entry * page + pos % page, NONE))
    t["positions"].copy_(torch.where(live, pos, 0))
    return _planned(t)


def _planned(t):
    return {name: t[name] for name in ("table", "offsets", "context", "slots", "positions",
                                       "taken")}


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(case, t):
    q, k, v = _split(case, t["rows"])
    cos, sin = t["cos"][t["positions"]][:, None], t["sin"][t["positions"]][:, None]
    live = (t["slots"] >= 0)[:, None, None]
    t["out"].copy_(torch.where(live, _rotate(q, cos, sin).to(q.dtype), t["out"]))
    # a token without a slot repeats the first token's write
    slot = torch.where(t["slots"] >= 0, t["slots"], t["slots"][0])
    page, row = slot // case["page"], slot % case["page"]
    rotated = _rotate(k, cos, sin).to(k.dtype)
    t["k_pages"][page, :, row] = torch.where(live, rotated, rotated[:1])
    t["v_pages"][page, :, row] = torch.where(live, v, v[:1])
    return {"q": t["out"], "k_pages": t["k_pages"], "v_pages": t["v_pages"]}


def _plain_attend(case, t, q, k, v, context):
    """Causal attention of padded requests: q [T, QH, D], k and v [S, KVH, keys, D]."""
    qh, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    group, n, s = qh // kvh, t["max_queries"], t["sequences"]
    start, fresh = t["offsets"][:-1].long(), (t["offsets"][1:] - t["offsets"][:-1]).long()
    each = torch.arange(n, device="cuda")
    padded = q[(start[:, None] + each[None]).clamp(max=q.shape[0] - 1)].float()
    padded = padded.view(s, n, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(s, kvh, group * n, d)
    scores = torch.matmul(padded, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    scores = scores.view(s, kvh, group, n, k.shape[2])
    last = (context.long() - fresh)[:, None] + each[None]
    hidden = torch.arange(k.shape[2], device="cuda")[None, None] > last[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores.div_(scores.sum(-1, keepdim=True))
    found = torch.matmul(scores.view(s, kvh, group * n, k.shape[2]), v)
    found = found.view(s, kvh, group, n, d).permute(0, 3, 1, 2, 4).reshape(s, n, qh, d)
    seq, at, live = _owner(t["offsets"], q.shape[0])
    found = found[seq, at.clamp(0, n - 1)].to(q.dtype)
    t["out"].copy_(torch.where(live[:, None, None], found, t["out"]))
    return {"out": t["out"]}


def _plain_packed(case, t):
    q, k, v = _split(case, t["rows"])
    each = torch.arange(t["max_queries"], device="cuda")
    rows = (t["offsets"][:-1].long()[:, None] + each[None]).clamp(max=t["tokens"] - 1)
    fresh = t["offsets"][1:] - t["offsets"][:-1]
    return _plain_attend(case, t, q, k[rows].transpose(1, 2).float().contiguous(),
                         v[rows].transpose(1, 2).float().contiguous(), fresh)


def _plain_paged(case, t):
    blocks = -(-t["max_context"] // case["page"])
    ids = t["table"][:, :blocks].clamp(min=0).long()
    s, kvh, d = t["sequences"], case["kv_heads"], case["head_dim"]
    k = t["k_pages"][ids].float().transpose(1, 2).reshape(s, kvh, blocks * case["page"], d)
    v = t["v_pages"][ids].float().transpose(1, 2).reshape(s, kvh, blocks * case["page"], d)
    return _plain_attend(case, t, t["q"], k, v, t["context"])


# --------------------------------------------------------- the framework's

_context = None


def _framework():
    """The process's one context, as a program on one GPU holds it.  Torch works on its stream
    from then on: what writes the inputs, the calls and what reads their outputs run in the
    order in which the program issues them."""
    global _context
    if _context is None:
        from rustllm_amd import abi

        _context = abi.Context(0)
        stream = torch.cuda.ExternalStream(_context.lib.rl_context_stream(_context.handle))
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
    return _context


def _buffers(state: dict) -> dict:
    """The library's view of the state's device memory (an rl_buffer owns nothing)."""
    if "buffers" not in state:
        from rustllm_amd import abi

        ctx, t, case = _framework(), state["t"], state["case"]
        names = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.uint32}

        def wrap(x, elements):
            raw = abi.RlBuffer(x.data_ptr(), elements, elements * x.element_size())
            return abi.DeviceBuffer(ctx, raw, names[x.dtype], tuple(x.shape))

        b = {name: wrap(x, x.numel()) for name, x in t.items() if isinstance(x, torch.Tensor)}
        if "rows" in t:
            for name, x in zip("qkv", _split(case, t["rows"])):
                reach = sum((n - 1) * m for n, m in zip(x.shape, x.stride())) + 1
                b[name] = (wrap(x, reach), tuple(x.shape), tuple(x.stride()))
        state["buffers"] = b
    return state["buffers"]


def _own_plan(ctx, case, t, b):
    ctx.paged_plan(b["cached"], b["fresh"], b["free"], b["table"], case["page"], t["pages"],
                   b["offsets"], b["context"], b["slots"], b["positions"], b["taken"])
    return _planned(t)


def _own_append(ctx, case, t, b):
    ctx.qkv_rope_paged_append(b["q"], b["k"], b["v"], b["cos"], b["sin"], b["positions"],
                              b["slots"], b["k_pages"], b["v_pages"], b["out"])
    return {"q": t["out"], "k_pages": t["k_pages"], "v_pages": t["v_pages"]}


def _own_packed(ctx, case, t, b):
    ctx.packed_attention(b["q"], b["k"], b["v"], b["offsets"], 1.0 / math.sqrt(case["head_dim"]),
                         t["max_queries"], b["out"])
    return {"out": t["out"]}


def _own_paged(ctx, case, t, b):
    ctx.paged_attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["offsets"], b["context"],
                        1.0 / math.sqrt(case["head_dim"]), t["max_queries"], t["max_context"],
                        b["out"])
    return {"out": t["out"]}


PLAIN = {"plan": _plain_plan, "append": _plain_append, "packed": _plain_packed,
         "paged": _plain_paged}
OWN = {"plan": _own_plan, "append": _own_append, "packed": _own_packed, "paged": _own_paged}


def run(state: dict) -> dict:
    """One pass.  With `own`, on the context's stream, which is torch's current one after the
    first pass; a caller that turns torch to another stream orders the two."""
    case, t = state["case"], state["t"]
    if own:
        return OWN[case["op"]](_framework(), case, t, _buffers(state))
    return PLAIN[case["op"]](case, t)


# -------------------------------------------------------------------- work


def work(case: dict) -> dict:
    spans = _spans(case)
    tokens = sum(n for _, n in spans)
    if case["op"] == "plan":
        page = case["page"]
        new = sum(-(-(c + n) // page) - -(-c // page) for c, n in spans)
        # lengths in, offsets, contexts, slots and positions out, new entries read and written,
        # one table entry for each new token on an old page
        old = sum(min(n, -c % page) > 0 for c, n in spans)
        return {"bytes": 4 * (4 * len(spans) + 2 * (tokens + case["padding"]) + 2 * new + old),
                "flops": 0}
    es = DTYPES[case["dtype"]][1]
    qh, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (qh + 2 * kvh) * d * es + tokens * (4 * d + 8), "flops": 0}
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in spans)
    keys = sum(c + n for c, n in spans)
    numel = 2 * tokens * qh * d + 2 * keys * kvh * d
    entries = sum(-(-(c + n) // case["page"]) for c, n in spans) if case["op"] == "paged" else 0
    return {"bytes": numel * es + 4 * (entries + 2 * len(spans)), "flops": 4 * d * qh * pairs}


# ------------------------------------------------------------------- exact


def _exact_plan(case, t):
    """Request by request, as a server on the host would keep its books."""
    page, pages = case["page"], t["pages"]
    cached, fresh, free = (t[name].tolist() for name in ("cached", "fresh", "free"))
    table = t["table"].cpu().numpy().copy()
    offsets, slots, positions, taken = [0], [], [], 0
    for i, (c, n) in enumerate(zip(cached, fresh)):
        for at in range(-(-c // page), -(-(c + n) // page)):
            if at < table.shape[1]:
                table[i, at] = free[taken] if taken < len(free) else NONE
                taken += 1
        for pos in range(c, c + n):
            entry = table[i, pos // page] if pos // page < table.shape[1] else NONE
            held = 0 <= entry < pages
            slots.append(int(entry) * page + pos % page if held else NONE)
            positions.append(pos if held else 0)
        offsets.append(offsets[-1] + n)
    room = t["slots"].numel() - len(slots)
    return {"table": _int(table), "offsets": _int(offsets),
            "context": _int([c + n for c, n in zip(cached, fresh)]),
            "slots": _int(slots + [NONE] * room), "positions": _int(positions + [0] * room),
            "taken": _int([taken])}


def _exact_append(case, t):
    qh, kvh, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rows = t["rows"].double()
    angle_cos, angle_sin = t["cos"].double(), t["sin"].double()
    got = {"q": t["out"].double(), "k_pages": t["k_pages"].double(),
           "v_pages": t["v_pages"].double()}
    keep = torch.nonzero(t["slots"] != NONE).flatten()
    at, where = t["positions"][keep].long(), t["slots"][keep].long()
    c, s = angle_cos[at].repeat(1, 2)[:, None], angle_sin[at].repeat(1, 2)[:, None]
    x = rows[keep].reshape(keep.numel(), qh + 2 * kvh, d)
    turned = torch.roll(x, d // 2, -1)  # each element's partner in the other half
    turned[..., :d // 2] *= -1.0
    rotated = x * c + turned * s
    got["q"][keep] = rotated[:, :qh]
    for h in range(kvh):
        got["k_pages"][where // page, h, where % page] = rotated[:, qh + h]
        got["v_pages"][where // page, h, where % page] = x[:, qh + kvh + h]
    return got


def _exact_attention(case, t):
    qh, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((t["tokens"], qh, d), dtype=torch.float64, device="cuda")
    first = 0
    for i, (c, n) in enumerate(t["spans"]):
        if n == 0:
            continue
        if case["op"] == "packed":
            rows = t["rows"][first:first + n].reshape(n, qh + 2 * kvh, d)
            q, k, v = rows[:, :qh], rows[:, qh:qh + kvh], rows[:, qh + kvh:]
        else:
            at = torch.arange(c + n, device="cuda")
            page, row = t["table"][i].long()[at // case["page"]], at % case["page"]
            q, k, v = t["q"][first:first + n], t["k_pages"][page, :, row], t["v_pages"][page, :, row]
        seen = torch.ones(n, c + n, dtype=torch.bool, device="cuda").tril(c)
        for h in range(qh):
            g = h * kvh // qh
            s = torch.mm(q[:, h].double(), k[:, g].double().t().contiguous()) / math.sqrt(d)
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            out[first:first + n, h] = torch.mm(p, v[:, g].double().contiguous())
        first += n
    return {"out": out}


def exact(case: dict, seed: int) -> dict:
    t = _inputs(case, seed)
    if case["op"] == "plan":
        return _exact_plan(case, t)
    return _exact_append(case, t) if case["op"] == "append" else _exact_attention(case, t)
