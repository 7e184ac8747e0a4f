"""Serving a batch on the GPU: the plan of a step, the append into pages, and
attention over pages and over packed prompts.

The plan is compared with a host's bookkeeping, exactly; the append with
rl_rope_* bit for bit; attention with float64 attention of every request by
itself under the forward error bound of its roundings (helpers.attention_bound,
"f32" / "f16_fused").  Whatever a call must not read holds NaN: page rows past
a request's context, pages of no request, table entries past its pages.
"""

import ctypes

import numpy as np
import pytest

from helpers import assert_bitexact, attention_bound
from rustllm_amd import abi, synth

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
DTYPES = [np.float32, np.float16]


class View(abi.DeviceBuffer):
    """Part of another buffer's memory: owns nothing."""

    def release(self):
        pass


def normal(shape, dtype, *key):
    return synth.normal(synth.seed_for("paged", *key), shape).astype(dtype)


# -------------------------------------------------------------------- plan


def plan_on_host(cached, fresh, free, table, page, pages, tokens):
    table = table.copy()
    offsets, slots, positions, taken = [0], [], [], 0
    blocks = table.shape[1]
    for i, (c, n) in enumerate(zip(cached, fresh)):
        have, whole = min(-(-c // page), blocks), min(-(-(c + n) // page), blocks)
        for b in range(have, whole):
            table[i, b] = free[taken + b - have] if taken + b - have < len(free) else NONE
        taken += whole - have
        for pos in range(c, c + n):
            entry = int(table[i, pos // page]) if pos // page < blocks else NONE
            slots.append(entry * page + pos % page if entry < pages else NONE)
            positions.append(pos if entry < pages else 0)
        offsets.append(offsets[-1] + n)
    room = tokens - len(slots)
    return {"table": table, "offsets": np.array(offsets, np.uint32),
            "context": np.array(cached, np.uint32) + np.array(fresh, np.uint32),
            "slots": np.array(slots + [NONE] * room, np.uint32),
            "positions": np.array(positions + [0] * room, np.uint32),
            "taken": np.array([taken], np.uint32)}


def run_plan(ctx, cached, fresh, free, table, page, pages, tokens):
    u32 = lambda v: ctx.upload(np.array(v, np.uint32))
    dt = u32(table)
    ctx.begin()
    got = ctx.paged_plan(u32(cached), u32(fresh), u32(free), dt, page, pages, tokens=tokens)
    ctx.finish()
    names = ("offsets", "context", "slots", "positions", "taken")
    return {**{n: b.numpy() for n, b in zip(names, got)}, "table": dt.numpy()}


def batch_of(rng, requests, longest, page, blocks, chunk=1):
    cached = [int(c) for c in rng.integers(0, longest + 1, requests)]
    fresh = [int(n) for n in rng.integers(0, chunk + 1, requests)]
    cached = [min(c, blocks * page - n) for c, n in zip(cached, fresh)]
    held = [-(-c // page) for c in cached]
    pages = sum(held) + sum(-(-(c + n) // page) for c, n in zip(cached, fresh)) + 3
    ids = rng.permutation(pages)
    table = np.full((requests, blocks), NONE, np.uint32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    return cached, fresh, ids[at:], table, pages


@pytest.mark.parametrize("requests,longest,page,blocks,chunk", [
    (1, 0, 16, 4, 1), (1, 63, 16, 4, 1), (3, 40, 1, 64, 5), (48, 500, 16, 40, 1),
    (257, 90, 8, 30, 40), (1023, 30, 4, 9, 2), (1024, 30, 4, 9, 2), (1025, 30, 4, 9, 2),
    (3000, 200, 64, 5, 30), (9, 4000, 128, 64, 3000), (2100, 0, 32, 1, 32)])
def test_plan_matches_a_hosts_books(ctx, requests, longest, page, blocks, chunk):
    rng = np.random.default_rng(requests * 7 + chunk)
    cached, fresh, free, table, pages = batch_of(rng, requests, longest, page, blocks, chunk)
    tokens = sum(fresh) + int(rng.integers(1, 40))
    got = run_plan(ctx, cached, fresh, free, table, page, pages, tokens)
    for name, want in plan_on_host(cached, fresh, free, table, page, pages, tokens).items():
        assert np.array_equal(got[name], want), name


def test_plan_when_pages_or_table_rows_run_out(ctx):
    """Tokens without a page have no slot; the count of pages says so; a free
    entry outside the pool counts as none; rows are cut at max_blocks."""
    page, pages, blocks = 8, 20, 3
    cached, fresh = [8, 3, 0, 20], [9, 30, 8, 2]
    table = np.full((4, blocks), NONE, np.uint32)
    table[0, 0], table[1, 0], table[3] = 7, 9, [1, 25, 2]  # 25: outside the pool
    for free in ([4, 99, 5], [], [4, 5, 6, 8, 10, 11]):
        want = plan_on_host(cached, fresh, free, table, page, pages, 60)
        dfree = np.array(free, np.uint32) if free else None
        u32 = lambda v: ctx.upload(np.array(v, np.uint32))
        dt = u32(table)
        nothing = View(ctx, abi.RlBuffer(None, 0, 0), np.uint32, (0,))
        got = ctx.paged_plan(u32(cached), u32(fresh), nothing if dfree is None else u32(dfree),
                             dt, page, pages, tokens=60)
        ctx.finish()
        names = ("offsets", "context", "slots", "positions", "taken")
        for name, b in [*zip(names, got), ("table", dt)]:
            assert np.array_equal(b.numpy(), want[name]), (free, name)
        assert want["taken"][0] == 2 + 2 + 1 + 0


def test_plan_sums_stop_at_their_type(ctx):
    """Lengths whose sums pass 32 bits saturate; tokens past the rows are not planned."""
    big = 0xFFFFFFF0
    got = run_plan(ctx, [5, big, 1], [3, 100, big], [0, 1], np.full((3, 2), NONE, np.uint32), 16,
                   9, 8)
    assert list(got["offsets"]) == [0, 3, 103, 0xFFFFFFFF]
    assert list(got["context"]) == [8, 0xFFFFFFFF, 0xFFFFFFF1]
    # request 0 has no page in its table, request 1's position lies past it
    assert list(got["slots"]) == [NONE] * 8 and list(got["positions"]) == [0] * 8


# ------------------------------------------------------------------ append


def rotated(ctx, x, cos, sin, position):
    """rl_rope_* of one token's [heads, D] at its position."""
    got = ctx.rope(ctx.upload(x[None, :, None, :]), ctx.upload(cos), ctx.upload(sin),
                   int(position))
    return got.numpy()[0, :, 0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,qh,kvh,d,page,layout", [
    (1, 15, 5, 64, 16, "rows"), (7, 9, 3, 64, 16, "rows"), (33, 4, 4, 128, 32, "heads"),
    (5, 3, 1, 80, 8, "rows"), (6, 2, 2, 20, 4, "rows"), (9, 2, 1, 2, 1, "rows"),
    (4, 6, 2, 64, 16, "odd"), (1100, 32, 8, 64, 16, "rows"), (1, 1, 1, 512, 1, "rows")])
def test_append_matches_rope_bit_for_bit(ctx, dtype, tokens, qh, kvh, d, page, layout):
    """Q, K and V of every token where they belong; skipped tokens and all
    other rows keep what they held."""
    key = (tokens, qh, kvh, d, page, layout)
    heads = qh + 2 * kvh
    x = normal((tokens, heads, d), dtype, "append", *key)
    rng = np.random.default_rng(tokens)
    pages, table_rows = -(-tokens // page) + 3, 50
    slots = rng.permutation(pages * page)[:tokens].astype(np.uint32)
    positions = rng.integers(0, table_rows, tokens).astype(np.uint32)
    skipped = []
    if tokens > 4:  # without a slot, past the pool, past the tables
        slots[1], slots[2], positions[3] = NONE, pages * page, table_rows
        skipped = [1, 2, 3]
    angle = np.arange(table_rows)[:, None] * 100.0 ** (-np.arange(0, d, 2) / d)[None]
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    if layout == "heads":  # [heads, tokens, D] in memory
        stored, strides = np.ascontiguousarray(x.transpose(1, 0, 2)), (d, tokens * d, 1)
        at = lambda h: h * tokens * d
    else:
        pad = 3 if layout == "odd" else 0  # rows off the 16-byte grid
        stored = np.zeros((tokens, heads * d + pad), dtype)
        stored[:, :heads * d] = x.reshape(tokens, -1)
        strides = (heads * d + pad, d, 1)
        at = lambda h: h * d
    dx = ctx.upload(stored)

    def view(first, n):
        start = at(first)
        reach = (tokens - 1) * strides[0] + (n - 1) * strides[1] + d
        es = dx.dtype.itemsize
        raw = abi.RlBuffer(dx.ptr + start * es, reach, reach * es)
        return View(ctx, raw, dtype, (reach,)), (tokens, n, d), strides

    kp = normal((pages, kvh, page, d), dtype, "kp", *key)
    vp = normal((pages, kvh, page, d), dtype, "vp", *key)
    q0 = normal((tokens, qh, d), dtype, "q0", *key)
    dk, dv, dq = ctx.upload(kp), ctx.upload(vp), ctx.upload(q0)
    ctx.begin()
    ctx.qkv_rope_paged_append(view(0, qh), view(qh, kvh), view(qh + kvh, kvh), ctx.upload(cos),
                              ctx.upload(sin), ctx.upload(positions), ctx.upload(slots), dk, dv,
                              dq)
    ctx.finish()
    check = range(tokens) if tokens < 50 else rng.choice(tokens, 20, replace=False)
    got_q = dq.numpy()
    want_k, want_v, got_k, got_v = kp.copy(), vp.copy(), dk.numpy(), dv.numpy()
    for t in range(tokens):
        if t in skipped:
            assert_bitexact(got_q[t], q0[t], f"skipped token {t}")
            continue
        page_at, row = slots[t] // page, slots[t] % page
        want_v[page_at, :, row] = x[t, qh + kvh:]
        if t not in check:
            want_k[page_at, :, row] = got_k[page_at, :, row]
            continue
        turned = rotated(ctx, x[t, :qh + kvh], cos, sin, positions[t])
        assert_bitexact(got_q[t], turned[:qh], f"Q of token {t}")
        want_k[page_at, :, row] = turned[qh:]
    assert_bitexact(got_k, want_k, "K pages")
    assert_bitexact(got_v, want_v, "V pages")


# --------------------------------------------------------------- attention


class Batch:
    """Requests of (cached, new) tokens over shuffled pages of NaN where
    nothing may be read."""

    def __init__(self, spans, qh, kvh, d, page, dtype, key, spare=3, sigma=1.0, padding=0,
                 blocks=None):
        self.spans, self.qh, self.kvh, self.d, self.page = spans, qh, kvh, d, page
        rng = np.random.default_rng(synth.seed_for(*key) & 0xFFFF)
        whole = [-(-(c + n) // page) for c, n in spans]
        self.pages = sum(whole) + spare
        self.blocks = blocks or max(max(whole), 1)
        ids = rng.permutation(self.pages)
        self.table = np.full((len(spans), self.blocks), NONE, np.uint32)
        self.offsets = np.cumsum([0] + [n for _, n in spans]).astype(np.uint32)
        self.context = np.array([c + n for c, n in spans], np.uint32)
        self.tokens = max(int(self.offsets[-1]) + padding, 1)
        self.q = (sigma * normal((self.tokens, qh, d), np.float32, "q", *key)).astype(dtype)
        self.kp = np.full((self.pages, kvh, page, d), np.nan, dtype)
        self.vp = np.full((self.pages, kvh, page, d), np.nan, dtype)
        self.k, self.v = [], []
        at = 0
        for i, (w, keys) in enumerate(zip(whole, self.context)):
            self.table[i, :w] = ids[at:at + w]
            at += w
            k = normal((int(keys), kvh, d), dtype, "k", i, *key)
            v = normal((int(keys), kvh, d), dtype, "v", i, *key)
            pos = np.arange(keys)
            self.kp[self.table[i, pos // page], :, pos % page] = k
            self.vp[self.table[i, pos // page], :, pos % page] = v
            self.k.append(k)
            self.v.append(v)
        self.scale = 1.0 / np.sqrt(d)
        self.max_queries = max(max(n for _, n in spans), 1)
        self.max_context = max(int(self.context.max()), 1)

    def upload(self, ctx):
        names = ("q", "kp", "vp", "table", "offsets", "context")
        return {n: ctx.upload(getattr(self, n)) for n in names}

    def run(self, ctx, **kw):
        b = self.upload(ctx)
        out = ctx.upload(np.full(self.q.shape, 7.0, self.q.dtype))
        ctx.begin()
        ctx.paged_attention(b["q"], b["kp"], b["vp"], b["table"], b["offsets"], b["context"],
                            self.scale, kw.get("max_queries", self.max_queries),
                            kw.get("max_context", self.max_context), out)
        ctx.finish()
        return out.numpy()

    def expect(self, i):
        """(rows, exact, bound) of request i, [QH, n, D]."""
        n = self.spans[i][1]
        rows = slice(int(self.offsets[i]), int(self.offsets[i]) + n)
        q = self.q[rows].transpose(1, 0, 2)[None]
        k, v = self.k[i].transpose(1, 0, 2)[None], self.v[i].transpose(1, 0, 2)[None]
        kind = "f16_fused" if self.q.dtype == np.float16 else "f32"
        exact, bound = attention_bound(q, k, v, self.scale, self.spans[i][0], None, kind)
        return rows, exact[0], bound[0]

    def check(self, got, skip=()):
        for i, (c, n) in enumerate(self.spans):
            if n == 0 or i in skip:
                continue
            rows, exact, bound = self.expect(i)
            have = got[rows].astype(np.float64).transpose(1, 0, 2)
            assert np.isfinite(have).all(), f"request {i} {c, n}: non-finite output"
            err = np.abs(have - exact)
            worst = np.unravel_index(np.argmax(err / bound), err.shape)
            assert np.all(err <= bound), (f"request {i} {c, n}: error {err[worst]:.3g} > bound "
                                          f"{bound[worst]:.3g} at {worst}")
        assert np.all(got[int(self.offsets[-1]):] == 7.0), "rows behind the last request"


# spans, q heads, KV heads, head size, page
PAGED = [
    ([(0, 1)], 15, 5, 64, 16),                      # the first token of all
    ([(1535, 1)], 15, 5, 64, 16),                   # one user
    ([(0, 1), (0, 0), (1, 1), (63, 1), (64, 1), (65, 1), (255, 1), (256, 1), (700, 1)],
     9, 3, 64, 16),
    ([(2000, 1), (17, 1), (999, 1)], 32, 8, 128, 16),
    ([(300, 1), (0, 0), (5, 1)], 8, 8, 128, 64),
    ([(1000, 2), (30, 3), (0, 4), (513, 1)], 12, 3, 64, 32),  # drafts of a few tokens
    ([(100, 1), (260, 1)], 12, 3, 96, 16),
    ([(100, 1), (260, 3)], 8, 8, 80, 128),
    ([(40, 1), (300, 2)], 15, 5, 32, 16),
    ([(700, 1), (3, 1)], 16, 1, 64, 16),            # 16 rows of one KV head
    ([(700, 1), (3, 2)], 32, 1, 64, 16),            # 32 rows and more
    ([(0, 37), (10, 129), (400, 1), (0, 0), (250, 64)], 9, 3, 64, 16),
    ([(500, 300), (0, 200), (90, 1), (1200, 1)], 15, 5, 64, 32),
    ([(64, 128), (200, 33)], 32, 8, 128, 16),
    ([(30, 150), (1, 1)], 8, 8, 96, 64),
    ([(100, 50), (0, 7)], 4, 2, 80, 16),
    ([(90, 100), (300, 1)], 6, 3, 32, 8),
    ([(33, 20), (7, 1)], 4, 4, 48, 1),              # pages of one position
    ([(33, 20), (7, 1)], 4, 2, 40, 2),
    ([(3, 5), (20, 1)], 2, 1, 200, 16),             # head sizes of the row kernel
    ([(3, 5), (20, 1)], 2, 1, 7, 16),
    ([(3, 2), (300, 1)], 2, 2, 512, 16),
    ([(2900, 600), (5, 1)], 8, 2, 64, 64),          # few tiles over many keys
    ([(3500, 130)], 4, 1, 128, 32),
    # enough rows for the wide tiles, and for ordering them by length
    ([(100, 300), (0, 310), (700, 290), (5, 1), (33, 300)], 32, 8, 64, 16),
    ([(100, 300), (0, 310), (5, 2), (300, 450)], 32, 8, 128, 32),
    ([(70, 500), (0, 310), (5, 1), (300, 300)], 32, 8, 96, 16),
    ([(70, 500), (0, 310), (5, 3), (300, 300)], 32, 8, 32, 64),
    ([(40, 200), (0, 310), (5, 1), (1300, 290)], 15, 5, 64, 16),
    ([(40, 300), (0, 310), (5, 1), (1300, 290)], 15, 5, 64, 16),
    *[([(100, 300), (0, 310), (700, 290), (5, 1), (33, 300)], 64, 16, d, 16)
      for d in (64, 56, 32, 24)],
    *[([(100, 300), (0, 310), (5, 2), (300, 450)], 32, 8, d, 32) for d in (112, 80)],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_attention_within_float64_bound(ctx, dtype, case):
    spans, qh, kvh, d, page = PAGED[case]
    b = Batch(spans, qh, kvh, d, page, dtype, ("paged", case), padding=case % 3)
    b.check(b.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_of_many_requests(ctx, dtype):
    """More requests than a wave has lanes, most of them short, some idle, one long."""
    rng = np.random.default_rng(3)
    spans = [(int(c), int(n)) for c, n in zip(rng.integers(0, 200, 150), rng.integers(0, 2, 150))]
    spans[77], spans[149] = (5000, 1), (600, 1)
    b = Batch(spans, 6, 2, 64, 16, dtype, ("many",), padding=2)
    b.check(b.run(ctx))
    spans[3], spans[140] = (10, 70), (300, 200)  # and chunks among them
    b = Batch(spans, 6, 2, 64, 16, dtype, ("many chunks",))
    b.check(b.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests,chunk", [(64, 2), (65, 2), (257, 2), (257, 40), (1500, 2),
                                            (5000, 1)])
def test_paged_attention_finds_its_requests(ctx, dtype, requests, chunk):
    """Many requests of a few keys, runs of idle ones and a long one among them."""
    rng = np.random.default_rng(requests + chunk)
    spans = [(int(c), int(n)) for c, n in zip(rng.integers(0, 40, requests),
                                              rng.integers(0, chunk + 1, requests))]
    idle = slice(requests // 5, requests // 5 + 100 if requests > 200 else requests // 5 + 9)
    spans[idle] = [(c, 0) for c, _ in spans[idle]]
    spans[requests // 2], spans[-1] = (3000, 1), (0, 1)
    b = Batch(spans, 6, 2, 64, 16, dtype, ("requests", requests, chunk), padding=1)
    b.check(b.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_bounds_may_be_loose(ctx, dtype):
    """max_queries, max_context and the table row far above what the batch has."""
    b = Batch([(100, 1), (7, 1), (40, 1)], 9, 3, 64, 16, dtype, ("loose",), blocks=4096)
    b.check(b.run(ctx, max_queries=500, max_context=4096 * 16))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_past_max_queries_are_left(ctx, dtype):
    """A request of more rows than max_queries: its first ones as they are, the rest
    not written; the same for packed prompts."""
    for most in (2, 40):
        b = Batch([(100, 60), (7, 1)], 6, 2, 64, 16, dtype, ("most", most))
        got = b.run(ctx, max_queries=most)
        _, exact, bound = b.expect(0)
        err = np.abs(got[:most].astype(np.float64).transpose(1, 0, 2) - exact[:, :most])
        assert np.all(err <= bound[:, :most])
        assert np.all(got[most:60] == 7.0)
        b.check(got, skip=(0,))


def test_one_workspace_serves_batches_of_many_sizes(ctx):
    """Calls of different numbers of requests and KV heads take turns with one
    workspace (its counters are zero again after each)."""
    workspace = ctx.paged_workspace(40, 8)
    batches = [Batch([(900, 1)] * n, qh, kvh, 64, 16, np.float16, ("turns", n, kvh))
               for n, qh, kvh in ((40, 8, 8), (1, 6, 2), (7, 15, 5), (40, 4, 1))]
    held = [(b, b.upload(ctx)) for b in batches]
    for _ in range(3):
        for b, d in held:
            out = ctx.upload(np.full(b.q.shape, 7.0, np.float16))
            ctx.paged_attention(d["q"], d["kp"], d["vp"], d["table"], d["offsets"], d["context"],
                                b.scale, 1, b.max_context, out, workspace)
            ctx.finish()
            b.check(out.numpy())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_paged_attention_marks_what_is_not_there(ctx, dtype, n):
    """Rows that see a key of a page outside the pool are NaN, so is a request
    past max_context; rows that see no key are zeros; the rest is untouched by it."""
    spans = [(200, n), (150, n), (90, n), (64, n)]
    b = Batch(spans, 6, 2, 64, 16, dtype, ("bad", n))
    # request 0's last page, which only its last rows see; request 1's first
    last = (200 + n - 1) // 16
    b.table[0, last], b.table[1, 0] = b.pages, NONE
    got = b.run(ctx)
    first_bad = last * 16 - 200  # the first row of request 0 that sees position last * 16
    rows = got[:n]
    if first_bad > 0:
        kept, b.spans[0] = b.spans[0], (200, n)
        _, exact, bound = b.expect(0)
        err = np.abs(rows[:first_bad].astype(np.float64).transpose(1, 0, 2) - exact[:, :first_bad])
        assert np.all(err <= bound[:, :first_bad])
    assert np.isnan(rows[max(first_bad, 0):]).all()
    assert np.isnan(got[n:2 * n]).all()
    b.check(got, skip=(0, 1))
    # a context past the bound, and one smaller than its rows
    b = Batch(spans, 6, 2, 64, 16, dtype, ("bad context", n))
    b.context[0] = b.max_context + 1
    b.context[2] = n // 2
    got = b.run(ctx)
    assert np.isnan(got[:n]).all()
    early = n - n // 2
    assert np.all(got[2 * n:2 * n + early] == 0.0)
    if n > 1:
        b.spans[2], b.k[2], b.v[2] = (early - n, n), b.k[2][:n // 2], b.v[2][:n // 2]
        q = b.q[2 * n + early:3 * n].transpose(1, 0, 2)[None]
        kind = "f16_fused" if dtype == np.float16 else "f32"
        exact, bound = attention_bound(q, b.k[2].transpose(1, 0, 2)[None],
                                       b.v[2].transpose(1, 0, 2)[None], b.scale, 0, None, kind)
        have = got[2 * n + early:3 * n].astype(np.float64).transpose(1, 0, 2)
        assert np.all(np.abs(have - exact[0]) <= bound[0])
    b.check(got, skip=(0, 2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_row_ranges_are_clamped_to_the_rows(ctx, dtype):
    """Offsets past the rows, or falling, reach no other memory; requests whose
    ranges are sound keep their results."""
    b = Batch([(50, 3), (20, 2), (9, 4)], 6, 2, 64, 16, dtype, ("clamped",))
    b.offsets[3] = 4000
    got = b.run(ctx)
    assert np.isfinite(got).all()
    b.offsets[3] = 9
    b.check(got)
    b.offsets[1:] = [3, 2, 0xFFFFFFFF]
    got = b.run(ctx)
    b.spans, b.offsets = b.spans[:1], np.array([0, 3], np.uint32)
    rows, exact, bound = b.expect(0)
    err = np.abs(got[:2].astype(np.float64).transpose(1, 0, 2) - exact[:, :2])
    assert np.all(err <= bound[:, :2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 900), (3, 300), (200, 40)])
def test_values_behind_a_row_do_not_reach_it(ctx, dtype, n, c):
    """Infinite and NaN keys and values of a request's later tokens reach only
    the rows that see them; neither do those of other requests."""
    b = Batch([(c, n), (c, n)], 6, 2, 64, 16, dtype, ("behind", n))
    got = b.run(ctx)
    b.check(got)
    last = c + n - 1
    at = b.table[0, last // 16], slice(None), last % 16
    for k, v in [(np.nan, np.inf), (1.0, np.nan), (np.inf, 0.0)]:
        b.kp[at], b.vp[at] = k, v
        again = b.run(ctx)
        rows, exact, bound = b.expect(0)
        err = np.abs(again[:n - 1].astype(np.float64).transpose(1, 0, 2) - exact[:, :n - 1])
        assert np.all(err <= bound[:, :n - 1])
        assert not np.isfinite(again[n - 1]).all()
        assert_bitexact(again[n:], got[n:], "the other request")


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_of_wide_scores(ctx, dtype):
    """Large queries: softmax weights that differ by e^80 and more."""
    b = Batch([(700, 1), (300, 90), (90, 2)], 6, 2, 64, 16, dtype, ("wide",), sigma=8.0)
    b.check(b.run(ctx))


def test_paged_attention_matches_the_contiguous_cache(ctx):
    """One request over pages against rl_attention_f16 over a [1, KVH, max, D] cache."""
    b = Batch([(900, 60)], 15, 5, 64, 16, np.float16, ("contiguous",))
    got = b.run(ctx)
    q = np.ascontiguousarray(b.q.transpose(1, 0, 2)[None])
    k = np.ascontiguousarray(b.k[0].transpose(1, 0, 2)[None])
    v = np.ascontiguousarray(b.v[0].transpose(1, 0, 2)[None])
    want = ctx.attention(ctx.upload(q), ctx.upload(k), ctx.upload(v), b.scale, 900).numpy()
    _, exact, bound = b.expect(0)
    both = np.abs(got.transpose(1, 0, 2).astype(np.float64) - want[0].astype(np.float64))
    assert np.all(both <= 2 * bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans", [[(400, 1), (30, 1)], [(100, 80), (600, 1)]])
def test_recorded_attention_follows_its_lengths(ctx, dtype, spans):
    """A recorded call, replayed with other lengths and tables in its buffers,
    eager work and waits between, against each replay's own batch."""
    first = Batch(spans, 6, 2, 64, 16, dtype, ("graph", len(spans), spans[0][1]), blocks=80)
    d = first.upload(ctx)
    out = ctx.upload(np.full(first.q.shape, 7.0, dtype))
    args = (d["q"], d["kp"], d["vp"], d["table"], d["offsets"], d["context"], first.scale, 90, 1200)
    ctx.paged_attention(*args, out)  # makes the workspace
    ctx.finish()
    ctx.capture_begin()
    ctx.paged_attention(*args, out)
    graph = ctx.capture_end()
    try:
        for turn, lengths in enumerate([spans, [(1, n) for _, n in spans],
                                        [(1100, n) for _, n in reversed(spans)], spans]):
            b = Batch(lengths, 6, 2, 64, 16, dtype, ("turn", turn, spans[0][1]), blocks=80,
                      spare=first.pages + 200)
            b.kp, b.vp = b.kp[:], b.vp[:]
            # the recorded pool is smaller: move the batch's pages into it
            used = np.unique(b.table[b.table != NONE])
            if used.size > first.pages:
                continue
            move = {int(p): j for j, p in enumerate(used)}
            kp, vp = np.full_like(first.kp, np.nan), np.full_like(first.vp, np.nan)
            for p, j in move.items():
                kp[j], vp[j] = b.kp[p], b.vp[p]
            table = np.array([[move.get(int(p), NONE) for p in row] for row in b.table], np.uint32)
            for name, value in (("q", b.q), ("kp", kp), ("vp", vp), ("table", table),
                                ("offsets", b.offsets), ("context", b.context)):
                ctx.copy(ctx.upload(value), d[name])
            ctx.finish()
            eager = ctx.upload(np.full(first.q.shape, 7.0, dtype))
            ctx.graph_launch(graph)
            ctx.paged_attention(*args, eager)
            ctx.finish()
            b.check(out.numpy())
            assert_bitexact(out.numpy(), eager.numpy(), "replay against eager")
    finally:
        ctx.graph_destroy(graph)


@pytest.mark.parametrize("dtype", DTYPES)
def test_recorded_steps_share_tables_pages_and_a_workspace(ctx, dtype):
    """Whole steps (plan, append, attention) as two graphs, one of single tokens
    and one of chunks, over the same requests: replayed in turn with the lengths
    and free pages of each step, against the same calls run eagerly on a copy of
    the tables and pools, bit for bit."""
    qh, kvh, d, page, blocks, pages, requests = 6, 2, 64, 16, 24, 60, 3
    heads = qh + 2 * kvh
    angle = np.arange(400)[:, None] * 100.0 ** (-np.arange(0, d, 2) / d)[None]
    cos, sin = (ctx.upload(f(angle).astype(np.float32)) for f in (np.cos, np.sin))
    state = [ctx.upload(np.full((requests, blocks), NONE, np.uint32)),
             *(ctx.upload(np.full((pages, kvh, page, d), np.nan, dtype)) for _ in range(2))]
    mirror = [ctx.clone(b) for b in state]
    u32 = lambda v: ctx.upload(np.array(v, np.uint32))

    class Step:
        def __init__(self, rows, chunk):
            self.rows, self.chunk = rows, chunk
            self.cached, self.fresh, self.free = u32([0] * 3), u32([0] * 3), u32([NONE] * pages)
            self.x = ctx.empty((rows, heads, d), dtype)
            self.planned = [ctx.empty((n,), np.uint32) for n in (requests + 1, requests, rows,
                                                                 rows, 1)]
            self.q, self.out = (ctx.empty((rows, qh, d), dtype) for _ in range(2))

        def run(self, state):
            table, dk, dv = state
            offsets, context, slots, positions, taken = self.planned
            ctx.paged_plan(self.cached, self.fresh, self.free, table, page, pages, offsets,
                           context, slots, positions, taken)
            views = [(View(ctx, abi.RlBuffer(self.x.raw.data + first * d * self.x.dtype.itemsize,
                                             self.x.len - first * d,
                                             self.x.byte_len - first * d * self.x.dtype.itemsize),
                           dtype, (self.x.len - first * d,)),
                      (self.rows, n, d), (heads * d, d, 1))
                     for first, n in ((0, qh), (qh, kvh), (qh + kvh, kvh))]
            ctx.qkv_rope_paged_append(*views, cos, sin, positions, slots, dk, dv, self.q)
            ctx.paged_attention(self.q, dk, dv, table, offsets, context, 0.125, self.chunk,
                                blocks * page, self.out)

        def results(self):
            return [b.numpy() for b in (*self.planned, self.out)]

    steps = {"one": Step(4, 2), "chunk": Step(90, 70)}
    graphs = {}
    for name, step in steps.items():
        step.run(state)  # three idle requests: makes the workspace, writes no page
        ctx.finish()
        ctx.capture_begin()
        step.run(state)
        graphs[name] = ctx.capture_end()
    cached, free = [0] * requests, list(np.random.default_rng(3).permutation(pages))
    try:
        for turn, (name, fresh) in enumerate([
                ("chunk", [60, 0, 7]), ("one", [1, 1, 1]), ("one", [1, 1, 2]),
                ("chunk", [1, 66, 1]), ("one", [0, 1, 1]), ("chunk", [70, 3, 17]),
                ("one", [1, 1, 1]), ("chunk", [0, 0, 0]), ("one", [2, 0, 1])]):
            step = steps[name]
            for buffer, value in ((step.cached, cached), (step.fresh, fresh),
                                  (step.free, free + [NONE] * (pages - len(free)))):
                ctx.copy(u32(value), buffer)
            ctx.copy(ctx.upload(normal((step.rows, heads, d), dtype, "step", turn)), step.x)
            ctx.copy(ctx.upload(np.full((step.rows, qh, d), 7.0, dtype)), step.out)
            ctx.graph_launch(graphs[name])
            ctx.finish()
            replayed = step.results()
            ctx.copy(ctx.upload(np.full((step.rows, qh, d), 7.0, dtype)), step.out)
            step.run(mirror)
            ctx.finish()
            for i, (got, want) in enumerate(zip(replayed, step.results())):
                assert_bitexact(got, want, f"turn {turn} output {i}")
            for got, want in zip(state, mirror):
                assert_bitexact(got.numpy(), want.numpy(), f"turn {turn} tables and pages")
            total = sum(fresh)
            assert np.isfinite(replayed[-1]).all() and np.all(replayed[-1][total:] == 7.0)
            assert total == 0 or not np.any(np.all(replayed[-1][:total] == 7.0, axis=(1, 2)))
            cached = [c + n for c, n in zip(cached, fresh)]
            free = free[int(replayed[4][0]):]
    finally:
        for graph in graphs.values():
            ctx.graph_destroy(graph)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_requests_share_a_prefix_behind_rows_of_none(ctx, dtype, n):
    """Two requests whose first pages are the same ones; the batch's first rows
    belong to no request."""
    b = Batch([(100, n), (130, 1), (99, n)], 6, 2, 64, 16, dtype, ("prefix", n), padding=5)
    b.table[1, :6] = b.table[0, :6]
    for x in (b.k, b.v):
        x[1][:96] = x[0][:96]
    b.offsets += 2
    got = b.run(ctx)
    b.check(got)
    assert np.all(got[:2] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_pools_past_4_gib(ctx, dtype, n):
    """Pages whose bytes and elements lie past 2^32 (two pools of 18 GiB, 36 in f32, of which a
    few pages are written and read)."""
    qh, kvh, d, page = 4, 2, 128, 64
    pages = 9 * (1 << 30) // (kvh * page * d)  # 9 Gi elements a pool
    spans = [(150, n), (70, n)]
    b = Batch(spans, qh, kvh, d, page, dtype, ("far", n))
    far = {int(p): pages - 1 - 100 * i for i, p in enumerate(b.table[b.table != NONE])}
    dk, dv = (ctx.empty((pages, kvh, page, d), dtype) for _ in range(2))
    tokens = int(b.context.sum())
    slots = np.concatenate([[far[int(b.table[i, p // page])] * page + p % page
                             for p in range(c + m)] for i, (c, m) in enumerate(spans)])
    ones, zeros = np.ones((1, d // 2), np.float32), np.zeros((1, d // 2), np.float32)
    k, v = np.concatenate(b.k), np.concatenate(b.v)
    q = np.zeros((tokens, qh, d), dtype)
    view = lambda x: (ctx.upload(x), x.shape, (x.shape[1] * d, d, 1))
    ctx.qkv_rope_paged_append(view(q), view(k), view(v), ctx.upload(ones), ctx.upload(zeros),
                              ctx.upload(np.zeros(tokens, np.uint32)),
                              ctx.upload(slots.astype(np.uint32)), dk, dv)
    table = np.array([[far.get(int(p), NONE) for p in row] for row in b.table], np.uint32)
    out = ctx.upload(np.full(b.q.shape, 7.0, dtype))
    ctx.paged_attention(ctx.upload(b.q), dk, dv, ctx.upload(table), ctx.upload(b.offsets),
                        ctx.upload(b.context), b.scale, b.max_queries, b.max_context, out)
    ctx.finish()
    b.check(out.numpy())
    dk.release()
    dv.release()
    abi.check(ctx.lib.rl_context_trim(ctx.handle))


def test_two_contexts_serve_their_own_batches(ctx):
    """Calls of two contexts (streams) at once, each with its own workspace."""
    other = abi.Context(0)
    try:
        batches = [Batch([(1500, 1), (800, 1)], 6, 2, 64, 16, np.float16, ("two", i))
                   for i in range(2)]
        held = [(c, b, b.upload(c)) for c, b in zip((ctx, other), batches)]
        outs = [c.upload(np.full(b.q.shape, 7.0, np.float16)) for c, b, _ in held]
        for _ in range(20):
            for (c, b, d), out in zip(held, outs):
                c.paged_attention(d["q"], d["kp"], d["vp"], d["table"], d["offsets"], d["context"],
                                  b.scale, 1, b.max_context, out)
        for (c, b, _), out in zip(held, outs):
            c.finish()
            b.check(out.numpy())
        del outs, held
    finally:
        other.close()


def test_the_workspace_is_this_contexts_and_large_enough(ctx):
    b = Batch([(100, 1)], 6, 2, 64, 16, np.float16, ("workspace",))
    d = b.upload(ctx)

    def go(workspace):
        return ctx.paged_attention(d["q"], d["kp"], d["vp"], d["table"], d["offsets"],
                                   d["context"], b.scale, 1, b.max_context, None, workspace)

    with pytest.raises(abi.RustLLMError, match="not one of rl_paged_attention_workspace"):
        go(ctx.empty((1 << 20,), np.uint8))
    good = ctx.paged_workspace(1, 2)
    go(good)
    ctx.finish()
    raw = abi.RlBuffer(good.raw.data, good.raw.len, good.raw.byte_len)
    good.release()
    with pytest.raises(abi.RustLLMError, match="not one of"):  # released
        go(View(ctx, raw, np.uint8, (raw.len,)))
    ctx.capture_begin()
    try:
        with pytest.raises(abi.RustLLMError, match="while recording"):
            ctx.paged_workspace(1, 2)
    finally:
        ctx.graph_destroy(ctx.capture_end())


def test_no_workspace_on_a_branch_of_a_recording(ctx):
    """A recording that another context joined by an event."""
    fork, join = ctx.event(), ctx.event()
    other = abi.Context(0)
    try:
        ctx.capture_begin()
        try:
            ctx.record(fork)
            other.wait(fork)
            with pytest.raises(abi.RustLLMError, match="while recording"):
                other.paged_workspace(1, 2)
            other.record(join)
            ctx.wait(join)
        finally:
            ctx.graph_destroy(ctx.capture_end())
        other.paged_workspace(1, 2).release()
    finally:
        other.close()
        ctx.destroy_event(fork)
        ctx.destroy_event(join)


# ------------------------------------------------------------------ packed


def packed_check(ctx, lengths, qh, kvh, d, dtype, key, padding=0, layout="rows", sigma=1.0,
                 max_queries=None, poison=None):
    tokens = sum(lengths) + padding
    heads = qh + 2 * kvh
    x = normal((tokens, heads, d), np.float32, "packed", *key)
    x[:, :qh] *= sigma
    x = x.astype(dtype)
    if padding:
        x[sum(lengths):] = np.nan
    if poison is not None:
        x[poison] = np.nan
    offsets = np.cumsum([0] + lengths).astype(np.uint32)
    pad = {"rows": 0, "odd": 1, "heads": 0}[layout]
    if layout == "heads":
        stored, strides = np.ascontiguousarray(x.transpose(1, 0, 2)), (d, tokens * d, 1)
        at = lambda h: h * tokens * d
    else:
        stored = np.zeros((tokens, heads * d + pad), dtype)
        stored[:, :heads * d] = x.reshape(tokens, -1)
        strides, at = (heads * d + pad, d, 1), lambda h: h * d
    dx = ctx.upload(stored)

    def view(first, n):
        reach = (tokens - 1) * strides[0] + (n - 1) * strides[1] + d
        es = np.dtype(dtype).itemsize
        raw = abi.RlBuffer(dx.ptr + at(first) * es, reach, reach * es)
        return View(ctx, raw, dtype, (reach,)), (tokens, n, d), strides

    out = ctx.upload(np.full((tokens, qh, d), 7.0, dtype))
    scale = 1.0 / np.sqrt(d)
    ctx.begin()
    ctx.packed_attention(view(0, qh), view(qh, kvh), view(qh + kvh, kvh), ctx.upload(offsets),
                         scale, max_queries or max(lengths), out)
    ctx.finish()
    got = out.numpy()
    kind = "f16_fused" if dtype == np.float16 else "f32"
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        part = x[offsets[i]:offsets[i + 1]].transpose(1, 0, 2)[None]
        seen = n
        if poison is not None and offsets[i] <= poison < offsets[i + 1]:
            seen = poison - int(offsets[i])
            assert np.isnan(got[poison:offsets[i + 1]]).all()
            if seen == 0:
                continue
            part = part[:, :, :seen]
        exact, bound = attention_bound(part[:, :qh], part[:, qh:qh + kvh], part[:, qh + kvh:],
                                       scale, 0, None, kind)
        have = got[offsets[i]:offsets[i] + seen].astype(np.float64).transpose(1, 0, 2)
        assert np.isfinite(have).all(), f"prompt {i} of {n}: non-finite output"
        err = np.abs(have - exact[0])
        worst = np.unravel_index(np.argmax(err / bound[0]), err.shape)
        assert np.all(err <= bound[0]), (f"prompt {i} of {n}: error {err[worst]:.3g} > "
                                         f"{bound[0][worst]:.3g} at {worst}")
    assert np.all(got[offsets[-1]:] == 7.0), "rows behind the last prompt"


PACKED = [
    ([1], 15, 5, 64), ([1, 1, 0, 1], 9, 3, 64), ([0, 0, 7], 8, 8, 64),
    ([31, 32, 33, 0, 1, 64, 65], 9, 3, 64), ([127, 128, 129, 5], 32, 8, 128),
    ([200, 17, 96], 15, 5, 64), ([300, 1, 44], 12, 3, 96), ([70, 130], 8, 8, 80),
    ([100, 50], 6, 3, 32), ([19, 40], 4, 2, 48), ([9, 6], 2, 1, 7), ([5, 9], 2, 2, 200),
    ([3, 8], 1, 1, 512), ([700, 600], 16, 1, 64), ([60, 90], 40, 1, 64), ([1500], 9, 3, 64),
    ([1100, 900, 3], 8, 8, 128), ([2, 3] * 100, 6, 2, 64),
    # enough rows for the wide tiles (and, the last, to order them by length)
    ([700, 500, 33, 64], 32, 8, 64), ([600, 511, 1], 32, 8, 128), ([400, 700], 32, 8, 96),
    ([900, 300], 32, 8, 32), ([260, 30, 511] * 6, 32, 8, 64), ([130, 300] * 10, 32, 8, 128),
    ([40] * 80 + [900], 32, 8, 64),
    *[([700, 500, 33, 64, 300, 500], 64, 16, d) for d in (64, 56, 32, 24)],
    *[([600, 511, 1], 64, 16, d) for d in (128, 112, 96, 80)],
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_attention_within_float64_bound(ctx, dtype, case):
    lengths, qh, kvh, d = PACKED[case]
    packed_check(ctx, lengths, qh, kvh, d, dtype, ("packed", case), padding=case % 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["odd", "heads"])
def test_packed_attention_strides(ctx, dtype, layout):
    packed_check(ctx, [40, 3, 130], 6, 2, 64, dtype, ("strides",), layout=layout, padding=2)
    packed_check(ctx, [40, 3, 130], 6, 2, 64, dtype, ("strides",), layout=layout,
                 max_queries=4000)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [0, 45, 99, 100, 230])
def test_packed_prompts_do_not_reach_each_other(ctx, dtype, poison):
    """A token of NaN reaches the rows that see it and no others."""
    packed_check(ctx, [100, 131, 60], 6, 2, 64, dtype, ("poison",), poison=poison)


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_attention_of_wide_scores(ctx, dtype):
    packed_check(ctx, [300, 90], 6, 2, 64, dtype, ("wide",), sigma=8.0)


# ------------------------------------------------------------ all together


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_servers_steps(ctx, dtype):
    """Prompts through plan, append and packed attention, then decode steps and
    a late prompt's chunks through plan, append and paged attention; every
    request's rows against float64 attention over its own rotated history."""
    qh, kvh, d, page, blocks, pages = 6, 2, 64, 16, 12, 64
    heads = qh + 2 * kvh
    requests = 5
    angle = np.arange(256)[:, None] * 100.0 ** (-np.arange(0, d, 2) / d)[None]
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    dcos, dsin = ctx.upload(cos), ctx.upload(sin)
    pool = np.full((pages, kvh, page, d), np.nan, dtype)
    dk, dv = ctx.upload(pool), ctx.upload(pool)
    table = ctx.upload(np.full((requests, blocks), NONE, np.uint32))
    free = list(np.random.default_rng(1).permutation(pages))
    cached = [0] * requests
    history = [np.zeros((0, kvh, d), dtype) for _ in range(2 * requests)]  # K, then V
    kind = "f16_fused" if dtype == np.float16 else "f32"
    scale = 1.0 / np.sqrt(d)
    for step, fresh in enumerate([[20, 33, 0, 1, 16], [1, 1, 50, 1, 1], [1, 1, 41, 1, 0],
                                  [1, 2, 1, 1, 3]]):
        tokens = sum(fresh) + 2
        x = normal((tokens, heads, d), dtype, "server", step)
        dx = ctx.upload(x)

        def view(first, n):
            reach = (tokens - 1) * heads * d + n * d
            es = np.dtype(dtype).itemsize
            raw = abi.RlBuffer(dx.ptr + first * d * es, reach, reach * es)
            return View(ctx, raw, dtype, (reach,)), (tokens, n, d), (heads * d, d, 1)

        u32 = lambda v: ctx.upload(np.array(v, np.uint32))
        dc, df, dfree = u32(cached), u32(fresh), u32(free)
        ctx.begin()
        offsets, context, slots, positions, taken = ctx.paged_plan(dc, df, dfree, table, page,
                                                                   pages, tokens=tokens)
        q = ctx.qkv_rope_paged_append(view(0, qh), view(qh, kvh), view(qh + kvh, kvh), dcos, dsin,
                                      positions, slots, dk, dv)
        out = ctx.paged_attention(q, dk, dv, table, offsets, context, scale, max(fresh),
                                  blocks * page)
        ctx.finish()
        free = free[int(taken.numpy()[0]):]
        got = out.numpy()
        at = 0
        for i, n in enumerate(fresh):
            rows = [rotated(ctx, x[at + j, :qh + kvh], cos, sin, cached[i] + j) for j in range(n)]
            if n:
                turned = np.stack(rows)
                history[i] = np.concatenate([history[i], turned[:, qh:]])
                history[requests + i] = np.concatenate([history[requests + i],
                                                        x[at:at + n, qh + kvh:]])
                exact, bound = attention_bound(turned[:, :qh].transpose(1, 0, 2)[None],
                                               history[i].transpose(1, 0, 2)[None],
                                               history[requests + i].transpose(1, 0, 2)[None],
                                               scale, cached[i], None, kind)
                err = np.abs(got[at:at + n].astype(np.float64).transpose(1, 0, 2) - exact[0])
                assert np.all(err <= bound[0]), (step, i)
            at += n
            cached[i] += n
        if step == 0:  # the packed form over [Q, K] rotated and V of the same prompts
            q_rows = q.numpy()
            packed = np.concatenate([q_rows, np.zeros((tokens, 2 * kvh, d), dtype)], 1)
            at = 0
            for i, n in enumerate(fresh):
                packed[at:at + n, qh:qh + kvh] = history[i]
                packed[at:at + n, qh + kvh:] = history[requests + i]
                at += n
            dx = ctx.upload(packed)
            p_out = ctx.packed_attention(view(0, qh), view(qh, kvh), view(qh + kvh, kvh), offsets,
                                         scale, max(fresh))
            ctx.finish()
            both = np.abs(p_out.numpy()[:at].astype(np.float64) - got[:at].astype(np.float64))
            limit = {np.float16: 2.0 ** -8, np.float32: 2.0 ** -16}[dtype]
            assert np.all(both <= limit * np.maximum(1.0, np.abs(got[:at].astype(np.float64))))


@pytest.mark.parametrize("name", ["paged_plan", "qkv_rope_paged_append_f16", "paged_attention_f16",
                                  "packed_attention_f16"])
def test_profile_counts_one_dispatch_a_call(ctx, name):
    ctx.profile_begin()
    test_a_servers_steps(ctx, np.float16)
    assert ctx.dispatches(name) == (1 if name.startswith("packed") else 4)
    ctx.profile_take()
