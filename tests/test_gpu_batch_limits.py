"""The batch operators near the limits of one launch."""

import numpy as np
import pytest

from helpers import attention_bound
from test_gpu_paged import DTYPES, NONE, Batch, normal, packed_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 20])
def test_paged_attention_of_millions_of_requests(ctx, dtype, n):
    """2.1 million requests of 3 KV heads, all but three without rows: the binding's own
    workspace is made for as many."""
    requests, qh, kvh, d, page = 2_100_000, 3, 3, 64, 64
    live = {5: 3, 1_000_003: 40, requests - 1: 64}  # request -> keys, at least its rows
    live = {i: max(keys, n) for i, keys in live.items()}
    fresh, context = np.zeros(requests, np.uint32), np.zeros(requests, np.uint32)
    table = np.full((requests, 1), NONE, np.uint32)
    for at, (i, keys) in enumerate(live.items()):
        fresh[i], context[i], table[i, 0] = n, keys, len(live) - 1 - at
    offsets = np.concatenate([[0], np.cumsum(fresh)]).astype(np.uint32)
    q = normal((3 * n, qh, d), dtype, "millions", "q", n)
    kp, vp = (normal((len(live), kvh, page, d), dtype, "millions", s, n) for s in "kv")
    out = ctx.upload(np.full(q.shape, 7.0, dtype))
    args = [ctx.upload(x) for x in (q, kp, vp, table, offsets, context)]
    ctx.paged_attention(*args, 0.125, n, 64, out)
    ctx.finish()
    got = out.numpy()
    for at, (i, keys) in enumerate(live.items()):
        p = len(live) - 1 - at
        exact, bound = attention_bound(q[at * n:(at + 1) * n].transpose(1, 0, 2)[None],
                                       kp[p][None, :, :keys], vp[p][None, :, :keys], 0.125,
                                       keys - n, None,
                                       "f16_fused" if dtype == np.float16 else "f32")
        err = np.abs(got[at * n:(at + 1) * n].astype(np.float64).transpose(1, 0, 2) - exact[0])
        assert np.all(err <= bound[0]), i
    ctx._workspaces.pop((requests, kvh)).release()  # 1.5 GiB of counters


@pytest.mark.parametrize("dtype,d", [(np.float32, d) for d in range(4, 129, 4)]
                         + [(np.float16, d) for d in range(8, 129, 8)])
def test_every_head_size_of_the_matrix_kernels(ctx, dtype, d):
    """Single tokens, a chunk, both in one call and packed prompts, at every head size of
    whole 16-byte pieces."""
    for n in (1, 25):
        b = Batch([(70, n), (300, 1), (0, 1)], 6, 2, d, 8, dtype, ("sizes", d, n), padding=1)
        b.check(b.run(ctx))
    packed_check(ctx, [40, 1, 90], 6, 2, d, dtype, ("sizes", d), padding=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1 << 10, 1 << 14])
@pytest.mark.parametrize("n", [1, 30])
def test_pages_longer_than_a_context(ctx, dtype, page, n):
    b = Batch([(700, n), (0, n), (1100, n)], 6, 2, 64, page, dtype, ("pages", page, n))
    b.check(b.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 24, 7])
def test_packed_keys_that_heads_share_by_a_stride_of_zero(ctx, dtype, d):
    """K and V views whose heads are one row each (stride 0), Q's heads outside its
    tokens."""
    lengths, qh, kvh = [33, 1, 80], 6, 2
    tokens = sum(lengths)
    q = normal((qh, tokens, d), dtype, "shared", "q", d)  # heads outside tokens
    k, v = (normal((tokens, d), dtype, "shared", s, d) for s in "kv")
    offsets = np.cumsum([0] + lengths).astype(np.uint32)
    scale = 1.0 / np.sqrt(d)
    got = ctx.packed_attention((ctx.upload(q), (tokens, qh, d), (d, tokens * d, 1)),
                               (ctx.upload(k), (tokens, kvh, d), (d, 0, 1)),
                               (ctx.upload(v), (tokens, kvh, d), (d, 0, 1)),
                               ctx.upload(offsets), scale, max(lengths)).numpy()
    for i, n in enumerate(lengths):
        rows = slice(int(offsets[i]), int(offsets[i + 1]))
        exact, bound = attention_bound(q[None, :, rows], k[None, None, rows], v[None, None, rows],
                                       scale, 0, None,
                                       "f16_fused" if dtype == np.float16 else "f32")
        err = np.abs(got[rows].astype(np.float64).transpose(1, 0, 2) - exact[0])
        assert np.all(err <= bound[0]), i
