"""The batch operators near the limits of one launch."""

import numpy as np
import pytest

from helpers import attention_bound
from test_gpu_paged import DTYPES, NONE, normal

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
