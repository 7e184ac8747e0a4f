"""Recorded batch calls replayed with lengths far from those they were recorded with."""

import numpy as np
import pytest

from helpers import assert_bitexact
from test_gpu_paged import DTYPES, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans", [[(400, 1), (30, 1)], [(100, 80), (600, 1)], [(3, 1), (0, 0)]])
def test_recorded_attention_follows_longer_contexts(ctx, dtype, spans):
    """Replays whose contexts are several times those of the recording (more keys a
    workgroup, more workgroups a request), then short ones again; eager work and waits
    between, each replay against its own batch."""
    blocks, pages = 200, 420
    first = Batch(spans, 6, 2, 64, 16, dtype, ("longer", len(spans), spans[0][1]), blocks=blocks,
                  spare=pages - sum(-(-(c + n) // 16) for c, n in spans))
    d = first.upload(ctx)
    out = ctx.upload(np.full(first.q.shape, 7.0, dtype))
    args = (d["q"], d["kp"], d["vp"], d["table"], d["offsets"], d["context"], first.scale, 90,
            blocks * 16)
    ctx.paged_attention(*args, out)  # makes the workspace
    ctx.finish()
    ctx.capture_begin()
    ctx.paged_attention(*args, out)
    graph = ctx.capture_end()
    try:
        fresh = [n for _, n in spans]
        for turn, cached in enumerate([(1100, 1000), (3000, 70), (5, 3100), (3100, 3100), (1, 0)]):
            lengths = list(zip(cached, fresh))
            used = sum(-(-(c + n) // 16) for c, n in lengths)
            assert used <= pages
            b = Batch(lengths, 6, 2, 64, 16, dtype, ("longer turn", turn, spans[0][1]),
                      blocks=blocks, spare=pages - used)
            assert b.kp.shape == first.kp.shape and b.q.shape == first.q.shape
            for name in ("q", "kp", "vp", "table", "offsets", "context"):
                ctx.copy(ctx.upload(getattr(b, name)), d[name])
            ctx.copy(ctx.upload(np.full(first.q.shape, 7.0, dtype)), out)
            ctx.finish()
            eager = ctx.upload(np.full(first.q.shape, 7.0, dtype))
            ctx.graph_launch(graph)
            ctx.paged_attention(*args, eager)
            ctx.finish()
            b.check(out.numpy())
            assert_bitexact(out.numpy(), eager.numpy(), "replay against eager")
    finally:
        ctx.graph_destroy(graph)
