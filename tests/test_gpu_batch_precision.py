"""The batch attentions where precision is easily lost: weights that differ by
hundreds of powers of two over long ranges of keys that every row sees."""

import numpy as np
import pytest

from helpers import attention_bound
from test_gpu_paged import DTYPES, Batch, normal, packed_check

pytestmark = pytest.mark.gpu

# lengths, q heads, KV heads, head size: of prompts that take each shape of tile
PACKED = [
    ([520, 700, 513, 600], 32, 8, 128), ([300, 257], 12, 3, 96), ([300, 257], 8, 2, 128),
    ([300, 257], 6, 2, 64), ([700, 500, 333, 600], 32, 8, 64), ([300, 257], 6, 3, 32),
]
PAGED = [
    ([(700, 33), (300, 1)], 6, 2, 64, 16), ([(700, 33), (900, 20)], 6, 2, 96, 16),
    ([(700, 70), (900, 20)], 8, 2, 128, 32), ([(700, 260), (300, 250)], 32, 8, 64, 16),
    ([(900, 1), (300, 2)], 8, 2, 128, 16),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sigma", [30.0, 100.0])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_attention_of_very_wide_scores(ctx, dtype, sigma, case):
    lengths, qh, kvh, d = PACKED[case]
    packed_check(ctx, lengths, qh, kvh, d, dtype, ("very wide", case), sigma=sigma)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sigma", [30.0, 100.0])
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_attention_of_very_wide_scores(ctx, dtype, sigma, case):
    spans, qh, kvh, d, page = PAGED[case]
    b = Batch(spans, qh, kvh, d, page, dtype, ("very wide", case), sigma=sigma)
    b.check(b.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sigma", [30.0, 100.0])
@pytest.mark.parametrize("qh,kvh,q_len,kv_len,d", [
    (15, 5, 200, 700, 64), (8, 2, 300, 300, 128), (6, 2, 130, 600, 96), (4, 4, 90, 400, 32)])
def test_attention_of_very_wide_scores(ctx, dtype, sigma, qh, kvh, q_len, kv_len, d):
    """rl_attention_* of one sequence, whose tiles take the same maxima."""
    key = ("very wide one", qh, q_len, d)
    q = (sigma * normal((1, qh, q_len, d), np.float32, "q", *key)).astype(dtype)
    k, v = (normal((1, kvh, kv_len, d), dtype, name, *key) for name in "kv")
    scale = 1.0 / np.sqrt(d)
    got = ctx.attention(ctx.upload(q), ctx.upload(k), ctx.upload(v), scale,
                        kv_len - q_len).numpy().astype(np.float64)
    kind = "f16_fused" if dtype == np.float16 else "f32"
    exact, bound = attention_bound(q, k, v, scale, kv_len - q_len, None, kind)
    assert np.isfinite(got).all()
    err = np.abs(got - exact)
    worst = np.unravel_index(np.argmax(err / bound), err.shape)
    assert np.all(err <= bound), f"error {err[worst]:.3g} > {bound[worst]:.3g} at {worst}"
