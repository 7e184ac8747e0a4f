"""The batch attentions where precision is easily lost: weights that differ by
hundreds of powers of two over long ranges of keys that every row sees."""

import numpy as np
import pytest

from helpers import attention_bound, attention_exact, ulp16
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


def heavy_and_light(spans, qh, kvh, d, dtype, light, key):
    """A batch whose every row sees one key of weight 1, whose values are zeros, and, of each
    other key, 2^light of that weight (to f16's steps of the scores), values of about 1."""
    b = Batch(spans, qh, kvh, d, 64, dtype, key)
    b.q[:] = 0.0
    b.q[:, :, 0] = np.sqrt(d)  # the score is the key's first element
    for i, keys in enumerate(b.context):
        k, v = b.k[i], b.v[i]
        k[:, :, 0] = 8.0 + light * np.log(2.0)
        v[:] = (1.0 + 0.125 * v.astype(np.float32)).astype(dtype)
        k[spans[i][0] // 3, :, 0], v[spans[i][0] // 3] = 8.0, 0.0
        pos = np.arange(keys)
        b.kp[b.table[i, pos // 64], :, pos % 64] = k
        b.vp[b.table[i, pos // 64], :, pos % 64] = v
    b.scale = 1.0 / np.sqrt(d)
    return b


def check_light_weights(b, got):
    """As attention_bound, but for its kv_len 2^-25 max|v| of f16 probabilities below the
    normal range: each is raised by 2^12 over the row's maximum, which leaves
    kv_len 2^-37 max|v|."""
    for i in range(len(b.spans)):
        rows, exact, bound = b.expect(i)
        if b.q.dtype == np.float16:
            vmax = np.max(np.abs(b.v[i].astype(np.float64)))
            bound = bound - int(b.context[i]) * (2.0 ** -25 - 2.0 ** -37) * vmax
        err = np.abs(got[rows].astype(np.float64).transpose(1, 0, 2) - exact)
        worst = np.unravel_index(np.argmax(err / bound), err.shape)
        assert np.all(err <= bound), (f"request {i}: error {err[worst]:.3g} > {bound[worst]:.3g} "
                                      f"of {exact[worst]:.3g} at {worst}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("d", [64, 128, 96, 80, 32])
@pytest.mark.parametrize("light", [-12.0, -16.5, -21.3, -27.4])
def test_many_light_keys_keep_their_weight(ctx, dtype, light, d, n):
    """One heavy key among a hundred thousand, and among thirty thousand, light ones."""
    b = heavy_and_light([(100000, n), (30001, 1)], 2, 1, d, dtype, light, ("light", d, n))
    check_light_weights(b, b.run(ctx))


@pytest.mark.parametrize("d", [64, 128, 96, 80, 32])
@pytest.mark.parametrize("light", [-10.0, -14.5, -16.5, -20.3])
def test_light_keys_of_a_packed_prompt(ctx, light, d):
    """The same within a prompt (f16): the heavy key is its first token."""
    tokens = 3000
    q, k, v = (np.zeros((tokens, 1, d), np.float16) for _ in range(3))
    q[:, :, 0] = np.sqrt(d)
    k[:, :, 0] = 8.0 + light * np.log(2.0)
    v[:] = 1.0 + 0.125 * normal(v.shape, np.float32, "light packed", d)
    k[0, :, 0], v[0] = 8.0, 0.0
    scale = 1.0 / np.sqrt(d)
    view = lambda x: (ctx.upload(x), x.shape, (d, d, 1))
    offsets = ctx.upload(np.array([0, tokens], np.uint32))
    got = ctx.packed_attention(view(q), view(k), view(v), offsets, scale, tokens).numpy()
    rows = np.r_[0:3, 31:34, 1000:1003, 2990:3000]
    for r in rows:
        exact, bound = attention_bound(q[r][None, None], k[:r + 1].transpose(1, 0, 2)[None],
                                       v[:r + 1].transpose(1, 0, 2)[None], scale, int(r), None,
                                       "f16_fused")
        vmax = np.max(np.abs(v[:r + 1].astype(np.float64)))
        bound = bound[0, :, 0] - (r + 1) * (2.0 ** -25 - 2.0 ** -37) * vmax
        err = np.abs(got[r].astype(np.float64) - exact[0, :, 0])
        assert np.all(err <= bound), (int(r), float(np.max(err / bound)))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_len", [1, 300])
def test_light_keys_of_one_sequence(ctx, q_len, d):
    """rl_attention_f16, whose probabilities stop at f16's own range: weights of 2^-16.5,
    in which its sum and its product have to agree."""
    keys = 30000
    q, k, v = np.zeros((1, 2, q_len, d)), np.zeros((1, 1, keys, d)), np.ones((1, 1, keys, d))
    q[..., 0], k[..., 0] = np.sqrt(d), 8.0 - 16.5 * np.log(2.0)
    k[:, :, 5, 0], v[:, :, 5] = 8.0, 0.0
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    got = ctx.attention(ctx.upload(q), ctx.upload(k), ctx.upload(v), 1.0 / np.sqrt(d),
                        keys - q_len).numpy().astype(np.float64)
    exact, bound = attention_bound(q[:, :, :1], k[:, :, :keys - q_len + 1],
                                   v[:, :, :keys - q_len + 1], 1.0 / np.sqrt(d), keys - q_len,
                                   None, "f16_fused")
    assert np.all(np.abs(got[:, :, :1] - exact) <= bound)


def check_22_bits(q, k, v, scale, start, got):
    """f16 outputs of probabilities that keep 22 bits (2^-22 of each, 2^-37 of the row's
    maximum below the normal range) beside sums in f32 and the outputs' own rounding."""
    exact, weight, _ = attention_exact(q, k, v, scale, start)
    _, bound = attention_bound(q, k, v, scale, start, None, "f32")
    vmax = np.max(np.abs(np.asarray(v, np.float64)))
    bound = bound + 2.0 ** -22 * weight + k.shape[2] * 2.0 ** -37 * vmax
    bound = bound + 0.5 * ulp16(np.abs(exact) + bound)
    err = np.abs(np.asarray(got, np.float64) - exact)
    worst = np.unravel_index(np.argmax(err / bound), err.shape)
    assert np.all(err <= bound), f"error {err[worst]:.4g} > {bound[worst]:.4g} at {worst}"


# Small query elements and few keys: the sums' roundings are then small beside those of
# probabilities held in one f16 part.
@pytest.mark.parametrize("n", [1, 9])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 72, 80, 88, 104, 112, 120, 32, 64, 96, 128])
def test_probabilities_of_a_paged_batch_keep_22_bits(ctx, d, n):
    """Of every head size where a request has few rows, of the sizes off the multiples of
    32 where it has more."""
    if n > 4 and d % 32 == 0:
        n = 4  # 16 rows of four heads
    b = Batch([(c, n) for c in (20, 3, 30, 12, 25)], 8, 2, d, 16, np.float16, ("22 bits", d, n),
              sigma=0.25)
    got = b.run(ctx)
    for i, (c, _) in enumerate(b.spans):
        rows = slice(int(b.offsets[i]), int(b.offsets[i + 1]))
        check_22_bits(b.q[rows].transpose(1, 0, 2)[None], b.k[i].transpose(1, 0, 2)[None],
                      b.v[i].transpose(1, 0, 2)[None], b.scale, c,
                      got[rows].transpose(1, 0, 2)[None])


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 72, 80, 88, 104, 112, 120])
def test_probabilities_of_packed_prompts_keep_22_bits(ctx, d, many):
    """Head sizes off the multiples of 32, in narrow and wide tiles."""
    lengths = [30, 7, 25] + ([33] * 110 if many else [])
    qh, kvh = (32, 8) if many else (8, 2)
    tokens, heads = sum(lengths), qh + 2 * kvh
    x = normal((tokens, heads, d), np.float32, "22 bits packed", d, many)
    x[:, :qh] *= 0.25
    x = x.astype(np.float16)
    parts = x[:, :qh], x[:, qh:qh + kvh], x[:, qh + kvh:]
    views = [(ctx.upload(np.ascontiguousarray(p)), p.shape, (p.shape[1] * d, d, 1)) for p in parts]
    offsets = np.cumsum([0] + lengths).astype(np.uint32)
    scale = 1.0 / np.sqrt(d)
    got = ctx.packed_attention(*views, ctx.upload(offsets), scale, max(lengths)).numpy()
    for i in (0, 1, 2, len(lengths) - 1):
        rows = slice(int(offsets[i]), int(offsets[i + 1]))
        q, k, v = (p[rows].transpose(1, 0, 2)[None] for p in parts)
        check_22_bits(q, k, v, scale, 0, got[rows].transpose(1, 0, 2)[None])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,cached", [(1, 5000), (2, 300), (40, 900), (300, 500)])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_scores_of_tens_of_millions_take_one_key(ctx, dtype, n, cached, d):
    """Scores so large that f32's steps between them are whole exponents: each row's
    output is the value row v of its largest score wherever the next one is far below it.
    The weight p of that key is not 1 but 2 to what the maximum's rounding left, in the sum
    as in the product: (p v) / p.  In f32 that is v up to the roundings of p v, of the
    quotient's two steps, of both sides' rescaling in two merges, and the split's: 8 of
    2^-24.  In f16 the rounding of the output takes it back to v."""
    b = Batch([(cached, n), (30, 1)], 4, 2, d, 32, dtype, ("millions", n, d), sigma=1e4)
    for i in range(2):
        b.k[i] = (1e3 * b.k[i].astype(np.float32)).astype(dtype)
        pos = np.arange(b.context[i])
        b.kp[b.table[i, pos // 32], :, pos % 32] = b.k[i]
    assert np.isfinite(b.q).all() and np.isfinite(b.k[0]).all()
    got = b.run(ctx)
    checked = 0
    for i, (c, m) in enumerate(b.spans):
        for j in range(m):
            row = int(b.offsets[i]) + j
            for h in range(4):
                s = b.k[i][:c + j + 1, h // 2].astype(np.float64) @ b.q[row, h].astype(np.float64)
                s *= b.scale
                top = int(np.argmax(s))
                s[top], best = -np.inf, s[top]
                # errors of two scores of D products each: D 2^-24 of their terms' sum
                terms = np.abs(b.q[row, h].astype(np.float64)) @ np.abs(
                    b.k[i][:c + j + 1, h // 2].astype(np.float64)).T
                unsure = 2 * b.scale * d * 2.0 ** -24 * terms.max()
                if best - np.max(s, initial=-np.inf) < unsure + 200:
                    continue
                v = b.v[i][top, h // 2].astype(np.float64)
                off = 8 * 2.0 ** -24 * np.abs(v) if dtype == np.float32 else 0.0
                assert np.all(np.abs(got[row, h] - v) <= off), (i, j, h)
                checked += 1
    assert checked > 2 * n
