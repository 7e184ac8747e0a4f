"""Arguments of the batch operators at the edge of what their types hold, and the
binding's own checks: no GPU needed."""

import ctypes

import pytest

from rustllm_amd import abi

lib = abi.load()
SHAPE, DEVICE = 2, 9


def buf(n, es):
    """An rl_buffer of n elements, lengths modulo 2^64."""
    return abi.RlBuffer(0x10000, n % (1 << 64), n * es % (1 << 64))


def u64s(*v):
    return (ctypes.c_uint64 * len(v))(*v)


@pytest.mark.parametrize("dims", [(), (4,), (4, 64), (1, 4, 2, 64)])
def test_views_of_another_rank_are_refused(dims):
    """The library reads three dims and three strides of a view."""
    good = (None, (4, 2, 64), (128, 64, 1))
    assert len(abi._view_addresses(good, good, good)[1]) == 6
    for views in [((None, dims, (128, 64, 1)), good, good),
                  (good, (None, (4, 2, 64), dims), good), (good, good, (None, dims, dims))]:
        with pytest.raises(ValueError, match="rank 3"):
            abi._view_addresses(*views)


@pytest.mark.parametrize("dt,es", [("f32", 4), ("f16", 2)])
def test_append_of_counts_that_wrap(dt, es):
    """Token and head counts of views with strides of zero whose element count is a
    multiple of 2^128."""
    tokens, q_heads, kv_heads, d = 1 << 63, (1 << 64) - 2, 1, 2
    q, kv, still = u64s(tokens, q_heads, d), u64s(tokens, kv_heads, d), u64s(0, 0, 1)
    row, table, per_token = buf(2, es), buf(8, 4), buf(tokens, 4)
    pool = buf(3 * 4 * d, es)
    held = [row, q, still, row, kv, still, row, kv, still, table, table, 8, per_token, per_token,
            buf(tokens * q_heads * d, es), pool, pool]
    status = getattr(lib, f"rl_qkv_rope_paged_append_{dt}")(
        None, *[ctypes.addressof(x) if not isinstance(x, int) else x for x in held], 3, 4)
    assert status == SHAPE and "exceeds u32" in abi.last_error()


@pytest.mark.parametrize("requests,kv_heads", [
    (1, 1), (3, 3), (64, 8), (2_100_000, 3), (5_000_000, 1), (1, 8_000_000), (699_050, 11)])
def test_the_bindings_workspace_fits_every_batch_a_call_takes(requests, kv_heads):
    """Sizes that rl_paged_attention_* accepts, rounded up or not, are accepted for the
    workspace that the binding makes."""
    made = abi._workspace_sizes(requests, kv_heads)
    assert made[0] >= requests and made[1] >= kv_heads
    for sizes in ((requests, kv_heads), made):
        status = lib.rl_paged_attention_workspace(None, *sizes, ctypes.byref(abi.RlBuffer()))
        assert status == DEVICE, (sizes, abi.last_error())
