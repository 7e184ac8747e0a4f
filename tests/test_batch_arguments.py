"""Arguments of the batch operators at the edge of what their types hold, and the
binding's own checks: no GPU needed."""

import ctypes

import pytest

from rustllm_amd import abi

lib = abi.load()
SHAPE, DEVICE = 2, 9


def buf(n, byte_len, addr=0x10000):
    return ctypes.byref(abi.RlBuffer(addr, n, byte_len))


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
