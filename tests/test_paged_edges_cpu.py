"""Calls of the paged cache that are refused for their size, without a GPU."""
import ctypes

import pytest

from tests.test_paged_cpu import full, lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("heads,dim,ok", [(1 << 23, 256, False), (1 << 24, 256, False), ((1 << 28) - 1, 8, True),
                                          (1 << 28, 8, False), ((1 << 23) - 1, 256, True)])
def test_write_refuses_tokens_of_2_31_query_values(lib, heads, dim, ok):  # noqa: F811
    """The kernel counts a token's query values in 32 bits; without a GPU an accepted call fails at the device instead."""
    from domino_b200 import _lib

    a = _lib.DDCacheWriteArgs(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, start=1 << 20, inv_freq=1 << 20, eps=1e-6,
                              factor=1.0, layer=0, tokens=1, heads=heads, rotary=8)
    c = full(head_dim=dim)
    c.device = 63  # no such device: nothing is launched on a machine with a GPU either
    rc = lib.dd_cache_write(ctypes.byref(c), ctypes.byref(a), None)
    assert rc < 0 and (rc == _lib.DD_EINVAL) != ok
    assert (b"chunk too large" in lib.dd_last_error(None)) != ok
