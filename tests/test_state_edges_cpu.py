"""Refusals of the state cache's calls, which need no GPU."""
import ctypes

import pytest

from dgs._lib import c_i64, lib
from dgs.state import StateCache, _CCache


def last(rc, msg):
    assert rc == -1 and msg in lib.dgs_last_error(), lib.dgs_last_error()


@pytest.mark.parametrize("heads, dim", [(2 ** 22 + 1, 256), (2 ** 30, 8), (2 ** 31 - 1, 256)])
def test_slots_of_too_many_channels_are_refused(heads, dim):
    """A slot's channels and groups are counted in 32 bits: past that rows were read in part."""
    with pytest.raises(RuntimeError, match="2\\^30"):
        StateCache(1, 1, heads, dim)
    c = _CCache(4096, 4096, 4096, 4096, 1, 1, heads, dim, dim)
    ref = ctypes.addressof(c)
    last(lib.dgs_state_read(ref, 4096, 1, 0, 4096, 4096, None), b"2^30")
    last(lib.dgs_state_write(ref, 4096, 4096, 0, 1, heads * dim, dim, heads * dim, dim, 4096, None),
         b"2^30")
    n = c_i64()
    last(lib.dgs_state_attend_workspace(ref, 1, heads, 1, 0, 0, ctypes.byref(n)), b"2^30")
    most = _CCache(4096, 4096, 4096, 4096, 1, 1, 2 ** 30 // dim, dim, dim)
    assert lib.dgs_state_read(ctypes.addressof(most), None, 0, 0, None, None, None) == 0
