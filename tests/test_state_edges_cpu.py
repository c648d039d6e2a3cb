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


def test_eviction_into_its_own_lengths_is_refused():
    """The heads of a row read its length while the first of them writes the new one."""
    rows, heads, cols = 2, 2, 64
    for lens, bytes_, out in ((4096, 4, 4096), (4096, 8, 4096), (4096, 8, 4104), (4104, 4, 4100)):
        last(lib.dgs_evict_rows(None, None, 0, 4, heads, 16, 1 << 20, None, 1 << 21, 1 << 22, rows, cols,
                                1 << 23, 4, 4, lens, bytes_, out, 8, 0, 0, None, 0, None), b"lens_out")
    many = rows * heads * cols * 4
    w, p, wo, po = (1 << k for k in (20, 21, 22, 23))
    for bad in ((w, p, w, po), (w, p, wo, p), (w, p, w + 4, po), (w, p, wo, p - many + 4), (w, p, wo, wo),
                (w, p, p, po), (w, None, wo, w - 4), (w, p, wo, w)):
        last(lib.dgs_evict_rows(None, None, 0, 4, heads, 16, *bad, rows, cols, 1 << 24, 4, 4, 4096, 4, 8192,
                                8, 0, 0, None, 0, None), b"other arrays")
    last(lib.dgs_evict_rows(None, None, 0, 4, 2 ** 30, 16, w, p, wo, po, 2, cols, 1 << 24, 4, 4, 4096, 4,
                            8192, 8, 0, 0, None, 0, None), b"too many rows")


@pytest.mark.parametrize("scale", [2.0 ** 100, -2.0 ** 100, 1e300, float("inf"), float("nan")])
def test_scales_past_the_sums_range_are_refused(scale):
    c = _CCache(4096, 4096, 4096, 4096, 4, 8, 2, 64, 32)
    last(lib.dgs_state_attend(ctypes.addressof(c), 4096, 0, 1, 2, 128, 64, 4096, 4, 1, 4096, 4, scale, None,
                              0, 1.0, 4096, None, 0, None), b"scale")


@pytest.mark.parametrize("off", [1, 4, 8])
def test_misaligned_workspaces_are_refused(off):
    """Parts are stored 16 bytes at a time."""
    c = _CCache(4096, 4096, 4096, 4096, 4, 8, 2, 64, 32)
    last(lib.dgs_state_attend(ctypes.addressof(c), 4096, 0, 1, 2, 128, 64, 4096, 4, 1000, 4096, 4, 1.0, None,
                              0, 1.0, 4096, 8192 + off, 1 << 30, None), b"attend: the workspace")
    last(lib.dgs_evict_rows(None, None, 0, 4, 2, 16, 1 << 20, None, 1 << 21, 1 << 22, 2, 2000, 1 << 24, 4, 4,
                            4096, 4, 8192, 300, 0, 0, 16384 + off, 1 << 30, None), b"evict: the workspace")
