"""What attention with masses (trx_attn_mass) refuses before it launches anything (no GPU)."""

import ctypes

import pytest

from trixium_amd import _lib
from test_kv_mass_gpu import Cache


@pytest.mark.parametrize("kv", [1, 2, 8])
def test_slots_past_a_grid_are_refused(kv):
    """The masses of long calls take 512 threads for 128 slots of a kv head: 2^30 slots would be a grid of 2^32 threads,
    refused by the launch when the attention and the rows' copies had run."""
    c = Cache(8, kv, 64, 40)
    lib, size, fake = _lib.lib(), ctypes.c_size_t(), ctypes.c_void_p(256)
    for slots, n in (((1 << 30) // kv, 1), ((1 << 30) // kv, 700), ((1 << 30) // kv - 127, 700)):
        shape = c.shape(slots=slots)
        assert lib.trx_attn_mass_geometry(ctypes.byref(shape), n, ctypes.byref(size)) == _lib.TRX_E_INVALID
        assert b"slots" in lib.trx_last_error()
        for state in (None, fake):
            assert lib.trx_attn_mass(ctypes.byref(shape), n, 0, 0, state, *[fake] * 7, None, fake, fake, None) == _lib.TRX_E_INVALID
            assert b"slots" in lib.trx_last_error()
    shape = c.shape(slots=(1 << 30) // kv - 128)
    assert lib.trx_attn_mass_geometry(ctypes.byref(shape), 700, ctypes.byref(size)) == _lib.TRX_OK
