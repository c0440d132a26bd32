"""8-bit paged KV cache without a GPU: what its calls refuse at the edges."""

import ctypes

from gemma4_fa4_kernels_b200 import _lib
from test_paged_cache_cpu import _kv8


def test_chunk_plan_wants_the_rows_of_missing_pages():
    a = _kv8()
    rc = _lib.load().g4_kv8_chunk_plan(ctypes.byref(a), 16, 32, 48, 64, None)
    assert rc == _lib.G4_ERR_INVALID and "holes" in _lib.last_error()


def test_the_end_of_a_chunk_wants_them_too():
    for over, code, needle in ((dict(), _lib.G4_ERR_INVALID, "holes"),
                               (dict(holes=0xd000, q=None), _lib.G4_ERR_INVALID, "q is required"),
                               (dict(holes=0xd000, tokens=1 << 24, batch=1024, page_size=128,
                                     pages_per_slot=1 << 23, max_seqlen_k=1 << 30),
                                _lib.G4_ERR_UNSUPPORTED, "tiles")):
        rc = _lib.load().g4_kv8_pad_rows(ctypes.byref(_kv8(**over)), None)
        assert rc == code and needle in _lib.last_error()
