"""8-bit paged KV cache without a GPU: what its calls refuse at the edges."""

import ctypes

import numpy as np
import pytest
import torch

from oracle.paged_cache import MAX_EXP, block_exponent, to_grid

from gemma4_fa4_kernels_b200 import _lib
from test_paged_cache_cpu import _kv8


def test_chunk_plan_wants_the_rows_of_missing_pages():
    a = _kv8()
    rc = _lib.load().g4_kv8_chunk_plan(ctypes.byref(a), 16, 32, 48, 64, None)
    assert rc == _lib.G4_ERR_INVALID and "holes" in _lib.last_error()


def test_equal_runs_have_a_place_for_their_parts():
    """Any call that is not one CTA per item needs the parts' workspace and their merge."""
    lib = _lib.load()
    size = lambda **o: lib.g4_kv8_attn_workspace_bytes(ctypes.byref(_kv8(**o)))  # noqa: E731
    assert size(max_seqlen_k=64) == 256  # one CTA per item
    for over in (dict(batch=200, num_slots=200, max_seqlen_k=1), dict(pages_per_slot=64, max_seqlen_k=4096)):
        # two parts per run and CTA, of 8 columns of 512 floats
        assert size(**over) > 148 * 6 * 2 * 8 * 512 * 4


def test_the_end_of_a_chunk_wants_them_too():
    for over, code, needle in ((dict(), _lib.G4_ERR_INVALID, "holes"),
                               (dict(holes=0xd000, q=None), _lib.G4_ERR_INVALID, "q is required"),
                               (dict(holes=0xd000, tokens=1 << 24, batch=1024, page_size=128,
                                     pages_per_slot=1 << 23, max_seqlen_k=1 << 30),
                                _lib.G4_ERR_UNSUPPORTED, "tiles")):
        rc = _lib.load().g4_kv8_pad_rows(ctypes.byref(_kv8(**over)), None)
        assert rc == code and needle in _lib.last_error()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_values_are_finite_and_close(fmt):
    """Every positive BF16 value alone in a block: off by half a step of int8, by 2^-4 of
    itself (or half the smallest step) in e4m3, the largest ones included."""
    bits = torch.arange(1, 0x7F80, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16).double().numpy()
    e = np.array([block_exponent(np.array([v]), fmt) for v in x])
    codes = np.array([float(to_grid(np.array([v / 2.0 ** k]), fmt, k)[0]) for v, k in zip(x, e)])
    assert e.max() == MAX_EXP[fmt] and np.isfinite(np.float32(codes * 2.0 ** e)).all()
    assert (codes * 2.0 ** e <= float(torch.finfo(torch.bfloat16).max)).all()
    y = x / 2.0 ** e
    assert (np.abs(codes - y) <= (0.5 if fmt == "int8" else np.maximum(y / 16, 2.0 ** -10))).all()
