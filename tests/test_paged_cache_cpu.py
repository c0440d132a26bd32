"""8-bit paged KV cache without a GPU: argument checks of the Python surface and
of the C ABI, and the oracle against dense attention."""

import ctypes

import numpy as np
import pytest
import torch

import oracle
from oracle.paged_cache import PagedCache, block_exponent, to_grid

from gemma4_fa4_kernels_b200 import PagedKVCache8, UnsupportedB200Path, _lib


def _cache(**over):
    kw = dict(num_layers=2, num_pages=6, num_kv_heads=4, head_dim=512, max_slots=3,
              pages_per_slot=4, page_size=16, dtype=torch.int8, device="cpu")
    kw.update(over)
    return PagedKVCache8(kw.pop("num_layers"), kw.pop("num_pages"), kw.pop("num_kv_heads"),
                         kw.pop("head_dim"), **kw)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("over,exc,needle", [
    (dict(page_size=24), UnsupportedB200Path, "page_size"),
    (dict(head_dim=128), UnsupportedB200Path, "head_dim"),
    (dict(dtype=torch.bfloat16), ValueError, "int8"),
    (dict(num_pages=0), ValueError, "num_pages"),
    (dict(max_slots=0), ValueError, "max_slots"),
])
def test_constructor_refuses(over, exc, needle):
    with pytest.raises(exc, match=needle):
        _cache(**over)


def test_new_cache_is_empty():
    c = _cache()
    assert c.k.shape == (2, 6, 4, 16, 512) and c.k.dtype == torch.int8
    assert c.capacity == 64 and int(c.refcounts.sum()) == 0 and int(c.tables.max()) == -1
    c.check()  # nothing has failed


def test_from_tensors_refuses_mismatched_parts():
    c = _cache()
    parts = [c.k, c.v, c.k_scale, c.v_scale, c.tables, c.lengths, c.refcounts]
    PagedKVCache8.from_tensors(*parts)
    for i, bad in ((1, c.v[:, :5].contiguous()), (2, c.k_scale.double()), (5, c.lengths[:2]),
                   (6, c.refcounts.long()), (4, c.tables.t()), (1, c.k),
                   (0, c.k.transpose(0, 1))):
        args = list(parts)
        args[i] = bad
        with pytest.raises((ValueError, UnsupportedB200Path)):
            PagedKVCache8.from_tensors(*args)


def test_operand_checks_come_before_the_device():
    c = _cache()
    k, rows = _bf(2, 1, 4, 512), (_i32(0, 1), _i32(0, 0), _i32(1, 1))
    with pytest.raises(IndexError):
        c.append(2, k, k, *rows)
    for bad in (_bf(2, 1, 3, 512), _bf(2, 1, 4, 256), _bf(2, 4, 512), k.float()):
        with pytest.raises(ValueError):
            c.append(0, bad, bad, *rows)
    with pytest.raises(ValueError, match="one shape"):
        c.append(0, k, _bf(2, 2, 4, 512), *rows)
    with pytest.raises(ValueError, match="unit stride"):
        c.append(0, _bf(2, 1, 512, 4).transpose(2, 3), k, *rows)
    with pytest.raises(ValueError, match="starts"):
        c.append(0, k, k, rows[0], rows[1].long(), rows[2])
    with pytest.raises(ValueError, match="entries"):
        c.append(0, k, k, _i32(0), rows[1], rows[2])
    with pytest.raises(UnsupportedB200Path, match="inference"):
        c.append(0, k.clone().requires_grad_(True), k, *rows)
    with pytest.raises(ValueError, match="query heads"):
        c.attention(0, _bf(2, 1, 6, 512), *rows)
    with pytest.raises(ValueError, match="window"):
        c.attention(0, _bf(2, 1, 8, 512), *rows, window=-1)
    with pytest.raises(ValueError, match="max_seqlen_k"):
        c.attention(0, _bf(2, 1, 8, 512), *rows, max_seqlen_k=0)
    with pytest.raises(ValueError, match="more rows than slots"):
        c.attention(0, _bf(4, 1, 8, 512), None, _i32(0, 0, 0, 0), _i32(1, 1, 1, 1))
    with pytest.raises(ValueError, match="counts"):
        c.extend(_i32(0, 1), _i32(1))
    with pytest.raises(ValueError, match="window"):
        c.trim(_i32(0), 0)
    with pytest.raises(UnsupportedB200Path, match="1024"):
        c.free(torch.zeros(1025, dtype=torch.int32))


def test_host_tensors_are_refused_before_any_work():
    c = _cache()
    k, q = _bf(1, 1, 4, 512), _bf(1, 1, 32, 512)
    rows = (_i32(0), _i32(0), _i32(1))
    for call in (lambda: c.append(0, k, k, *rows), lambda: c.read(0, *rows, 1),
                 lambda: c.attention(0, q, *rows), lambda: c.extend(_i32(0), 1),
                 lambda: c.attention(0, _bf(1, 40, 32, 512), *rows),
                 lambda: c.fork(_i32(0), _i32(1)), lambda: c.free(_i32(0)),
                 lambda: c.trim(_i32(0), 16), lambda: c.compact(),
                 lambda: c.copy_pages(_i32(0), _i32(1))):
        with pytest.raises(UnsupportedB200Path, match="CUDA device"):
            call()


def test_empty_calls_need_no_device():
    c = _cache()
    none = torch.zeros(0, dtype=torch.int32)
    c.append(0, _bf(0, 1, 4, 512), _bf(0, 1, 4, 512), none, none, none)
    out, lse = c.attention(0, _bf(0, 1, 32, 512), none, none, none)
    assert out.shape == (0, 1, 32, 512) and lse.shape == (0, 32, 1)
    k, v = c.read(0, none, none, none, 3)
    assert k.shape == (0, 3, 4, 512) == v.shape
    starts, ends = c.extend(none, none)
    assert starts.shape == ends.shape == (0,)
    c.fork(none, none)
    c.free(none)
    c.copy_pages(none, none)


# ---- C ABI ------------------------------------------------------------------------
def _kv8(**over):
    a = _lib.G4Kv8Args()
    a.k_pages, a.v_pages, a.k_scale, a.v_scale, a.tables = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000
    a.starts, a.ends, a.q, a.o, a.lse, a.k, a.v = (0x6000, 0x7000, 0x8000, 0x9000, 0xa000, 0xb000,
                                                   0xc000)
    a.num_pages, a.page_size, a.num_kv_heads, a.head_dim = 8, 64, 4, 512
    a.num_slots, a.pages_per_slot, a.batch, a.tokens = 2, 4, 2, 1
    for f in ("k_stride", "v_stride"):
        getattr(a, f)[:] = [4 * 512, 4 * 512, 512]
    for f in ("q_stride", "o_stride"):
        getattr(a, f)[:] = [32 * 512, 32 * 512, 512]
    a.lse_stride[:] = [32, 1]
    a.num_q_heads, a.max_seqlen_k = 32, 256
    for key, value in over.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("fn,over,code,needle", [
    ("g4_kv8_append", dict(k_pages=None), _lib.G4_ERR_INVALID, "required"),
    ("g4_kv8_append", dict(v_pages=0x1000), _lib.G4_ERR_INVALID, "distinct"),
    ("g4_kv8_append", dict(k_pages=0x1008), _lib.G4_ERR_INVALID, "aligned"),
    ("g4_kv8_append", dict(format=2), _lib.G4_ERR_UNSUPPORTED, "e4m3"),
    ("g4_kv8_append", dict(page_size=8), _lib.G4_ERR_UNSUPPORTED, "page_size"),
    ("g4_kv8_append", dict(batch=1025), _lib.G4_ERR_UNSUPPORTED, "1024"),
    ("g4_kv8_append", dict(tokens=0), _lib.G4_ERR_INVALID, "tokens"),
    ("g4_kv8_append", dict(k=0xb002), _lib.G4_ERR_INVALID, "aligned"),
    ("g4_kv8_append", dict(v=None), _lib.G4_ERR_INVALID, "required"),
    ("g4_kv8_read", dict(v=0xb000), _lib.G4_ERR_INVALID, "second"),
    ("g4_kv8_read", dict(starts=None), _lib.G4_ERR_INVALID, "starts"),
    ("g4_kv8_attn", dict(num_q_heads=30), _lib.G4_ERR_INVALID, "multiple of KV heads"),
    ("g4_kv8_attn", dict(window=-1), _lib.G4_ERR_INVALID, "window"),
    ("g4_kv8_attn", dict(max_seqlen_k=257), _lib.G4_ERR_INVALID, "max_seqlen_k"),
    ("g4_kv8_attn", dict(head_dim=64), _lib.G4_ERR_UNSUPPORTED, "head_dim"),
    ("g4_kv8_attn", dict(lse=None), _lib.G4_ERR_INVALID, "lse"),
    ("g4_kv8_attn", dict(), _lib.G4_ERR_WORKSPACE, "workspace"),
    ("g4_kv8_attn", dict(batch=1024, tokens=1 << 20, workspace=0x10000, workspace_bytes=1 << 40),
     _lib.G4_ERR_UNSUPPORTED, "tiles"),
    # a product of sizes past 64 bits
    ("g4_kv8_attn", dict(batch=1024, tokens=1 << 24, num_q_heads=65535 * 64, num_kv_heads=65535,
                         page_size=16, num_pages=1, pages_per_slot=1 << 26,
                         max_seqlen_k=((1 << 13) - 2) * 128, workspace=0x10000,
                         workspace_bytes=1 << 40), _lib.G4_ERR_UNSUPPORTED, "tiles"),
    ("g4_kv8_attn", dict(batch=1, tokens=1 << 24, num_q_heads=512), _lib.G4_ERR_UNSUPPORTED,
     "columns"),
    ("g4_kv8_pad_rows", dict(o=None), _lib.G4_ERR_INVALID, "o is required"),
])
def test_cache_calls_fail_before_launch(fn, over, code, needle):
    assert getattr(_lib.load(), fn)(ctypes.byref(_kv8(**over)), None) == code
    assert needle in _lib.last_error()


def test_strides_must_be_16_byte_multiples():
    a = _kv8()
    a.k_stride[1] = 4 * 512 + 4
    assert _lib.load().g4_kv8_append(ctypes.byref(a), None) == _lib.G4_ERR_INVALID
    assert "multiples of 8" in _lib.last_error()


def test_pools_of_more_than_31_bits_of_rows_are_refused():
    for fn in ("g4_kv8_append", "g4_kv8_read", "g4_kv8_attn"):
        a = _kv8(num_pages=1 << 25, page_size=16)
        assert getattr(_lib.load(), fn)(ctypes.byref(a), None) == _lib.G4_ERR_UNSUPPORTED
        assert "rows must fit 31 bits" in _lib.last_error()


def test_chunk_plan_refuses_rows_past_31_bits():
    a = _kv8(batch=1024, tokens=1 << 22)
    rc = _lib.load().g4_kv8_chunk_plan(ctypes.byref(a), 16, 32, 48, 64, None)
    assert rc == _lib.G4_ERR_UNSUPPORTED and "31 bits" in _lib.last_error()


def test_workspace_queries_need_no_device():
    lib = _lib.load()
    assert lib.g4_kv8_attn_workspace_bytes(ctypes.byref(_kv8())) > 0
    assert lib.g4_kv8_attn_workspace_bytes(ctypes.byref(_kv8(batch=0))) == 0


def _pages(**over):
    a = _lib.G4PagesArgs()
    a.tables, a.lengths, a.refcounts, a.status = 0x1000, 0x2000, 0x3000, 0x4000
    a.k_pages, a.v_pages, a.k_scale, a.v_scale = 0x5000, 0x6000, 0x7000, 0x8000
    a.num_layers, a.num_pages, a.page_size, a.num_kv_heads, a.head_dim = 2, 9, 16, 4, 256
    a.num_slots, a.pages_per_slot, a.batch = 3, 4, 2
    a.first, a.second, a.counts, a.starts, a.ends = 0x9000, 0xa000, 0xb000, 0xc000, 0xd000
    for key, value in over.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("fn,over,code,needle", [
    ("g4_pages_extend", dict(counts=None), _lib.G4_ERR_INVALID, "counts"),
    ("g4_pages_extend", dict(batch=1025), _lib.G4_ERR_UNSUPPORTED, "1024"),
    ("g4_pages_extend", dict(status=None), _lib.G4_ERR_INVALID, "status"),
    ("g4_pages_fork", dict(second=None), _lib.G4_ERR_INVALID, "children"),
    ("g4_pages_fork", dict(), _lib.G4_ERR_WORKSPACE, "workspace"),
    ("g4_pages_free", dict(batch=0), _lib.G4_ERR_INVALID, "batch"),
    ("g4_pages_free", dict(window=-2), _lib.G4_ERR_INVALID, "window"),
    ("g4_pages_compact", dict(), _lib.G4_ERR_WORKSPACE, "workspace"),
    ("g4_pages_compact", dict(num_pages=1 << 27), _lib.G4_ERR_UNSUPPORTED, "pages"),
    ("g4_pages_copy", dict(k_pages=None), _lib.G4_ERR_INVALID, "k_pages"),
    ("g4_pages_copy", dict(v_pages=0x6008), _lib.G4_ERR_INVALID, "aligned"),
])
def test_page_calls_fail_before_launch(fn, over, code, needle):
    assert getattr(_lib.load(), fn)(ctypes.byref(_pages(**over)), None) == code
    assert needle in _lib.last_error()


# ---- oracle -------------------------------------------------------------------------
def test_oracle_grid_is_the_format():
    x = np.linspace(-460, 460, 4001)
    want = torch.tensor(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(to_grid(x, "e4m3"), want)
    small = np.linspace(-0.1, 0.1, 4001)
    want = torch.tensor(small).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(to_grid(torch.tensor(small).float().double().numpy(), "e4m3"), want)
    assert to_grid(np.array([np.nan, np.inf, -np.inf]), "int8").tolist() == [0, 127, -127]
    assert block_exponent(np.array([448.0]), "e4m3") == 0
    assert block_exponent(np.array([449.0, np.inf]), "e4m3") == 1
    assert block_exponent(np.array([127.0, np.nan]), "int8") == 0
    assert block_exponent(np.zeros(3), "int8") == -100


@pytest.mark.parametrize("window", [0, 20])
def test_oracle_attention_is_the_dense_one(window):
    rng = np.random.default_rng(3)
    c = PagedCache("int8", 1, 8, 2, 16, 8, 2, 4)
    starts, ends = c.extend([1], [50])
    k, v = rng.standard_normal((2, 1, 50, 2, 8))
    c.append(0, k, v, [1], starts, ends)
    kq, vq = c.read(0, [1], [0], [50], 50)
    assert np.abs(kq - k).max() <= np.abs(k).max() / 63.5 / 2  # half a step of at least amax / 127
    q = rng.standard_normal((1, 50, 4, 8))
    out, lse, _, _, _ = c.attention(0, q, [1], [0], [50], window)
    ref, ref_lse = oracle.attention_fwd(q.transpose(0, 2, 1, 3), kq.transpose(0, 2, 1, 3),
                                        vq.transpose(0, 2, 1, 3), sliding_window=window or None)
    assert np.abs(out.transpose(0, 2, 1, 3) - ref).max() < 1e-12
    # that LSE is returned in float32: half a step of it
    assert ref_lse.dtype == np.float32
    assert np.abs(lse - ref_lse).max() <= 2.0 ** -24 * np.abs(lse).max()
