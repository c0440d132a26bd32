"""GPU: the paged cache at the edges of what its calls serve, against the 64-bit oracle."""

import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gemma4_fa4_kernels_b200 import PagedKVCache8, _lib, paged_cache  # noqa: E402
from gemma4_fa4_kernels_b200.paged_cache import DIRECT_COLUMNS  # noqa: E402
from test_gpu_paged_cache import Pair, bf16, check_attention, f64, i32  # noqa: E402

BAD = _lib.G4_PAGES_BAD_INDEX


# ------------------------------------------------------------------------------------
# missing pages under a chunk of a prompt
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads,group,window", [(512, 1, 8, 0), (512, 2, 8, 60), (256, 2, 2, 0),
                                                 (256, 2, 4, 50), (512, 1, 3, 0)])
def test_chunks_mask_missing_pages(fmt, d, heads, group, window):
    rng = np.random.default_rng(41)
    tokens = DIRECT_COLUMNS[d] // group + 3
    lens = [tokens + 90, tokens + 40, 150, tokens + 20, tokens, 40]
    p = Pair(fmt, heads=heads, d=d, page=16, pages=80, slots=7, per_slot=20)
    p.fill(list(range(6)), lens, rng)
    p.ref.tables[0, 1:3] = -1                       # a hole before the chunk
    p.ref.tables[1, :] = -1                         # nothing at all
    p.ref.tables[2, (lens[2] - 20) // 16] = 80      # a bad id under the chunk's own tokens
    p.ref.tables[3, 0] = -1                         # a leading hole
    p.ref.tables[5, (lens[5] - 1) // 16] = -1       # the last page: some queries' own keys
    p.dev.tables.copy_(i32(p.ref.tables))
    n = [tokens, tokens - 2, 30, tokens, tokens, 7, 0, 3]
    rows = [0, 1, 2, 3, 4, 5, 6, 9]
    ends = [*lens, 0, 5]
    q = 0.2 * rng.standard_normal((8, tokens, heads * group, d))
    poison = torch.full((1 << 25,), float("nan"), device="cuda")  # what the next buffers hold
    del poison
    check_attention(p, 0, q, rows, [e - m for e, m in zip(ends, n)], ends, window=window)


def test_a_hole_means_the_same_on_both_sides_of_the_direct_bound():
    """Three of seven pages are missing; the last 32 of 33 tokens see what 32 tokens see."""
    rng = np.random.default_rng(42)
    p = Pair("e4m3", heads=1, d=512, page=16, pages=12, slots=1, per_slot=12)
    p.fill([0], [100], rng)
    p.ref.tables[0, 1:4] = -1
    p.dev.tables.copy_(i32(p.ref.tables))
    q = 0.05 * rng.standard_normal((1, 33, 8, 512))
    many = check_attention(p, 0, q, [0], [67], [100])
    few = check_attention(p, 0, q[:, 1:], [0], [68], [100])
    # BF16 outputs (2^-8 of each) and a chunk's P (2^-7 of sum p |v|, which is up to 1.5 max)
    assert np.abs(many[:, 1:] - few).max() <= 2.0 ** -5 * np.abs(few).max()


def test_a_chunk_over_trimmed_pages():
    """Positions that are run again after a trim see what is left."""
    rng = np.random.default_rng(43)
    p = Pair("int8", heads=2, d=256, page=16, pages=40, slots=2, per_slot=20)
    p.fill([0, 1], [250, 100], rng)
    p.ref.free([0], 100)
    p.dev.trim(i32([0]), 100)
    q = 0.2 * rng.standard_normal((2, 80, 4, 256))
    check_attention(p, 0, q, [0, 1], [170, 20], [250, 100], window=140)
    p.same()


def test_captured_chunks_see_the_pages_of_their_replay():
    rng = np.random.default_rng(46)
    p = Pair("e4m3", heads=2, d=256, page=16, pages=40, slots=2, per_slot=20)
    p.fill([0, 1], [200, 90], rng)
    q, _ = bf16(0.2 * rng.standard_normal((2, 40, 4, 256)))
    args = (0, q, i32([0, 1]), i32([160, 55]), i32([200, 90]))
    p.dev.attention(*args)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(p.dev.attention(*args))
    for hole in (None, (0, 3), (1, 5), None):
        p.dev.tables.copy_(i32(p.ref.tables))
        if hole:
            p.dev.tables[hole] = -1
        want = p.dev.attention(*args)
        for g in graphs:
            g.replay()
        for out in outs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


# ------------------------------------------------------------------------------------
# rows out of range
# ------------------------------------------------------------------------------------
def _calls(p, tokens_of):
    """Every call that takes rows, at its direct, wide and chunk sizes."""
    d, h = p.ref.k.shape[4], p.ref.k.shape[2]

    def append(rows):
        k, _ = bf16(np.ones((len(rows[0]), 3, h, d)))
        p.dev.append(0, k, k.clone(), *map(i32, rows))

    def read(rows):
        k, v = p.dev.read(0, *map(i32, rows), 3)
        assert not k[1].any() and not v[1].any()

    def attention(rows, tokens, **kw):
        q, _ = bf16(np.ones((len(rows[0]), tokens, 2 * h, d)))
        out, lse = p.dev.attention(0, q, *map(i32, rows), **kw)
        assert not out[1].any() and torch.isneginf(lse[1]).all()

    calls = {"append": append, "read": read}
    for name, tokens in tokens_of.items():
        calls[name] = lambda rows, t=tokens, **kw: attention(rows, t, **kw)
    return calls


@pytest.mark.parametrize("call", ["append", "read", "decode", "wide", "chunk"])
@pytest.mark.parametrize("per_slot", [2, 60])
def test_rows_out_of_range_are_reported(call, per_slot):
    """Row 1 of two: a bad slot, a negative position, a position past the table."""
    p = Pair("int8", heads=1, d=256, page=16, pages=8, slots=3, per_slot=per_slot)
    p.extend([0, 1, 2], [20, 20, 20])
    run = _calls(p, {"decode": 1, "wide": 9, "chunk": 40})[call]
    cap = 16 * per_slot
    for slot, start, end in ((-1, 0, 3), (3, 0, 1), (1 << 30, 5, 7), (1, -1, 1), (1, -5, -4),
                             (1, cap - 1, cap + 1), (1, cap, cap + 2), (2, 0, 2 ** 31 - 1)):
        assert int(p.dev.status.item()) == 0
        run(([0, slot], [0, start], [1, end]))
        assert int(p.dev.status.item()) == BAD, (slot, start, end)
        with pytest.raises(RuntimeError, match="out of range"):
            p.dev.check()
    # a row that asks for nothing is none of these, whatever its slot
    for slot, start, end in ((1, 4, 4), (1, 0, 0), (-1, 0, 0), (9, 7, 7), (1, 5, 2)):
        run(([0, slot], [0, start], [1, end]))
        p.dev.check()


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_rows_beyond_the_bound_of_a_call_are_reported(tokens):
    p = Pair("e4m3", heads=1, d=256, page=16, pages=12, slots=2, per_slot=60)
    p.fill([0, 1], [60, 60], np.random.default_rng(44))
    run = _calls(p, {"a": tokens})["a"]
    run(([0, 1], [9, 50], [10, 51]), max_seqlen_k=50)
    with pytest.raises(RuntimeError, match="out of range"):
        p.dev.check()
    q, _ = bf16(np.ones((2, tokens, 2, 256)))
    p.dev.attention(0, q, i32([0, 1]), i32([9, 49]), i32([10, 50]), max_seqlen_k=50)
    p.dev.check()


def test_rows_that_ask_for_nothing_may_repeat_a_slot():
    """The padding of a batch, before and behind the rows that it lists again."""
    rng = np.random.default_rng(45)
    p = Pair("e4m3")
    starts, ends = p.extend([0, 2], [20, 5])
    k, v = rng.standard_normal((2, 5, 20, 2, 256))
    p.append(0, k, v, [0, 0, 2, 0, 2], [0, starts[0], starts[1], 20, 3],
             [0, ends[0], ends[1], 20, 1])
    assert p.ref.status == 0 and p.ref.k[0, 0].any()
    p.same()
    p.append(0, v, k, [2, 0, 2, 0, 2], [0, 3, 1, 4, 3], [0, 9, 4, 5, 3])  # row 3 is a repeat
    assert p.ref.status == BAD
    p.same()


# ------------------------------------------------------------------------------------
# a pool that runs out
# ------------------------------------------------------------------------------------
def test_a_refused_row_leaves_its_pages_to_the_rows_behind_it():
    p = Pair("int8", pages=5, slots=6, per_slot=12, page=16)
    p.extend([0, 1], [160, 16])                 # ten pages are not there, one is
    assert p.ref.lengths.tolist() == [0, 16, 0, 0, 0, 0]
    assert p.ref.status == _lib.G4_PAGES_EXHAUSTED
    p.same()
    p.extend([2, 3, 0, 4, 5], [70, 48, 33, 0, 16])   # 5, 3, 3, 0, 1 of four free pages
    assert p.ref.lengths.tolist() == [0, 16, 0, 48, 0, 16]
    p.same()


@pytest.mark.parametrize("seed", range(6))
def test_a_scarce_pool_serves_what_fits_in_order(seed):
    rng = np.random.default_rng(70 + seed)
    rows = int(rng.choice([3, 33, 200, 1024]))
    p = Pair("int8", heads=1, pages=int(rng.integers(1, 2 * rows)), slots=rows, per_slot=6, page=16,
             seed=seed)
    for _ in range(4):
        order = rng.permutation(rows)[:int(rng.integers(1, rows + 1))]
        p.extend(list(order), list(rng.integers(0, 50, len(order))))
        p.same()
        gone = rng.choice(rows, max(1, rows // 4), replace=False)
        p.ref.free(list(gone))
        p.dev.free(i32(gone))
    p.same()


def test_rows_that_ask_for_more_than_31_bits_of_pages_together():
    per_slot, rows = (2 ** 31 - 1 - 65536) // 16, 17
    tables = torch.full((rows, per_slot), -1, dtype=torch.int32, device="cuda")
    codes = [torch.zeros(1, 3, 1, 16, 256, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.ones(1, 3, 1, device="cuda") for _ in range(2)]
    cache = PagedKVCache8.from_tensors(*codes, *scales, tables, i32([0] * rows), i32([0] * 3))
    counts = [16 * per_slot] * (rows - 1) + [33]
    starts, ends = cache.extend(i32(range(rows)), i32(counts))
    assert starts.tolist() == [0] * rows and ends.tolist() == [0] * (rows - 1) + [33]
    assert cache.lengths.tolist() == ends.tolist()
    assert cache.refcounts.tolist() == [1, 1, 1] and tables[-1, :4].tolist() == [0, 1, 2, -1]
    with pytest.raises(RuntimeError, match="too few free pages"):
        cache.check()
    del tables, cache
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------
# lengths that were lowered from outside: rejected drafts
# ------------------------------------------------------------------------------------
def _lower(p, slots, lengths):
    for s, n in zip(slots, lengths):
        p.ref.lengths[s] = n
        p.dev.lengths[s] = n


def test_pages_behind_a_lowered_length_are_used_again_and_given_back():
    rng = np.random.default_rng(50)
    p = Pair("e4m3", pages=20, slots=5, per_slot=150, page=16)
    p.fill([0, 1, 2], [30, 33, 16], rng)
    for step in range(6):                       # five drafts a step, most of them rejected
        starts, ends = p.fill([0, 1, 2], [5, 5, 5], rng)
        q = 0.3 * rng.standard_normal((3, 5, 4, 256))
        check_attention(p, 0, q, [0, 1, 2], starts, ends)
        _lower(p, [0, 1, 2], [s + 1 + step % 3 for s in starts])
        p.same()
    assert int((p.ref.refcounts > 0).sum()) == sum(int((p.ref.tables[s] >= 0).sum()) for s in range(5))
    _lower(p, [0, 2], [0, 17])                  # a whole prompt taken back
    p.fill([0, 2], [100, 20], rng)
    p.same()
    _lower(p, [0], [3])
    p.ref.free([0, 1, 0, 2])
    p.dev.free(i32([0, 1, 0, 2]))
    p.same()
    assert not p.ref.refcounts.any()


def test_many_pages_behind_a_lowered_length_are_given_back():
    p = Pair("int8", heads=1, pages=420, slots=2, per_slot=400, page=16)
    p.extend([0, 1], [6000, 100])
    _lower(p, [0], [20])
    p.ref.free([0, 0])
    p.dev.free(i32([0, 0]))
    p.same()
    assert int(p.ref.refcounts.sum()) == 7


def test_shared_pages_behind_a_lowered_length_are_not_written():
    rng = np.random.default_rng(51)
    p = Pair("e4m3", pages=20, slots=6, per_slot=8, page=16)
    p.fill([0, 1], [48, 20], rng)
    p.ref.fork([0], [2])
    p.dev.fork(i32([0]), i32([2]))
    before = f64(p.dev.read(0, i32([2]), i32([0]), i32([48]), 48)[0])
    for n in (30, 16, 0):                       # inside a shared page, at the start of one
        _lower(p, [0], [n])
        starts, ends = p.extend([0, 1], [4, 4])
        assert starts[0] == ends[0] and p.ref.status == BAD
        _lower(p, [1], [20])
        p.same()
    assert np.array_equal(before, f64(p.dev.read(0, i32([2]), i32([0]), i32([48]), 48)[0]))
    p.ref.fork([1], [0])                        # a child that still holds pages is not empty
    p.dev.fork(i32([1]), i32([0]))
    p.same()
    p.ref.free([0])
    p.dev.free(i32([0]))
    p.fill([2, 1], [1, 1], rng)                 # the pages are the child's alone now
    p.same()


@pytest.mark.parametrize("seed", range(6))
def test_random_page_traffic_with_lowered_lengths(seed):
    rng = np.random.default_rng(900 + seed)
    pages = int(rng.integers(8, 90))
    p = Pair("int8", heads=1, pages=pages, slots=12, per_slot=9, page=16, seed=seed)
    for _ in range(40):
        act, n = rng.integers(0, 8), int(rng.integers(1, 8))
        slots = [int(s) for s in rng.choice(14, n, replace=False) - 1]
        if act <= 1:
            p.fill(slots, [int(x) for x in rng.integers(0, 60, n)], rng)
        elif act == 2:
            p.extend(slots, [int(x) for x in rng.integers(-1, 90, n)])
        elif act == 3:
            kids = [int(x) for x in rng.choice(12, n, replace=False)]
            p.ref.fork(slots, kids)
            p.dev.fork(i32(slots), i32(kids))
        elif act == 4:
            window = int(rng.choice([0, 0, 20, 60]))
            p.ref.free(slots, window)
            p.dev.trim(i32(slots), window) if window else p.dev.free(i32(slots))
        elif act == 5:
            p.ref.compact()
            p.dev.compact()
        else:
            live = [s for s in slots if 0 <= s < 12 and p.ref.lengths[s] > 0]
            # (to nothing only where the first page is still listed: an empty slot is a child)
            _lower(p, live, [int(rng.integers(p.ref.tables[s, 0] < 0, p.ref.lengths[s] + 1))
                             for s in live])
        p.same()


# ------------------------------------------------------------------------------------
# the largest values
# ------------------------------------------------------------------------------------
LARGEST = float(torch.finfo(torch.bfloat16).max)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_the_largest_values_stay_finite(fmt):
    """Up to the largest BF16 value: codes and scales as the oracle's, read back finite
    and off by at most 2^-4 of the value (e4m3) or half a step (int8)."""
    rng = np.random.default_rng(60)
    p = Pair(fmt, pages=12, slots=6, per_slot=4, page=16, d=256, heads=2)
    x = LARGEST * rng.uniform(-1, 1, (5, 20, 2, 256))
    x[0, 0, :, 0], x[1, 17, :, 3] = LARGEST, -LARGEST
    x[2] *= 0.875                                 # up to 448 * 2^119
    x[2, 5, :, 9] = 448 * 2.0 ** 119
    x[3, 1, :, 7], x[3, 2, :, 8], x[3, 3, :, 9] = LARGEST, np.inf, np.nan
    x[4], x[4, 4] = 1e-3 * x[4] / LARGEST, LARGEST  # ordinary ones under the largest scale
    k, hk = bf16(x)
    starts, ends = p.extend(list(range(5)), [20] * 5)
    p.append(0, (k, hk), (-k, -hk), list(range(5)), starts, ends)
    p.same()
    p.fill(list(range(5)), [1] * 5, rng, magnitude=1e30)  # joins their pages
    p.same()
    got, _ = p.dev.read(0, i32(range(5)), i32(starts), i32(ends), 20)
    got = f64(got)
    assert np.isfinite(got).all()
    ok = np.isfinite(hk) & (np.abs(hk) >= 2.0 ** 120)
    err = np.abs(got - hk)[ok] / np.abs(hk)[ok]
    if fmt == "e4m3":
        assert err.max() <= 2.0 ** -4
    else:
        assert np.abs(got - hk)[ok].max() <= 2.0 ** 120
    assert (np.abs(got[~np.isfinite(hk)]) <= LARGEST).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tokens", [1, 3, 9])
def test_attention_over_the_largest_values(fmt, tokens):
    """Decode and both wide shapes; V up to the largest BF16 value."""
    rng = np.random.default_rng(61)
    n = 150
    p = Pair(fmt, heads=1, d=512, page=16, pages=12, slots=1, per_slot=10)
    starts, ends = p.extend([0], [n])
    k = rng.standard_normal((1, n, 1, 512))
    v = LARGEST * rng.uniform(-1, 1, (1, n, 1, 512))
    v[0, :, 0, 5] = LARGEST
    p.append(0, k, v, [0], starts, ends)
    q = 0.1 * rng.standard_normal((1, tokens, 8, 512))
    got = check_attention(p, 0, q, [0], [n - tokens], [n])
    assert np.isfinite(got).all()


# ------------------------------------------------------------------------------------
# the largest windows
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5])
def test_windows_past_31_bits_reach_every_key(window):
    rng = np.random.default_rng(62)
    p = Pair("int8", heads=2, d=256, page=16, pages=30, slots=2, per_slot=12)
    p.fill([0, 1], [150, 40], rng)
    for tokens in (1, 9, 40):
        q = 0.3 * rng.standard_normal((2, tokens, 4, 256))
        at = [0, 1], [150 - tokens, 40 - tokens], [150, 40]
        dq, _ = bf16(q)
        want = p.dev.attention(0, dq, *map(i32, at))
        got = p.dev.attention(0, dq, *map(i32, at), window=window)
        # another mask may run another kernel of the packed forward: P's 8 bits at most
        assert (got[0] - want[0]).abs().max() <= 2.0 ** -6 * want[0].abs().max()
        assert (got[1] - want[1]).abs().max() <= 1e-4
    p.dev.trim(i32([0, 1]), window)
    p.same()


# ------------------------------------------------------------------------------------
# memory
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("most", [None, 1 << 30])
def test_the_copy_of_a_chunk_is_bounded_by_memory_not_by_rows(most, monkeypatch):
    """64 rows of 40 tokens in slots of 32768 tokens: the bound alone would make the copy
    of their keys 17 GB, and the forward's scratch 22."""
    if most:
        monkeypatch.setattr(paged_cache, "CHUNK_COPY_BYTES", most)
    rng = np.random.default_rng(63)
    rows, tokens = 64, 40
    cache = PagedKVCache8(1, 64 * 4, 4, 512, max_slots=rows + 1, pages_per_slot=512, page_size=64)
    lens = i32(rng.integers(tokens, 200, rows))
    slots = i32(rng.permutation(rows))
    starts, ends = cache.extend(slots, lens)
    k, _ = bf16(rng.standard_normal((rows, 200, 4, 512)))
    cache.append(0, k, -k, slots, starts, ends)
    q, _ = bf16(0.2 * rng.standard_normal((rows, tokens, 32, 512)))
    tight, tight_lse = cache.attention(0, q, slots, ends - tokens, ends, max_seqlen_k=200)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = cache.attention(0, q, slots, ends - tokens, ends)
    torch.cuda.synchronize()
    # the forward's scratch is about 1.4 times the copy
    assert torch.cuda.max_memory_allocated() - before < 2.5 * paged_cache.CHUNK_COPY_BYTES
    assert out.shape == tight.shape and lse.shape == tight_lse.shape
    # another bound may run another kernel of the packed forward: P's 8 bits at most
    assert (out - tight).abs().max() <= 2.0 ** -6 * tight.abs().max()
    assert (lse - tight_lse).abs().max() <= 1e-4
    every = cache.attention(0, q, None, *_by_slot(slots, ends - tokens, ends))
    order = slots.long().argsort()
    want = cache.attention(0, q, i32(range(rows)), (ends - tokens)[order], ends[order])
    assert torch.equal(every[0], want[0]) and torch.equal(every[1], want[1])
    cache.check()
    torch.cuda.empty_cache()


def _by_slot(slots, starts, ends):
    order = slots.long().argsort()
    return starts[order], ends[order]


# ------------------------------------------------------------------------------------
# host threads
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 5])
def test_host_threads_with_batches_of_different_size(tokens):
    """Calls of one kernel from six host threads, 1024 rows in three, one in the others."""
    caches, args = [], []
    for rows in (1024, 1):
        cache = PagedKVCache8(1, rows, 1, 512, max_slots=rows, pages_per_slot=100, page_size=16)
        slots = i32(range(rows))
        starts, ends = cache.extend(slots, i32([7] * rows))
        k, _ = bf16(np.ones((rows, 7, 1, 512)))
        cache.append(0, k, k.clone(), slots, starts, ends)
        q, _ = bf16(0.01 * np.ones((rows, tokens, 8, 512)))
        caches.append(cache)
        args.append((0, q, slots, ends - tokens, ends))
    want = [c.attention(*a) for c, a in zip(caches, args)]
    torch.cuda.synchronize()
    errors, last = [], [None] * 6
    go = threading.Barrier(6)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            go.wait(30)
            with torch.cuda.stream(stream):
                for _ in range(3000):  # no waits: the launch queue is full
                    last[i] = caches[i % 2].attention(*args[i % 2])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    for i, (out, lse) in enumerate(last):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])
