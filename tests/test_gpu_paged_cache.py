"""GPU parity of the 8-bit paged KV cache against the 64-bit oracle.

Codes, scales, tables, counters and copied bytes have to be equal.  Attention
outputs are held to the roundings that the kernels make, see ``bounds``.
"""

import numpy as np
import pytest
import torch

from oracle import paged_cache as ref

pytestmark = pytest.mark.gpu

cuda = pytest.importorskip("torch").cuda
if not cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gemma4_fa4_kernels_b200 import PagedKVCache8, _lib  # noqa: E402
from gemma4_fa4_kernels_b200.paged_cache import DIRECT_COLUMNS  # noqa: E402

DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def f64(t):
    return t.double().cpu().numpy()


def bf16(x):
    """(tensor on the device, the values it holds)."""
    t = torch.tensor(x, dtype=torch.float32).to(torch.bfloat16)
    return t.cuda(), t.double().numpy()


class Pair:
    """The cache and the oracle, driven by the same calls."""

    def __init__(self, fmt, layers=1, pages=24, heads=2, page=16, d=256, slots=6, per_slot=8, seed=0):
        self.fmt = fmt
        self.dev = PagedKVCache8(layers, pages, heads, d, max_slots=slots, pages_per_slot=per_slot,
                                 page_size=page, dtype=DTYPES[fmt])
        self.ref = ref.PagedCache(fmt, layers, pages, heads, page, d, slots, per_slot)
        # recycled pages: old codes everywhere, and scales that are no power of two
        rng = np.random.default_rng(seed + 1000)
        for codes, mine in ((self.dev.k, self.ref.k), (self.dev.v, self.ref.v)):
            x = rng.integers(-100, 100, codes.shape)
            mine[:] = ref.to_grid(x.astype(float), fmt)
            codes.copy_(torch.tensor(mine, dtype=torch.float32).to(DTYPES[fmt]))
        for s, mine in ((self.dev.k_scale, self.ref.k_scale), (self.dev.v_scale, self.ref.v_scale)):
            mine[:] = 3.0
            s.fill_(3.0)

    def extend(self, slots, counts):
        starts, ends = self.ref.extend(slots, counts)
        ds, de = self.dev.extend(i32(slots), i32(counts))
        assert ds.tolist() == list(starts) and de.tolist() == list(ends)
        return starts, ends

    def append(self, layer, k, v, slots, starts, ends):
        dk, hk = k if isinstance(k, tuple) else bf16(k)
        dv, hv = v if isinstance(v, tuple) else bf16(v)
        self.ref.append(layer, hk, hv, list(slots), list(starts), list(ends))
        self.dev.append(layer, dk, dv, i32(slots), i32(starts), i32(ends))

    def same(self):
        for name in ("tables", "lengths", "refcounts"):
            assert np.array_equal(getattr(self.dev, name).cpu().numpy(), getattr(self.ref, name)), name
        for name in ("k", "v"):
            got = getattr(self.dev, name).float().cpu().double().numpy()
            assert np.array_equal(got, getattr(self.ref, name)), name
        for name in ("k_scale", "v_scale"):
            assert np.array_equal(f64(getattr(self.dev, name)), getattr(self.ref, name)), name
        assert int(self.dev.status.item()) == self.ref.status

    def fill(self, slots, counts, rng, layer=0, magnitude=1.0):
        starts, ends = self.extend(slots, counts)
        n = max(1, max(counts))
        h, d = self.ref.k.shape[2], self.ref.k.shape[4]
        k = magnitude * rng.standard_normal((len(slots), n, h, d))
        v = magnitude * rng.standard_normal((len(slots), n, h, d))
        self.append(layer, k, v, slots, starts, ends)
        return starts, ends


def bounds(out, lse, spread, grain, size, d, p_bits, p_step):
    """Largest errors of O and LSE.

    S: d products summed in fp32, at most d/16 + 3 rounded (or truncated: 2^-23)
    additions of partial sums no larger than size = sum |q k|, and four roundings
    around them (scales, log2(e), LSE); exp2 and log2 good to 2^-22 with an argument
    rounded to 2^-24 of a few hundred at most (2^-15).  P is rounded to p_bits
    significant bits, and all of these move O by at most twice (numerator and
    denominator) their share of sum p |v|.  O itself is rounded to bf16: 2^-8 of it,
    plus the smallest bf16 step.  The kernels hold 2^11 s_v P (more than 8 columns:
    2^5 s_v P) in fp16 relative to its maximum, whose steps do not shrink below 2^-24:
    half a step is 2^-36 (2^-30) of the largest s_v P, for every key, which grain =
    max(p s_v) sum |v8| adds up."""
    ds = (d / 16 + 7) * 2.0 ** -23 * size + 2.0 ** -15
    o = 2.0 ** -8 * np.abs(out) + (2.0 ** -p_bits + 2 * ds.transpose(0, 2, 1)[..., None]) * spread
    o = o + p_step * grain
    return o + 2.0 ** -126, ds + 2.0 ** -21 * np.abs(np.where(np.isfinite(lse), lse, 0))


def check_attention(pair, layer, q, slots, starts, ends, **kw):
    dq, hq = q if isinstance(q, tuple) else bf16(q)
    out, lse, spread, grain, size = pair.ref.attention(layer, hq, list(slots), list(starts), list(ends),
                                                kw.get("window", 0),
                                                kw.get("max_seqlen_k") or 1 << 40)
    got, got_lse = pair.dev.attention(layer, dq, i32(slots), i32(starts), i32(ends), **kw)
    assert got.shape == dq.shape and got.dtype == torch.bfloat16
    assert got_lse.shape == (dq.shape[0], dq.shape[2], dq.shape[1])
    d, group = dq.shape[3], dq.shape[2] // pair.ref.k.shape[2]
    direct = dq.shape[1] * group <= DIRECT_COLUMNS[d]
    # the chunk path holds K and V (when scales are no powers of two) and P in bf16
    o_tol, l_tol = bounds(out, lse, spread, grain, size, d, 11 if direct else 7,
                          2.0 ** -36 if dq.shape[1] * group <= 8 else 2.0 ** -30)
    got, got_lse = f64(got), f64(got_lse)
    assert np.array_equal(np.isneginf(got_lse), np.isneginf(lse)), "masked rows differ"
    fin = np.isfinite(lse)
    over = ~(np.abs(got - out) <= o_tol)  # (row, token, head, dim); NaN is over
    assert not over.any(), (int(over.sum()), np.argwhere(over)[:8].tolist())
    over = ~(np.abs(got_lse[fin] - lse[fin]) <= l_tol[fin])
    assert not over.any(), (int(over.sum()), np.argwhere(fin)[over][:8].tolist())
    dead = ~fin.transpose(0, 2, 1)
    assert np.all(got[dead] == 0)
    return got


# ------------------------------------------------------------------------------------
# append and read
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("page,heads,d", [(16, 2, 256), (32, 1, 512), (64, 3, 256), (128, 4, 512)])
def test_append_codes_and_scales(fmt, page, heads, d):
    rng = np.random.default_rng(page + d)
    p = Pair(fmt, heads=heads, page=page, d=d, pages=20, per_slot=6)
    # a prompt that ends inside a page, one that fills its pages, one token, none
    p.fill([4, 0, 2, 5], [page + 7, 2 * page, 1, 0], rng)
    p.same()
    # larger tokens join the page (its scale grows), smaller ones (it stays)
    p.fill([4, 0, 2], [3, 1, page + 1], rng, magnitude=37.0)
    p.same()
    for _ in range(3):
        p.fill([2, 4, 0], [1, 1, 1], rng, magnitude=1e-3)
    p.fill([2, 4], [page - 1, 2], rng, magnitude=3e4)
    p.same()
    lens = [int(p.ref.lengths[s]) for s in (4, 0, 2, 5)]
    k, v = p.dev.read(0, i32([4, 0, 2, 5]), i32([0, 3, 1, 0]), i32(lens), max(lens))
    hk, hv = p.ref.read(0, [4, 0, 2, 5], [0, 3, 1, 0], lens, max(lens))
    assert np.array_equal(f64(k), hk) and np.array_equal(f64(v), hv)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_extreme_values(fmt):
    rng = np.random.default_rng(5)
    p = Pair(fmt, page=16, d=256, heads=2)
    x = rng.standard_normal((6, 20, 2, 256))
    x[0] = 0.0                                # zeros: the least scale
    x[1, 3, 0, 7], x[1, 4, 1, 0] = np.nan, np.inf
    x[1, 18] = np.nan                         # a page of NaN and a few numbers
    x[2] *= 1e38
    x[3] *= 1e-38
    x[4, :16, 0] = 448.0                      # on the format's edge, and a step above
    x[4, :16, 1, 5], x[4, 16:] = 127.0, 450.0
    x[5] = np.where(x[5] > 0, np.inf, -np.inf)
    slots = list(range(6))
    starts, ends = p.extend(slots, [20] * 6)
    p.append(0, x, -x, slots, starts, ends)
    p.same()
    # the next token is ordinary: zeros stay zeros under the larger scale
    p.fill(slots, [1] * 6, rng)
    p.same()


def test_append_strides_padding_and_layers():
    rng = np.random.default_rng(6)
    p = Pair("e4m3", layers=3, heads=2, d=256)
    starts, ends = p.extend([1, 3, 0], [5, 2, 9])
    big, _ = bf16(rng.standard_normal((3, 9, 3, 2, 256)))  # (rows, tokens, q/k/v, heads, d)
    k, v = big[:, :, 1], big[:, :, 2]
    k[1, 2:] = float("nan")  # padding of row 1 is never read into the page
    p.append(1, (k, f64(k)), (v, f64(v)), [1, 3, 0], starts, ends)
    p.same()
    bh, _ = bf16(rng.standard_normal((3, 2, 9, 256)))      # heads before tokens
    t = bh.transpose(1, 2)
    p.append(2, (t, f64(t)), (v, f64(v)), [1, 3, 0], starts, ends)
    p.same()


def test_append_leaves_out_what_it_cannot_place():
    rng = np.random.default_rng(7)
    p = Pair("int8")
    starts, ends = p.extend([0, 1, 2, 3], [20, 20, 20, 20])
    p.ref.tables[1, 1] = -1
    p.ref.tables[2, 0] = 10 ** 6
    p.dev.tables.copy_(i32(p.ref.tables))
    k, v = rng.standard_normal((2, 8, 20, 2, 256))
    # missing and out-of-range pages, the same slot twice, bad slots and positions
    p.append(0, k, v, [0, 1, 2, 0, 9, -1, 3, 4], [*starts[:3], 0, 0, 0, -3, 130],
             [*ends[:3], 20, 20, 20, 17, 150])
    assert p.ref.status == _lib.G4_PAGES_BAD_INDEX
    p.same()
    with pytest.raises(RuntimeError, match="out of range"):
        p.dev.check()
    p.dev.check()
    # reading the holes gives zeros
    k, v = p.dev.read(0, i32([1, 2, 9]), i32([0, 0, 0]), i32([20, 20, 20]), 24)
    hk, hv = p.ref.read(0, [1, 2, 9], [0, 0, 0], [20, 20, 20], 24)
    assert np.array_equal(f64(k), hk) and np.array_equal(f64(v), hv)


# ------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads,group,page", [(256, 2, 2, 16), (512, 1, 8, 64), (512, 2, 3, 32),
                                                 (256, 1, 16, 128), (256, 3, 1, 32)])
@pytest.mark.parametrize("window", [0, 40])
def test_decode_lengths(fmt, d, heads, group, page, window):
    """One query token per row at lengths around tiles, pages and the window."""
    rng = np.random.default_rng(d + heads + page)
    lens = [1, 2, 15, 16, 17, 39, 40, 41, 56, 127, 128, 129, 300]
    n = len(lens)
    p = Pair(fmt, heads=heads, page=page, d=d, pages=2 * n + sum(-(-x // page) for x in lens),
             slots=n, per_slot=-(-300 // page))
    p.fill(list(range(n)), lens, rng)
    q = 0.3 * rng.standard_normal((n, 1, heads * group, d))
    order = rng.permutation(n)
    ends = [lens[i] for i in order]
    check_attention(p, 0, q, order, [e - 1 for e in ends], ends, window=window)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads,group", [(256, 2, 2), (512, 1, 8), (512, 1, 5)])
@pytest.mark.parametrize("tokens,window", [(2, 0), (5, 0), (5, 33), (9, 7)])
def test_several_queries_causal_and_padded(fmt, d, heads, group, tokens, window):
    rng = np.random.default_rng(tokens)
    lens = [9, 30, 64, 100, 33]
    p = Pair(fmt, heads=heads, d=d, page=32, pages=30, slots=6, per_slot=4)
    p.fill([0, 1, 2, 3, 4], lens, rng)
    n = [tokens, 1, max(1, tokens - 1), tokens, 0]
    q = 0.3 * rng.standard_normal((5, tokens, heads * group, d))
    check_attention(p, 0, q, [0, 1, 2, 3, 4], [e - m for e, m in zip(lens, n)], lens, window=window)


@pytest.mark.parametrize("d,heads,group,page,lens", [
    (512, 4, 8, 64, [4000]),             # one row over every SM
    (256, 16, 2, 16, [1, 700, 33, 2000, 128]),
    (512, 2, 8, 128, [5, 1500, 5, 64, 900, 2]),
    (256, 4, 4, 32, [100] * 70),         # more items than warps' runs are long
])
def test_decode_work_split(d, heads, group, page, lens):
    """Items inside one warp's run, across warps of a CTA and across CTAs."""
    rng = np.random.default_rng(len(lens))
    need = sum(-(-x // page) for x in lens)
    p = Pair("e4m3", heads=heads, page=page, d=d, pages=need + 2, slots=len(lens),
             per_slot=-(-max(lens) // page))
    p.fill(list(range(len(lens))), lens, rng)
    q = 0.2 * rng.standard_normal((len(lens), 1, heads * group, d))
    got = check_attention(p, 0, q, range(len(lens)), [x - 1 for x in lens], lens)
    for tight in (max(lens), max(lens) + 1000):  # the bound changes the launch, not the result
        again = check_attention(p, 0, q, range(len(lens)), [x - 1 for x in lens], lens,
                                max_seqlen_k=tight)
        assert np.array_equal(got, again) or tight != max(lens)


def test_empty_rows_masked_pages_and_stale_slots():
    rng = np.random.default_rng(11)
    p = Pair("e4m3", heads=2, d=256, page=16, pages=40, slots=8, per_slot=8)
    lens = [100, 37, 50, 20, 1]
    p.fill([0, 1, 2, 3, 4], lens, rng)
    # everything no row may see is poisoned: NaN codes behind the ends, NaN scales of free pages
    codes = p.dev.k.view(torch.uint8), p.dev.v.view(torch.uint8)
    used = p.ref.refcounts > 0
    for page in range(40):
        if not used[page]:
            for c in codes:
                c[:, page] = 0x7F
            p.dev.k_scale[:, page] = float("nan")
            p.dev.v_scale[:, page] = float("inf")
    for slot, n in enumerate(lens):
        last = int(p.ref.tables[slot, (n - 1) // 16])
        if n % 16:
            for c in codes:
                c[:, last, :, n % 16:] = 0x7F
    # a page is missing in row 1, all of row 2's are, row 3 lists a bad id
    p.ref.tables[1, 1] = -1
    p.ref.tables[2, :] = -1
    p.ref.tables[3, 0] = 40
    p.dev.tables.copy_(i32(p.ref.tables))
    q = 0.3 * rng.standard_normal((9, 2, 4, 256))
    check_attention(p, 0, q, [0, 1, 2, 3, 4, 5, 9, -2, 0], [98, 35, 48, 18, 0, 0, 3, 3, 126],
                    [100, 37, 50, 20, 1, 0, 5, 5, 129])
    # rows past max_seqlen_k count as empty
    got = check_attention(p, 0, q[:2], [0, 1], [98, 35], [100, 37], max_seqlen_k=99)
    assert not got[0].any() and got[1].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_scales_of_any_size(fmt):
    """Blocks whose scales differ by many powers of two, and queries of very
    different magnitude."""
    rng = np.random.default_rng(12)
    p = Pair(fmt, heads=1, d=512, page=16, pages=12, slots=2, per_slot=10)
    p.extend([0], [150])
    p.ref.k_scale[:] = 2.0 ** rng.integers(-9, -4, p.ref.k_scale.shape)
    p.ref.v_scale[:] = 2.0 ** rng.integers(-90, 90, p.ref.v_scale.shape)
    p.ref.v_scale[0, 3, 0] = 1.37
    p.dev.k_scale.copy_(torch.tensor(p.ref.k_scale))
    p.dev.v_scale.copy_(torch.tensor(p.ref.v_scale))
    p.ref.k_scale[:], p.ref.v_scale[:] = f64(p.dev.k_scale), f64(p.dev.v_scale)
    q = rng.standard_normal((1, 1, 4, 512)) * np.array([1e-30, 1e-4, 0.05, 0.4])[:, None]
    q[0, 0, 1, 9] = 1e-20  # far below the column's largest
    check_attention(p, 0, q, [0], [149], [150])


def test_attention_is_repeatable_and_reads_strided_queries():
    rng = np.random.default_rng(13)
    p = Pair("int8", heads=4, d=256, page=32, pages=80, slots=8, per_slot=20)
    lens = [600, 31, 480]
    p.fill([0, 1, 2], lens, rng)
    big, _ = bf16(0.3 * rng.standard_normal((3, 3, 5, 8, 256)))
    q = big[:, :, 2]
    args = [0, 1, 2], [e - 3 for e in lens], lens
    a = check_attention(p, 0, (q, f64(q)), *args)
    b = check_attention(p, 0, (q.contiguous(), f64(q)), *args)
    assert np.array_equal(a, b)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)  # heads before tokens
    assert np.array_equal(a, check_attention(p, 0, (t, f64(q)), *args))
    with pytest.raises(ValueError, match="stride"):
        p.dev.attention(0, q[:1].expand(3, -1, -1, -1), *map(i32, args))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads,group,tokens,page,window,lens", [
    (512, 1, 8, 4, 64, 0, [900, 128, 129, 4]),          # 32 columns, all of them used
    (512, 2, 8, 5, 16, 300, [700, 40, 301, 300, 5]),    # 40 of 64, pages inside a tile
    (512, 1, 3, 11, 128, 0, [1500, 11]),                # 33 of 64
    (512, 1, 8, 32, 32, 0, [400, 33, 1000]),            # four groups of 64 columns
    (512, 1, 8, 17, 32, 100, [17, 600]),                # 64, 64 and 8
    (256, 2, 2, 12, 32, 1024, [2500, 12, 130, 1100]),   # 24 of 32
    (256, 3, 16, 2, 64, 0, [2, 1000]),                  # 32, few keys and many
    (256, 16, 2, 5, 16, 64, [70] * 40),                 # many items per CTA
])
def test_wide_shapes(fmt, d, heads, group, tokens, page, window, lens):
    """More than 8 columns: every launch shape, groups of columns, windows, padding."""
    rng = np.random.default_rng(tokens + len(lens))
    p = Pair(fmt, heads=heads, d=d, page=page, pages=2 + sum(-(-x // page) for x in lens),
             slots=len(lens), per_slot=-(-max(lens) // page))
    rows = list(range(len(lens)))
    p.fill(rows, lens, rng)
    n = [tokens - (b % 3 if b else 0) for b in rows]
    q = 0.3 * rng.standard_normal((len(lens), tokens, heads * group, d))
    check_attention(p, 0, q, rows, [e - m for e, m in zip(lens, n)], lens, window=window)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,group,tokens", [(512, 8, 2), (512, 8, 6), (256, 4, 8)])
def test_wide_maxima_that_rise_and_scales_of_any_size(fmt, d, group, tokens):
    """Scores that grow along the keys, so that every tile renews the references, with
    V scales that differ by many powers of two and queries of very different size."""
    rng = np.random.default_rng(d + tokens)
    n, page = 1000, 16
    p = Pair(fmt, heads=1, d=d, page=page, pages=66, slots=1, per_slot=64)
    p.extend([0], [n])
    u = rng.standard_normal(d)
    u /= np.linalg.norm(u)
    k = rng.standard_normal((1, n, 1, d)) + (np.arange(n) / 8.0)[None, :, None, None] * u
    v = rng.standard_normal((1, n, 1, d))
    p.append(0, k, v, [0], [0], [n])
    p.ref.v_scale[:] = 2.0 ** rng.integers(-40, 40, p.ref.v_scale.shape)
    p.ref.v_scale[0, 5, 0] = 1.37
    p.dev.v_scale.copy_(torch.tensor(p.ref.v_scale))
    p.ref.v_scale[:] = f64(p.dev.v_scale)
    size = np.array([1e-30, 1e-3, 0.2, 1.0])[np.arange(group) % 4][:, None]
    q = size * (u + 0.02 * rng.standard_normal((1, tokens, group, d)))
    check_attention(p, 0, q, [0], [n - tokens], [n])


@pytest.mark.parametrize("seed", range(8))
def test_random_batches_over_the_tile_list(seed):
    """Rows of any length (none among them) in any order, bad slots, missing pages, padded
    tokens, windows: in slots long enough that items share CTAs and span them."""
    rng = np.random.default_rng(500 + seed)
    d, heads, group = ((512, 1, 8), (256, 2, 2), (512, 2, 4), (256, 3, 1))[seed % 4]
    tokens = (1, 1, 2, 7)[(seed + seed // 4) % 4]
    page = int(rng.choice([16, 32, 64, 128]))
    window = int(rng.choice([0, 100]))
    n = int(rng.integers(3, 40))
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(700), n))]
    p = Pair("e4m3" if seed % 2 else "int8", heads=heads, page=page, d=d, slots=n,
             pages=2 + sum(-(-x // page) for x in lens), per_slot=2048 // page)
    p.fill(list(range(n)), lens, rng)
    for slot in rng.choice(n, 2, replace=False):  # holes
        p.ref.tables[slot, rng.integers(0, -(-lens[slot] // page))] = -1
    p.dev.tables.copy_(i32(p.ref.tables))
    rows = [int(x) for x in rng.permutation(n)]
    ends = [lens[r] for r in rows]
    new = [min(int(rng.integers(0, tokens + 1)), e) for e in ends]
    rows[1] = n + 3
    q = 0.3 * rng.standard_normal((n, tokens, heads * group, d))
    check_attention(p, 0, q, rows, [e - m for e, m in zip(ends, new)], ends, window=window)


def test_empty_rows_and_holes_in_long_slots():
    rng = np.random.default_rng(23)
    p = Pair("int8", heads=2, d=256, page=16, pages=80, slots=8, per_slot=64)
    lens = [100, 37, 900, 20, 1]
    p.fill([0, 1, 2, 3, 4], lens, rng)
    p.ref.tables[1, :] = -1
    p.ref.tables[2, 3:20] = -1
    p.dev.tables.copy_(i32(p.ref.tables))
    q = 0.3 * rng.standard_normal((9, 2, 4, 256))
    args = ([0, 1, 2, 3, 4, 5, 9, -2, 0], [98, 35, 898, 18, 0, 0, 3, 3, 1022],
            [100, 37, 900, 20, 1, 0, 5, 5, 1025])
    check_attention(p, 0, q, *args)
    check_attention(p, 0, q, *args, window=64)
    got = check_attention(p, 0, q, *args, max_seqlen_k=899)
    assert not got[2].any() and got[0].any()


def test_calls_of_one_cache_on_two_streams():
    """Reads of one cache need no order among themselves."""
    rng = np.random.default_rng(24)
    p = Pair("e4m3", heads=2, d=512, page=32, pages=140, slots=4, per_slot=80)
    lens = [2000, 31, 1500, 400]
    p.fill([0, 1, 2, 3], lens, rng)
    slots, ends = i32([0, 1, 2, 3]), i32(lens)
    ops = []
    for tokens in (1, 4, 9):  # decode, wide of 32 and of 64 columns (group 4 and 8)
        q, _ = bf16(0.3 * rng.standard_normal((4, tokens, 16, 512)))
        ops.append((q, i32([x - tokens for x in lens])))
    want = [p.dev.attention(0, q, slots, s, ends) for q, s in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for rep in range(4):
        for i, (q, s) in enumerate(ops):
            with torch.cuda.stream(streams[(i + rep) % 2]):
                got.append((i, p.dev.attention(0, q, slots, s, ends)))
    torch.cuda.synchronize()
    for i, (out, lse) in got:
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_wide_empty_rows_masked_pages_and_stale_slots():
    rng = np.random.default_rng(21)
    p = Pair("e4m3", heads=1, d=512, page=16, pages=40, slots=8, per_slot=20)
    lens = [250, 37, 50, 20, 6]
    p.fill([0, 1, 2, 3, 4], lens, rng)
    codes = p.dev.k.view(torch.uint8), p.dev.v.view(torch.uint8)
    for page in np.flatnonzero(p.ref.refcounts == 0):
        for c in codes:
            c[:, page] = 0x7F
        p.dev.k_scale[:, page] = float("nan")
        p.dev.v_scale[:, page] = float("inf")
    for slot, n in enumerate(lens):
        if n % 16:
            for c in codes:
                c[:, int(p.ref.tables[slot, (n - 1) // 16]), :, n % 16:] = 0x7F
    p.ref.tables[0, 3] = p.ref.tables[1, 1] = -1   # holes, a row of them, a bad id
    p.ref.tables[0, 8:16] = -1                     # a whole tile
    p.ref.tables[2, :] = -1
    p.ref.tables[3, 0] = 40
    p.dev.tables.copy_(i32(p.ref.tables))
    q = 0.3 * rng.standard_normal((9, 5, 8, 512))
    check_attention(p, 0, q, [0, 1, 2, 3, 4, 5, 9, -2, 0], [245, 35, 45, 18, 1, 0, 3, 3, 318],
                    [250, 37, 50, 20, 6, 0, 5, 5, 321])
    got = check_attention(p, 0, q[:2], [0, 1], [246, 35], [250, 37], max_seqlen_k=249)
    assert not got[0].any() and got[1].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads,group,window", [(512, 1, 8, 0), (256, 2, 2, 0), (256, 2, 2, 50)])
def test_chunks_of_prompts(fmt, d, heads, group, window):
    """More queries than the direct kernel takes: ragged, padded and empty rows."""
    rng = np.random.default_rng(14)
    tokens = DIRECT_COLUMNS[d] // group + 3
    lens = [tokens, tokens + 90, 200, 5]
    p = Pair(fmt, heads=heads, d=d, page=64, pages=30, slots=5, per_slot=6)
    p.fill([0, 1, 2, 3], lens, rng)
    n = [tokens, tokens - 2, 1, 5]
    q = 0.2 * rng.standard_normal((5, tokens, heads * group, d))
    poison = torch.full((1 << 25,), float("nan"), device="cuda")  # what the next buffers hold
    del poison
    check_attention(p, 0, q, [0, 1, 2, 3, 4], [*[e - m for e, m in zip(lens, n)], 0], [*lens, 0],
                    window=window, max_seqlen_k=300)


def test_positions_past_31_bits_of_bytes():
    """A pool of more than 2^32 bytes: the pages at its end."""
    page_bytes = 16 * 128 * 512
    pages = (1 << 32) // page_bytes + 8
    pool = [torch.zeros(1, pages, 16, 128, 512, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.ones(1, pages, 16, device="cuda") for _ in range(2)]
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-3:] = 0
    cache = PagedKVCache8.from_tensors(*pool, *scales, torch.full((2, 4), -1, dtype=torch.int32,
                                                                  device="cuda"),
                                       torch.zeros(2, dtype=torch.int32, device="cuda"), refs)
    rng = np.random.default_rng(15)
    k, hk = bf16(rng.standard_normal((1, 130, 16, 512)))
    starts, ends = cache.extend(i32([1]), 130)
    assert cache.tables[1].tolist() == [pages - 3, pages - 2, -1, -1]
    cache.append(0, k, k.clone(), i32([1]), starts, ends)
    back, _ = cache.read(0, i32([1]), starts, ends, 130)
    assert np.abs(f64(back) - hk).max() <= 2.0 ** -4 * 4  # half a step of 2^-5 at magnitude < 4.1
    cache.copy_pages(i32([pages - 3]), i32([0]))
    assert torch.equal(cache.k[0, 0], cache.k[0, pages - 3])
    small = PagedKVCache8.from_tensors(
        cache.k[:, -3:].contiguous(), cache.v[:, -3:].contiguous(),
        cache.k_scale[:, -3:].contiguous(), cache.v_scale[:, -3:].contiguous(),
        i32([[0, 1]]), i32([130]), i32([1, 1, 0]))
    q, _ = bf16(0.2 * rng.standard_normal((1, 1, 32, 512)))
    a = cache.attention(0, q, i32([1]), i32([129]), i32([130]), max_seqlen_k=256)
    b = small.attention(0, q, i32([0]), i32([129]), i32([130]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    cache.check()


# ------------------------------------------------------------------------------------
# pages
# ------------------------------------------------------------------------------------
def test_extend_serves_rows_in_order():
    p = Pair("int8", pages=10, slots=6, per_slot=4, page=16)
    p.extend([3, 0], [17, 16])
    p.extend([3, 0, 1], [15, 1, 0])
    p.extend([1, 1, 7, -1, 2], [5, 5, 5, 5, -2])    # twice, out of range, a negative count
    p.same()
    p.ref.status = 0
    p.dev.status.zero_()
    p.extend([0, 2, 4, 1], [100, 65, 1, 3])          # tables of four pages are full
    assert p.ref.status == _lib.G4_PAGES_ROW_FULL
    p.same()
    p.extend([4, 2, 5, 3], [15, 64, 1, 0])           # five pages are left, then none
    p.extend([5, 4, 0], [16, 1, 1])
    assert p.ref.status == _lib.G4_PAGES_ROW_FULL | _lib.G4_PAGES_EXHAUSTED
    p.same()


def test_fork_shares_whole_pages_and_copies_the_last():
    rng = np.random.default_rng(20)
    p = Pair("e4m3", layers=2, pages=20, slots=8, per_slot=5, page=32)
    p.fill([0, 1, 2], [70, 64, 0], rng)
    p.ref.fork([0, 0, 1, 2], [4, 5, 6, 7])
    p.dev.fork(i32([0, 0, 1, 2]), i32([4, 5, 6, 7]))
    p.same()
    # each continues on its own: the parent's tokens stay
    before = f64(p.dev.read(0, i32([0]), i32([0]), i32([70]), 70)[0])
    p.fill([4, 5, 6], [3, 40, 1], rng, magnitude=50.0)
    p.same()
    assert np.array_equal(before, f64(p.dev.read(0, i32([0]), i32([0]), i32([70]), 70)[0]))
    # occupied, doubled, bad children; a child of itself; a child that is a parent
    p.ref.fork([0, 0, 0, 9, 1, 7], [4, 3, 3, 3, -1, 7])
    p.dev.fork(i32([0, 0, 0, 9, 1, 7]), i32([4, 3, 3, 3, -1, 7]))
    assert p.ref.status == _lib.G4_PAGES_BAD_INDEX
    p.same()
    p.ref.free([4, 0, 4, 12])
    p.dev.free(i32([4, 0, 4, 12]))
    p.same()


def test_fork_of_an_exhausted_pool_leaves_the_child_empty():
    rng = np.random.default_rng(21)
    p = Pair("int8", pages=6, slots=6, per_slot=4, page=16)
    p.fill([0, 1], [30, 32], rng)
    p.ref.fork([0, 0, 1, 0], [2, 3, 4, 5])   # two free pages for three copies
    p.dev.fork(i32([0, 0, 1, 0]), i32([2, 3, 4, 5]))
    assert p.ref.status == _lib.G4_PAGES_EXHAUSTED and p.ref.lengths[5] == 0
    p.same()


@pytest.mark.parametrize("window", [1, 16, 17, 40, 500])
def test_trim_frees_what_the_window_left(window):
    rng = np.random.default_rng(22)
    p = Pair("e4m3", heads=1, pages=40, slots=5, per_slot=10, page=16)
    lens = [100, 16, 15, 32, 0]
    p.fill([0, 1, 2, 3], lens[:4], rng)
    p.ref.free([0, 1, 2, 3, 4], window)
    p.dev.trim(i32([0, 1, 2, 3, 4]), window)
    p.same()
    starts, ends = p.fill([0, 1, 2, 3], [1, 1, 1, 1], rng)   # decoding goes on as if nothing left
    q = 0.3 * rng.standard_normal((4, 1, 2, 256))
    check_attention(p, 0, q, [0, 1, 2, 3], starts, ends, window=window)
    p.ref.free([0, 1, 2, 3])
    p.dev.free(i32([0, 1, 2, 3]))
    p.same()
    assert not p.ref.refcounts.any()


@pytest.mark.parametrize("seed", range(4))
def test_random_page_traffic(seed):
    """Many calls in a row, indices out of range among them; everything equal."""
    rng = np.random.default_rng(seed)
    pages = int(rng.integers(30, 90))
    p = Pair("int8" if seed % 2 else "e4m3", layers=2, heads=1, pages=pages, slots=12, per_slot=9,
             page=int(rng.choice([16, 32])), seed=seed)
    for _ in range(25):
        act = rng.integers(0, 6)
        n = int(rng.integers(1, 6))
        slots = rng.choice(14, n, replace=False) - 1
        if act <= 1:
            p.fill([int(s) for s in slots], [int(x) for x in rng.integers(0, 50, n)], rng, layer=1)
        elif act == 2:
            kids = rng.choice(12, n, replace=False)
            p.ref.fork(list(slots), list(kids))
            p.dev.fork(i32(slots), i32(kids))
        elif act == 3:
            p.ref.free(list(slots))
            p.dev.free(i32(slots))
        elif act == 4:
            p.ref.compact()
            p.dev.compact()
        else:
            src, dst = rng.integers(-1, pages + 1, 6), rng.integers(0, pages, 6)
            if p.ref.refcounts[dst].any():  # only free pages are written over
                continue
            p.ref.copy_pages(list(src), list(dst))
            p.dev.copy_pages(i32(src), i32(dst))
    p.same()
    p.ref.compact()
    p.dev.compact()
    p.same()
    live = int((p.ref.refcounts > 0).sum())
    assert not p.ref.refcounts[live:].any()


def test_a_large_pool_and_a_full_batch():
    """1024 rows and more pages than one pass of the block takes."""
    pages, rows = 5000, 1024
    cache = PagedKVCache8(1, pages, 1, 256, max_slots=rows, pages_per_slot=5, page_size=16)
    mine = ref.PagedCache("e4m3", 1, 1, 1, 16, 1, rows, 5)
    mine.refcounts = np.zeros(pages, dtype=np.int64)
    rng = np.random.default_rng(30)
    for counts in (rng.integers(0, 40, rows), rng.integers(0, 40, rows), rng.integers(0, 60, rows)):
        order = rng.permutation(rows)
        starts, ends = mine.extend(list(order), list(counts))
        ds, de = cache.extend(i32(order), i32(counts))
        assert ds.tolist() == list(starts) and de.tolist() == list(ends)
        gone = rng.choice(rows, 300, replace=False)
        mine.free(list(gone))
        cache.free(i32(gone))
        assert np.array_equal(cache.tables.cpu().numpy(), mine.tables)
        assert np.array_equal(cache.refcounts.cpu().numpy(), mine.refcounts)
    live = int((mine.refcounts > 0).sum())
    cache.compact()
    assert int((cache.refcounts[:live] > 0).sum()) == live and not cache.refcounts[live:].any()
    q = torch.zeros(rows, 1, 2, 256, dtype=torch.bfloat16, device="cuda")
    ends = cache.lengths.clone()
    out, lse = cache.attention(0, q, None, (ends - 1).clamp(min=0), ends)
    # zero queries: every visible key weighs the same, LSE is the log of their number
    want = torch.log(ends.double())[:, None, None].expand(-1, 2, 1)
    assert torch.allclose(lse.double(), want, atol=2e-6)
    assert not out.any()  # the values are zeros


# ------------------------------------------------------------------------------------
# as a serving loop uses them
# ------------------------------------------------------------------------------------
def _loop_step(cache, q, k, v, slots, counts, window):
    starts, ends = cache.extend(slots, counts)
    outs = []
    for layer in range(cache.num_layers):
        cache.append(layer, k[layer], v[layer], slots, starts, ends)
        outs += cache.attention(layer, q[layer], slots, starts, ends, window=window)
    return outs


@pytest.mark.parametrize("window", [0, 48])
def test_serving_loop_prompt_decode_fork_trim_compact(window):
    rng = np.random.default_rng(40)
    heads, d, group = 2, 256, 2
    p = Pair("e4m3", layers=2, heads=heads, d=d, pages=60, slots=8, per_slot=12, page=16)

    def step(slots, counts):
        n = max(counts)
        starts, ends = p.extend(slots, counts)
        for layer in range(2):
            k, v = rng.standard_normal((2, len(slots), n, heads, d))
            p.append(layer, k, v, slots, starts, ends)
            q = 0.3 * rng.standard_normal((len(slots), n, heads * group, d))
            check_attention(p, layer, q, slots, starts, ends, window=window)

    step([0, 1, 2], [70, 33, 5])
    for _ in range(3):
        step([2, 0, 1], [1, 1, 1])
    p.ref.fork([0, 0, 2], [3, 4, 5])
    p.dev.fork(i32([0, 0, 2]), i32([3, 4, 5]))
    step([0, 3, 4, 5, 1], [1, 1, 2, 1, 0])
    p.ref.free([0, 1])
    p.dev.free(i32([0, 1]))
    if window:
        p.ref.free([2, 3, 4, 5], window)
        p.dev.trim(i32([2, 3, 4, 5]), window)
    p.ref.compact()
    p.dev.compact()
    p.same()
    step([3, 4, 5, 0], [1, 1, 1, 20])
    p.same()
    p.dev.check()


def test_captured_step_replays_as_the_eager_calls():
    """extend, append and attention in one CUDA graph: lengths and pages advance on
    the device at every replay."""
    def make():
        return PagedKVCache8(2, 40, 2, 256, max_slots=4, pages_per_slot=8, page_size=16,
                             dtype=torch.int8)

    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(2, 3, 1, h, 256, generator=g, device="cuda").to(torch.bfloat16)
               for h in (4, 2, 2))
    slots, counts = i32([2, 0, 1]), i32([1, 1, 1])
    eager, graphed = make(), make()
    for c in (eager, graphed):
        c.extend(i32([0, 1, 2]), i32([14, 40, 3]))
    want = []
    for i in range(5):
        want.append([x.clone() for x in _loop_step(eager, q + i, k - i, v, slots, counts, 0)])
    sq, sk = q.clone(), k.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a warm-up on another cache
        _loop_step(make(), sq, sk, v, slots, counts, 0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _loop_step(graphed, sq, sk, v, slots, counts, 0)
    for i in range(5):
        sq.copy_(q + i)
        sk.copy_(k - i)
        graph.replay()
        for a, b in zip(outs, want[i]):
            assert torch.equal(a, b)
    assert torch.equal(eager.k, graphed.k) and torch.equal(eager.tables, graphed.tables)
    assert graphed.lengths.tolist() == [19, 45, 8, 0]


def test_two_caches_on_two_streams():
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (0.2 * torch.randn(3, 2, 8, 512, generator=g, device="cuda")).to(torch.bfloat16)
    k = torch.randn(3, 400, 1, 512, generator=g, device="cuda").to(torch.bfloat16)
    caches = [PagedKVCache8(1, 60, 1, 512, max_slots=3, pages_per_slot=20, page_size=32)
              for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for c, s, o in zip(caches, streams, outs):
            with torch.cuda.stream(s):
                slots = i32([0, 1, 2])
                starts, ends = c.extend(slots, i32([100, 57, 2]))
                c.append(0, k[:, :100].contiguous(), k[:, 100:200].contiguous(), slots, starts, ends)
                o.append(c.attention(0, q, slots, ends - 2, ends))
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
