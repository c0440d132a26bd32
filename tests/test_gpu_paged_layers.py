"""Decode layers over the paged 8-bit cache at the Gemma-4 31B geometry: prompts in
chunks, decode, drafted tokens, against a composition in float64 and, captured into a
graph, against the eager calls."""

import numpy as np
import pytest
import torch

from oracle.paged_cache import PagedCache

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("needs a CUDA device", allow_module_level=True)

from gemma4_fa4_kernels_b200 import PagedKVCache8  # noqa: E402
from gemma4_fa4_kernels_b200 import decode_ops as d  # noqa: E402
from gemma4_fa4_kernels_b200.prep import prep_fwd  # noqa: E402

H = d.HIDDEN_SIZE


def _bf(x):
    return torch.as_tensor(x, dtype=torch.float32).bfloat16().cuda()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Layer:
    """One layer's weights and its calls."""

    def __init__(self, kind, seed):
        g = torch.Generator().manual_seed(seed)
        self.kind = kind
        self.hq, self.hkv, self.d = d.GLOBAL_GEOMETRY if kind == "global" else d.LOCAL_GEOMETRY
        self.window = 0 if kind == "global" else d.LOCAL_WINDOW
        mat = lambda o, i: _bf(torch.randn(o, i, generator=g) / i ** 0.5)  # noqa: E731
        self.wq, self.wk = mat(self.hq * self.d, H), mat(self.hkv * self.d, H)
        self.wv = mat(self.hkv * self.d, H) if kind == "local" else None
        self.wo = mat(H, self.hq * self.d)
        # query norms of d ** -0.25 keep the scores of d-dim unit vectors moderate
        self.qn = _bf(self.d ** -0.25 * (1 + 0.1 * torch.randn(self.d, generator=g)))
        self.kn = _bf(self.d ** -0.25 * (1 + 0.1 * torch.randn(self.d, generator=g)))

    def rope(self, starts, tokens):
        """Rotary tables (rows, tokens, d) of positions starts + 0 .. tokens - 1."""
        pos = starts[:, None] + torch.arange(tokens, device="cuda")
        freq = 1e4 ** -(torch.arange(self.d // 2, device="cuda") / (self.d // 2))
        ang = pos[..., None].float() * freq
        ang = torch.cat((ang, ang), -1)
        return ang.cos().bfloat16(), ang.sin().bfloat16()

    def __call__(self, cache, h, slots, starts, ends, **kw):
        cos, sin = self.rope(starts, h.shape[1])
        if self.kind == "global":
            return d.global_paged_cache_decode_fwd(cache, 0, h, cos, sin, slots, starts, ends,
                                                   self.wq, self.wk, self.wo, self.qn, self.kn,
                                                   **kw)
        return d.local_paged_cache_decode_fwd(cache, 0, h, cos, sin, slots, starts, ends, self.wq,
                                              self.wk, self.wv, self.wo, self.qn, self.kn, **kw)

    def operands(self, h, starts):
        """(q, k, v) as the layer forms them, BF16."""
        cos, sin = self.rope(starts, h.shape[1])
        lin = torch.nn.functional.linear
        head = lambda w, n: lin(h, w).view(*h.shape[:2], n, self.d)  # noqa: E731
        q, _ = prep_fwd(head(self.wq, self.hq), self.qn, cos, sin, self.d)
        k, v = prep_fwd(head(self.wk, self.hkv), self.kn, cos, sin, self.d, want_plain=True)
        if self.wv is not None:
            _, v = prep_fwd(head(self.wv, self.hkv), None, None, None, 0, want_rot=False,
                            want_plain=True)
        return q, k, v


@pytest.mark.parametrize("kind,fmt", [("global", "e4m3"), ("local", "int8")])
@torch.no_grad()
def test_layer_prompt_then_drafts_then_decode(kind, fmt):
    """Three calls of each kind of step; every one against the oracle fed with the same
    q, k, v.  The attention's result is within 2^-8 of each row's size (its rounding to
    BF16, 2^-9 in the mean square, and P's 2^-8 in a chunk, which averages out over the
    keys), the projection's rounding adds 2^-9: 2^-7 of the row's L2 norm holds both."""
    g = torch.Generator().manual_seed(3)
    dtype = torch.float8_e4m3fn if fmt == "e4m3" else torch.int8
    layer = Layer(kind, 5)
    pages, slots, per_slot = 12, 4, 5
    cache = PagedKVCache8(1, pages, layer.hkv, layer.d, max_slots=slots, pages_per_slot=per_slot,
                          page_size=32, dtype=dtype)
    ref = PagedCache(fmt, 1, pages, layer.hkv, 32, layer.d, slots, per_slot)
    for counts in ([70, 45, 0], [3, 1, 2], [1, 1, 1]):
        rows, tokens = [2, 0, 3], max(counts)
        s, e = ref.extend(rows, counts)
        ds, de = cache.extend(_i32(rows), _i32(counts))
        assert ds.tolist() == list(s) and de.tolist() == list(e)
        h = torch.randn(3, tokens, H, generator=g).bfloat16().cuda()
        out, lse = layer(cache, h, _i32(rows), ds, de)
        q, k, v = (x.double().cpu().numpy() for x in layer.operands(h, ds))
        ref.append(0, k, v, rows, list(s), list(e))
        for name in ("k", "v"):
            assert np.array_equal(getattr(cache, name).float().cpu().double().numpy(),
                                  getattr(ref, name)), name
        want, want_lse, *_ = ref.attention(0, q, rows, list(s), list(e), layer.window, 1 << 40)
        want = torch.from_numpy(want).cuda().flatten(2) @ layer.wo.double().t()
        assert out.shape == (3, tokens, H) and out.dtype == torch.bfloat16
        assert lse.shape == (3, layer.hq, tokens)
        for b, n in enumerate(counts):
            assert not out[b, n:].any() and torch.isneginf(lse[b, :, n:]).all()
            err = (out[b, :n].double() - want[b, :n]).norm(dim=-1)
            assert (err <= 2.0 ** -7 * want[b, :n].norm(dim=-1)).all(), (err / want[b, :n].norm(dim=-1))
            # fp32 scores of d products of moderate size (see the attention's own bounds)
            assert np.abs(lse[b, :, :n].double().cpu().numpy() - want_lse[b, :, :n]).max(initial=0) < 1e-3
    cache.check()


@pytest.mark.parametrize("kind", ["global", "local"])
@torch.no_grad()
def test_captured_layer_steps_are_the_eager_ones(kind):
    g = torch.Generator().manual_seed(4)
    layer = Layer(kind, 6)
    make = lambda: PagedKVCache8(1, 8, layer.hkv, layer.d, max_slots=2,  # noqa: E731
                                 pages_per_slot=4, page_size=16)
    eager, graphed = make(), make()
    slots = _i32([0, 1])
    prompt = torch.randn(2, 14, H, generator=g).bfloat16().cuda()
    for c in (eager, graphed):
        layer(c, prompt, slots, *c.extend(slots, _i32([14, 9])))
    steps = torch.randn(6, 2, 1, H, generator=g).bfloat16().cuda()
    h, counts = steps[0].clone(), _i32([1, 1])
    spare = make()  # warms the libraries up; capture itself runs nothing
    layer(spare, h, slots, *spare.extend(slots, counts))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = layer(graphed, h, slots, *graphed.extend(slots, counts))
    for step in steps:
        h.copy_(step)
        graph.replay()
        want, want_lse = layer(eager, step, slots, *eager.extend(slots, counts))
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert graphed.lengths.tolist() == [20, 15]
    graphed.check()
