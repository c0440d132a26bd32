"""Decode layers over the paged 8-bit cache: what they refuse, without a GPU."""

import pytest
import torch

from gemma4_fa4_kernels_b200 import PagedKVCache8, UnsupportedB200Path
from gemma4_fa4_kernels_b200 import decode_ops as d


def _args(kind, rows=2, tokens=3):
    hq, hkv, dim = d.GLOBAL_GEOMETRY if kind == "global" else d.LOCAL_GEOMETRY
    bf = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cpu")  # noqa: E731
    cache = PagedKVCache8(1, 4, hkv, dim, max_slots=4, pages_per_slot=2, page_size=16,
                          device="cpu")
    rows_i = torch.empty(rows, dtype=torch.int32, device="cpu")
    out = dict(cache=cache, layer=0, hidden_states=bf(rows, tokens, d.HIDDEN_SIZE),
               cos=bf(rows, tokens, dim), sin=bf(rows, tokens, dim), slots=rows_i, starts=rows_i,
               ends=rows_i, q_proj_weight=bf(hq * dim, d.HIDDEN_SIZE),
               k_proj_weight=bf(hkv * dim, d.HIDDEN_SIZE),
               o_proj_weight=bf(d.HIDDEN_SIZE, hq * dim), q_norm_weight=bf(dim),
               k_norm_weight=bf(dim))
    if kind == "local":
        out["v_proj_weight"] = bf(hkv * dim, d.HIDDEN_SIZE)
    return out


OPS = {"global": d.global_paged_cache_decode_fwd, "local": d.local_paged_cache_decode_fwd}


@pytest.mark.parametrize("kind", ["global", "local"])
def test_layers_require_no_grad_mode(kind):
    with torch.enable_grad(), pytest.raises(UnsupportedB200Path, match="no-grad"):
        OPS[kind](**_args(kind))
    args = _args(kind)
    args["cos"].requires_grad_(True)
    with torch.no_grad(), pytest.raises(UnsupportedB200Path, match="requires_grad"):
        OPS[kind](**args)


@pytest.mark.parametrize("kind", ["global", "local"])
@pytest.mark.parametrize("name,change,exc,needle", [
    ("cache", lambda t: None, ValueError, "PagedKVCache8"),
    ("hidden_states", lambda t: t[0], UnsupportedB200Path, "hidden states"),
    ("hidden_states", lambda t: t[..., :-8], UnsupportedB200Path, "hidden states"),
    ("hidden_states", lambda t: t.float(), ValueError, "BF16"),
    ("hidden_states", lambda t: torch.empty_like(t, device="meta"), ValueError, "device"),
    ("cos", lambda t: t[:1], ValueError, "rotary"),
    ("sin", lambda t: t[..., :128], ValueError, "rotary"),
    ("q_proj_weight", lambda t: t[:-1], ValueError, "locked layer"),
    ("k_norm_weight", lambda t: t.float(), ValueError, "BF16"),
])
@torch.no_grad()
def test_layers_refuse(kind, name, change, exc, needle):
    args = _args(kind)
    args[name] = change(args[name])
    with pytest.raises(exc, match=needle):
        OPS[kind](**args)


@torch.no_grad()
def test_layers_refuse_a_cache_of_the_other_geometry():
    args = _args("global")
    args["cache"] = _args("local")["cache"]
    with pytest.raises(UnsupportedB200Path, match="4 KV heads of 512"):
        OPS["global"](**args)
