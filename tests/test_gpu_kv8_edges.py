"""The 8-bit paged cache where it can go wrong: weights far below the maximum, steps that went
stale, ids that the GPU has to refuse, views at odd offsets (tests/_kv8_ref.py has the plain
64-bit forms)."""

from __future__ import annotations

import pytest
import torch

import _kv8_ref as ref
from test_gpu_kv8 import DEV, _batch, _no_device_error  # noqa: F401  (the fixture reads the error word)

pytestmark = pytest.mark.gpu


def _peaked(lengths, hq, hkv, d, dtype, every, drop, v_bytes, seed=0):
    """Scores of `drop` at every `every`-th key, whose V row is zero, and 0 at the others, whose
    V rows are 200 to 448 times one of the scales `v_bytes`: with scale 1 a weight is e^-drop of
    the maximum, and all of the output comes from such weights."""
    query, pools, tables, ctx, ql = _batch(lengths, hq, hkv, d, 16, dtype, seed=seed)
    query[..., 0] = 1.0
    g = torch.Generator(device=DEV).manual_seed(seed)
    k, v = (p.view(torch.uint8).view(-1, hkv, d) for p in pools[:2])
    for i, (c, _) in enumerate(lengths):
        pos = torch.arange(c, device=DEV)
        slots = tables[i].long()[pos // 16] * 16 + pos % 16
        peak = pos % every == 0
        row = torch.zeros(c, hkv, d, device=DEV)
        row[peak, :, 0] = drop
        k[slots] = row.to(ref.E4M3).view(torch.uint8)
        vals = (torch.rand(c, hkv, d, generator=g, device=DEV) * 248 + 200) * (~peak)[:, None, None]
        v[slots] = vals.to(ref.E4M3).view(torch.uint8)
        pools[2][slots // 16, :, slots % 16] = 127
        pick = torch.randint(0, len(v_bytes), (c, hkv), generator=g, device=DEV)
        pools[3][slots // 16, :, slots % 16] = torch.tensor(v_bytes, dtype=torch.uint8, device=DEV)[pick]
    return query, pools, tables, ctx, ql


TILES = 2.0 ** -32     # of the largest weight: half of fp16's least step under the kernel's shift


def _check_tight(pkg, query, pools, tables, ctx, ql, scale, most, floor):
    k, v = (ref.dequantise(pools[i].view(torch.uint8), pools[i + 2]) for i in (0, 1))
    got = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, scale, max_query_len=most)
    c, q = ctx.tolist(), ql.tolist()
    want, mean, slip = ref.attention(query, k, v, tables, c, q, scale)
    tol = ref.tight_tolerance(want, mean, slip, ref.lost_weight(tables, c, q, v, query.shape[1], floor), query.dtype,
                              query.shape[2])
    worst = ((got.double() - want).abs() / tol).max().item()
    assert worst <= 1.0, worst
    return got


# ------------------------------------------------------------------ weights far below the maximum
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("lengths", [[(700, 300)], [(2000, 60), (130, 30)]])
def test_long_chunks_keep_small_weights(pkg, dtype, hq, hkv, d, lengths):
    """Weights of e^-15 of the maximum, which was five steps of fp16's least number."""
    batch = _peaked(lengths, hq, hkv, d, dtype, 64, 15.0, (113, 120), seed=d)
    _check_tight(pkg, *batch, 1.0, max(q for _, q in lengths), TILES)
    assert "kv8_tiles" in pkg._lib.last_launches()
