"""The 8-bit cache's host side, no GPU: exported symbols, the tiling, refusals."""

from __future__ import annotations

import ctypes
import re
import subprocess

import numpy as np
import pytest
import torch

from _kv8_ref import e4m3_table, quantise


def test_library_exports_the_kv8_symbols(pkg):
    declared = pkg._lib.declared_symbols(pkg._lib.HEADER_KV8)
    assert len(declared) == 8
    dyn = subprocess.run(["nm", "-D", "--defined-only", str(pkg._lib.LIB_PATH)], capture_output=True, text=True).stdout
    for name in declared:
        assert f" T {name}" in dyn, name
        assert name in pkg._lib._SIGNATURES, name


def test_header_values_match_the_binding(pkg):
    text = pkg._lib.HEADER_KV8.read_text()
    values = dict(re.findall(r"^#define (PA_\w+) (\d+)", text, flags=re.M))
    assert len(values) >= 9
    for name, value in values.items():
        assert getattr(pkg._lib, name) == int(value), name


def test_header_is_plain_c(pkg, tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "paged_kv8_b200.h"\nint main(void) { pa_kv8_tiling t; t.row_groups = 0; return t.row_groups; }\n')
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Werror", "-I", str(pkg._lib.HEADER_KV8.parent), "-c", str(src),
                    "-o", str(tmp_path / "t.o")], check=True)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 12, 16])
def test_tiling_fits_its_kernels(pkg, group):
    for most in (0, 1, 2, 3, 4, 5, 8, 9, 16, 31, 33, 100, 4096):
        t = pkg.kv8._tiling(group, most, 10, 2 * most)
        assert t.row_groups in (1, 2, 3)
        assert t.small_tokens >= 1
        assert t.small_tokens * group <= 8 * t.row_groups
        assert 1 <= t.large_tokens * group <= 256
        assert t.small_max >= 0


def test_tiling_leaves_the_first_class_out_where_no_chunk_can_be_short(pkg):
    assert pkg.kv8._tiling(4, 500, 1, 500).small_max == 0
    assert pkg.kv8._tiling(4, 500, 3, 1007).small_max == 0     # 500 + 500 + 7
    assert pkg.kv8._tiling(4, 500, 3, 1006).small_max == 6
    assert pkg.kv8._tiling(4, 6, 1, 6).small_max == 6          # few rows: their kernel


def test_tiling_refusals(pkg):
    with pytest.raises(NotImplementedError, match="at most 16"):
        pkg.kv8._tiling(17, 1, 1, 1)
    with pytest.raises(ValueError):
        pkg.kv8._tiling(0, 1, 1, 1)


def test_the_reference_quantiser_is_torchs_rounding():
    """The tests' own e4m3 rounding agrees with torch's conversion where no scale is needed,
    so a payload compared with it is compared with the type's definition."""
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(40, 64, generator=g) * s for s in (0.01, 1.0, 60.0)]).clamp(-448, 448)
    x[:, 0] = 448.0                                 # the scale is 1
    codes, scale = quantise(x.numpy())
    assert (scale == 127).all()
    assert np.array_equal(codes, x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert np.array_equal(e4m3_table()[:127], torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())


def _cpu_pools(nb=4, bs=16, hkv=2, d=64):
    p = torch.zeros(nb, bs, hkv, d, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(nb, hkv, bs, dtype=torch.uint8)
    return p, p.clone(), s, s.clone()


def test_cpu_tensors_are_refused_without_a_fallback(pkg):
    k, v, ks, vs = _cpu_pools()
    row = torch.zeros(1, 2, 64)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="CUDA"):
        pkg.reshape_and_cache_kv8(row, row, k, v, ks, vs, one)
    with pytest.raises(NotImplementedError, match="CUDA"):
        pkg.paged_attention_kv8(row.half(), k, v, ks, vs, torch.zeros(1, 1, dtype=torch.int32), one, one, 1.0)
    with pytest.raises(NotImplementedError, match="CUDA"):
        pkg.device_step(torch.zeros(1, 1, dtype=torch.int32), one, one, num_tokens=1, max_query_len=1, num_blocks=4,
                        block_size=16)
    with pytest.raises(NotImplementedError, match="CUDA"):
        pkg.DeviceBlockTables(4, 4, 4, 16, "cpu")


def test_query_shape_is_checked_first(pkg):
    k, v, ks, vs = _cpu_pools()
    with pytest.raises(ValueError, match=r"\[num_tokens, heads, dim\]"):
        pkg.paged_attention_kv8(torch.zeros(4, 64), k, v, ks, vs, torch.zeros(1, 1, dtype=torch.int32),
                                torch.ones(1), torch.ones(1), 1.0)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(block_size=24), dict(block_size=8), dict(block_size=8192)])
def test_pool_refuses_shapes_without_a_kernel(pkg, kw):
    args = dict(num_layers=1, num_blocks=2, block_size=16, num_kv_heads=1, head_dim=64, device="cpu") | kw
    with pytest.raises(NotImplementedError):
        pkg.KV8Pool(**args)


def test_pool_layout(pkg):
    p = pkg.KV8Pool(2, 5, 32, 3, 128, "cpu")
    assert len(p.k) == len(p.v) == len(p.k_scale) == len(p.v_scale) == 2
    assert p.k[0].shape == (5, 32, 3, 128) and p.k[0].dtype == torch.float8_e4m3fn
    assert p.k_scale[1].shape == (5, 3, 32) and p.k_scale[1].dtype == torch.uint8
    assert p.nbytes == 2 * 2 * 5 * 32 * 3 * 129
    assert p.num_slots == 160


# ---- the C entry points check what the host can see before they touch the GPU
def _tiling(pkg, **kw):
    t = pkg._lib.Kv8Tiling(1, 1, 32, 1)
    for k, v in kw.items():
        setattr(t, k, v)
    return ctypes.byref(t)


_STEP = dict(row_ids=None, lens=16, query_lens=16, tables=16, stride=4, held=None, free=None, num_free=None, cap=0,
             rows=1, slots=1, width=4, bs=16, blocks=8, tokens=1, most=1, tiling=None, out_tables=None, ctx=16, ql=16,
             held_out=16, cu=16, seq=16, pos=16, slot=16, nf=16, work=16, stream=None)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(rows=-1), ValueError, "bad sizes"),
    (dict(width=5), ValueError, "bad sizes"),
    (dict(bs=0), ValueError, "bad sizes"),
    (dict(rows=4097, slots=5000), NotImplementedError, "at most 4096"),
    (dict(slots=131073), NotImplementedError, "request slots"),
    (dict(most=(1 << 20) + 1), NotImplementedError, "2\\^20"),
    (dict(blocks=1 << 28), NotImplementedError, "2\\^31"),
    (dict(rows=2), ValueError, "more rows than slots"),
    (dict(lens=None), ValueError, "NULL"),
    (dict(work=None), ValueError, "NULL"),
    (dict(tables=None), ValueError, "NULL"),
    (dict(held=16), ValueError, "NULL"),
    (dict(tiling="small_tokens"), ValueError, "tiling"),
])
def test_build_step_refusals(pkg, kw, exc, match):
    a = _STEP | kw
    a["tiling"] = _tiling(pkg, **({a["tiling"]: 0} if a["tiling"] else {}))
    with pytest.raises(exc, match=match):
        pkg._lib.check(pkg._lib.lib().pa_kv8_build_step(*a.values()))


_ATTN = dict(q=4096, qst=512, qsh=64, tokens=1, heads=8, dim=64, k=4096, v=4096, ks=4096, vs=4096, blocks=8, bs=16,
             hkv=8, dtype=1, scale=1.0, seqs=1, most=1, tables=16, stride=4, width=4, ctx=16, ql=16, cu=16, work=16, out=4096, ost=512,
             osh=64, ws=4096, wsb=1 << 40, stream=None)


@pytest.mark.parametrize("kw,exc,match", [
    (dict(dtype=0), NotImplementedError, "float16 and bfloat16"),
    (dict(dim=96), NotImplementedError, "head_dim 96"),
    (dict(hkv=3), ValueError, "not divisible"),
    (dict(heads=24, hkv=1), NotImplementedError, "at most 16"),
    (dict(bs=24), NotImplementedError, "block_size 24"),
    (dict(bs=8), NotImplementedError, "block_size 8"),
    (dict(blocks=1 << 28), NotImplementedError, "2\\^31"),
    (dict(tokens=-1), ValueError, "non-negative"),
    (dict(q=None), ValueError, "NULL"),
    (dict(ws=None), ValueError, "NULL"),
    (dict(q=4104), ValueError, "16-byte"),
    (dict(qst=516), ValueError, "16-byte"),
    (dict(out=4104), ValueError, "16-byte"),
    (dict(k=4100), ValueError, "16-byte"),
    (dict(vs=4100), ValueError, "16-byte"),
    (dict(wsb=16), RuntimeError, "workspace holds"),
    (dict(work=None), ValueError, "NULL"),
    (dict(cu=None), ValueError, "NULL"),
    (dict(work=None, cu=None, ql=None), ValueError, "NULL"),
    (dict(ws=4100), ValueError, "256-byte"),
])
def test_attention_refusals(pkg, kw, exc, match):
    a = _ATTN | kw
    with pytest.raises(exc, match=match):
        pkg._lib.check(pkg._lib.lib().pa_kv8_attention(*a.values()))


@pytest.mark.parametrize("kw,exc,match", [
    (dict(dtype=7), NotImplementedError, "dtype code"),
    (dict(dim=80), NotImplementedError, "head_dim 80"),
    (dict(hkv=0), ValueError, "append shape"),
    (dict(slots=None), ValueError, "NULL"),
    (dict(kp=4100), ValueError, "16-byte"),
    (dict(tokens=1 << 30, hkv=4), NotImplementedError, "2\\^31"),
])
def test_append_refusals(pkg, kw, exc, match):
    a = dict(key=16, kst=64, ksh=64, value=16, vst=64, vsh=64, tokens=1, hkv=1, dim=64, dtype=1, kp=4096, vp=4096,
             ks=4096, vs=4096, blocks=4, bs=16, slots=16, stream=None) | kw
    with pytest.raises(exc, match=match):
        pkg._lib.check(pkg._lib.lib().pa_kv8_append(*a.values()))


def test_commit_and_release_refusals(pkg):
    lib, check = pkg._lib.lib(), pkg._lib.check
    with pytest.raises(ValueError, match="NULL"):
        check(lib.pa_kv8_commit(None, 16, None, 16, None, 1, 1, 16, 16, 16, None))
    with pytest.raises(ValueError, match="bad sizes"):
        check(lib.pa_kv8_release(16, -1, 16, 4, 4, 1, 16, 16, 16, 4, 16, None))
    with pytest.raises(NotImplementedError, match="at most"):
        check(lib.pa_kv8_release(16, 5000, 16, 4, 4, 1, 16, 16, 16, 4, 16, None))
    check(lib.pa_kv8_release(None, 0, None, 4, 4, 1, None, None, None, 4, None, None))  # nothing to do


def test_attention_over_a_pool_without_blocks_is_refused(pkg):
    """It returned at once, the output unwritten and nothing reported."""
    with pytest.raises(ValueError, match="no blocks"):
        pkg._lib.check(pkg._lib.lib().pa_kv8_attention(*(_ATTN | dict(blocks=0)).values()))
    for nothing in (dict(tokens=0), dict(seqs=0)):
        pkg._lib.check(pkg._lib.lib().pa_kv8_attention(*(_ATTN | dict(blocks=0) | nothing).values()))
