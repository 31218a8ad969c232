"""The 8-bit paged cache on the GPU against plain 64-bit forms (tests/_kv8_ref.py)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _kv8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error(pkg, request):
    yield
    word = pkg.read_kv8_error(DEV)
    if "reports" not in request.node.name:
        assert word == 0


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ tables and slots
def _state(rng, requests, width, bs, most):
    lens = rng.integers(0, most + 1, size=requests).astype(np.int32)
    held = (-(-lens // bs) + rng.integers(0, 2, size=requests)).clip(0, width).astype(np.int32)
    nb = int(held.sum()) + 4 * requests + 64
    perm = rng.permutation(nb).astype(np.int32)
    tables = rng.integers(0, nb, size=(requests, width)).astype(np.int32)   # stale ids behind the held ones
    at = 0
    for r in range(requests):
        tables[r, :held[r]] = perm[at:at + held[r]]
        at += held[r]
    return lens, held, tables, perm[at:].copy(), nb


STEP_OUT = ["context_lens", "query_lens", "held", "cu_query_lens", "seq_idx", "q_pos", "slot_mapping", "num_free"]


@pytest.mark.parametrize("bs", [1, 16, 24, 64])
@pytest.mark.parametrize("requests,rows,chunk", [(1, 1, 1), (7, 5, 3), (40, 33, 17), (600, 513, 1), (1100, 1025, 5),
                                                 (30, 9, 700)])
def test_reserve_matches_the_loops(pkg, bs, requests, rows, chunk):
    rng = np.random.default_rng(requests * 100 + chunk + bs)
    most = 40 * bs
    width = -(-(most + chunk) // bs) + 3
    lens, held, tables, free, nb = _state(rng, requests, width, bs, most)
    free = np.concatenate([free, nb + np.arange(rows * (-(-chunk // bs) + 1), dtype=np.int32)])
    nb = max(nb, int(free.max()) + 1)
    ids = rng.permutation(requests)[:rows].astype(np.int32)
    ql = rng.integers(0, chunk + 1, size=rows).astype(np.int32)
    ql[0] = chunk
    if rows > 4:
        ids[2] = -1                                  # a padding row in the middle and at the end
        ids[rows - 1] = -1
    tokens = int(ql[ids >= 0].sum()) + 5             # five tokens of padding
    nf = len(free) - 3                               # the list's capacity is more than its length
    want = ref.step_tables(ids, ql, tables, lens, held, free, nf, width, bs, tokens)
    bt = pkg.DeviceBlockTables.adopt(_i32(tables), _i32(lens), _i32(held), _i32(free), _i32([nf]), num_blocks=nb,
                                     block_size=bs)
    step = bt.reserve(_i32(ids), _i32(ql), num_tokens=tokens, max_query_len=chunk)
    for name in STEP_OUT + ["block_tables"]:
        np.testing.assert_array_equal(getattr(step, name).cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(bt.tables.cpu().numpy(), want["tables"])
    np.testing.assert_array_equal(bt.lens.cpu().numpy(), lens)          # nothing counts before commit
    again = bt.reserve(_i32(ids).long(), _i32(ql).long(), num_tokens=tokens, max_query_len=chunk, out=step)
    assert again is step
    for name in STEP_OUT + ["block_tables"]:
        np.testing.assert_array_equal(getattr(step, name).cpu().numpy(), want[name], err_msg=name)


def test_step_work_sums_are_the_keys_of_the_tiles(pkg):
    """work[class, i]: keys that the tiles of the sequences before i visit."""
    rng = np.random.default_rng(4)
    for group, most in ((1, 1), (4, 1), (4, 5), (3, 40), (8, 300)):
        b = 65
        ql = rng.integers(0, most + 1, size=b)
        ctx = ql + rng.integers(0, 500, size=b)
        t = pkg.kv8._tiling(group, most, b, int(ql.sum()))
        step = pkg.device_step(torch.zeros(b, 64, dtype=torch.int32, device=DEV), _i32(ctx), _i32(ql),
                               num_tokens=int(ql.sum()), max_query_len=most, num_blocks=1, block_size=16, group=group)
        want = np.zeros((2, b + 1), np.int64)
        for i in range(b):
            few = ql[i] <= t.small_max
            tt = t.small_tokens if few else t.large_tokens
            keys = sum(int(ctx[i] - ql[i]) + min(a + tt, int(ql[i])) for a in range(0, int(ql[i]), tt))
            want[:, i + 1] = want[:, i]
            want[0 if few else 1, i + 1] += keys
        np.testing.assert_array_equal(step.work.cpu().numpy(), want)


@pytest.mark.parametrize("b,width,chunk,bs", [(1, 1, 1, 16), (3, 5, 4, 16), (70, 40, 9, 32), (1030, 8, 1, 16)])
def test_device_step_over_given_tables(pkg, b, width, chunk, bs):
    rng = np.random.default_rng(b)
    nb = 500
    wide = rng.integers(0, nb, size=(b, width + 3)).astype(np.int32)
    ctx = rng.integers(chunk, width * bs + 1, size=b).astype(np.int32)
    ql = rng.integers(0, chunk + 1, size=b).astype(np.int32)
    ctx[-1], ql[-1] = 0, 0
    tokens = int(ql.sum()) + 2
    tables = _i32(wide)[:, :width]                                      # rows of a wider table
    step = pkg.device_step(tables, _i32(ctx), _i32(ql), num_tokens=tokens, max_query_len=chunk, num_blocks=nb,
                           block_size=bs)
    seq, pos, slot = np.full(tokens, -1), np.full(tokens, -1), np.full(tokens, -1)
    at = 0
    for i in range(b):
        for t in range(ql[i]):
            p = ctx[i] - ql[i] + t
            seq[at], pos[at], slot[at] = i, p, wide[i, p // bs] * bs + p % bs
            at += 1
    np.testing.assert_array_equal(step.seq_idx.cpu().numpy(), seq)
    np.testing.assert_array_equal(step.q_pos.cpu().numpy(), pos)
    np.testing.assert_array_equal(step.slot_mapping.cpu().numpy(), slot)
    np.testing.assert_array_equal(step.cu_query_lens.cpu().numpy(), np.concatenate([[0], np.cumsum(ql)]))
    assert step.block_tables.data_ptr() == tables.data_ptr()


def test_tables_over_many_steps(pkg):
    """Admission, chunks, partly accepted speculation and release, against loops over Python
    lists; the blocks of the slots and the free list stay a partition of the pool."""
    rng = np.random.default_rng(11)
    requests, width, bs, nb = 12, 20, 16, 150
    bt = pkg.DeviceBlockTables(requests, width, nb, bs, DEV)
    tables, lens, held = np.zeros((requests, width), np.int32), np.zeros(requests, int), np.zeros(requests, int)
    free, nf = np.arange(nb - 1, -1, -1), nb
    for step_no in range(40):
        live = rng.permutation(requests)[:int(rng.integers(1, requests + 1))]
        room = width * bs - lens[live]
        chunk = int(rng.choice([1, 4, 50]))
        ql = np.minimum(rng.integers(0, chunk + 1, size=len(live)), room)
        need = np.maximum(-(-(lens[live] + ql) // bs) - held[live], 0).sum()
        if need > nf:
            drop = live[:max(1, len(live) // 2)]
            bt.release(_i32(drop))
            for r in drop:
                free[nf:nf + held[r]] = tables[r, :held[r]][::-1]
                nf += held[r]
                lens[r] = held[r] = 0
            assert int(bt.num_free) == nf
            np.testing.assert_array_equal(bt.free.cpu().numpy()[:nf], free[:nf])
            continue
        tokens = int(ql.sum())
        want = ref.step_tables(live, ql, tables, lens, held, free, nf, width, bs, tokens)
        step = bt.reserve(_i32(live), _i32(ql), num_tokens=tokens, max_query_len=chunk)
        for name in STEP_OUT + ["block_tables"]:
            np.testing.assert_array_equal(getattr(step, name).cpu().numpy(), want[name], err_msg=name)
        accepted = rng.integers(0, 60, size=len(live)) if step_no % 3 == 0 else None
        bt.commit(step, None if accepted is None else _i32(accepted))
        tables, nf = want["tables"], int(want["num_free"][0])
        lens[live] += ql if accepted is None else np.minimum(accepted, ql)
        held[live] = want["held"]
        np.testing.assert_array_equal(bt.lens.cpu().numpy(), lens)
        np.testing.assert_array_equal(bt.held.cpu().numpy(), held)
        assert int(bt.num_free) == nf
        owned = [tables[r, j] for r in range(requests) for j in range(held[r])] + list(free[:nf])
        assert sorted(owned) == list(range(nb))


@pytest.mark.parametrize("what", ["twice", "range", "negative", "tokens", "chunk", "width", "blocks", "list"])
def test_a_bad_step_is_emptied_and_reports(pkg, what):
    requests, width, bs, nb = 8, 4, 16, 20
    bt = pkg.DeviceBlockTables(requests, width, nb, bs, DEV)
    ids, ql, tokens, bit = [0, 3, 5], [2, 7, 1], 10, pkg._lib.PA_KV8_ERR_STEP
    if what == "twice":
        ids = [0, 3, 0]
    elif what == "range":
        ids = [0, 8, 5]
    elif what == "negative":
        ql = [2, -1, 1]
    elif what == "tokens":
        tokens = 9
    elif what == "chunk":
        ql = [2, 9, 1]
    elif what == "width":
        bt.lens[3] = 60
        bt.held[3] = 4
    elif what == "blocks":
        bt.num_free.fill_(2)
        bit = pkg._lib.PA_KV8_ERR_NO_BLOCKS
    else:
        bt.num_free.fill_(nb + 1)
    before = [t.clone() for t in (bt.tables, bt.lens, bt.held, bt.num_free)]
    step = bt.reserve(_i32(ids), _i32(ql), num_tokens=tokens, max_query_len=8)
    assert int(step.num_free) == -1
    assert not step.context_lens.any() and not step.cu_query_lens.any() and not step.work.any()
    assert not step.block_tables.any() and not step.held.any() and not step.query_lens.any()
    assert (step.slot_mapping == -1).all() and (step.seq_idx == -1).all() and (step.q_pos == -1).all()
    bt.commit(step)
    for a, b in zip(before, (bt.tables, bt.lens, bt.held, bt.num_free)):
        assert torch.equal(a, b)
    assert pkg.read_kv8_error(DEV) == bit
    assert pkg.read_kv8_error(DEV) == 0


def test_release_of_a_slot_twice_changes_nothing_and_reports(pkg):
    bt = pkg.DeviceBlockTables(4, 4, 20, 16, DEV)
    step = bt.reserve(_i32([0, 1]), _i32([20, 3]), num_tokens=23, max_query_len=20)
    bt.commit(step)
    before = [t.clone() for t in (bt.lens, bt.held, bt.num_free, bt.free)]
    bt.release(_i32([1, -1, 1]))
    for a, b in zip(before, (bt.lens, bt.held, bt.num_free, bt.free)):
        assert torch.equal(a, b)
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP
    bt.release(_i32([1, -1, 0]))
    assert int(bt.num_free) == 20 and not bt.lens.any() and not bt.held.any()
    assert sorted(bt.free.tolist()) == list(range(20))


def test_block_ids_outside_the_pool_are_not_mapped_and_reports(pkg):
    tables = _i32([[0, 9], [12, 1]])
    step = pkg.device_step(tables, _i32([17, 3]), _i32([2, 1]), num_tokens=3, max_query_len=2, num_blocks=9,
                           block_size=16)
    assert step.slot_mapping.tolist() == [15, -1, -1]
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_BLOCK


# ------------------------------------------------------------------ append
def _pools(nb, bs, hkv, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    def one(*shape):
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(DEV)
    return (one(nb, bs, hkv, d).view(ref.E4M3), one(nb, bs, hkv, d).view(ref.E4M3), one(nb, hkv, bs),
            one(nb, hkv, bs))


def _check_append(pkg, key, value, nb, bs, slots):
    t, hkv, d = key.shape
    pools = _pools(nb, bs, hkv, d)
    before = [p.view(torch.uint8).cpu().numpy().copy() for p in pools]
    pkg.reshape_and_cache_kv8(key, value, *pools, slots)
    torch.cuda.synchronize()
    at = slots.cpu().numpy()
    for x, payload, scale, got_p, got_s in ((key, before[0], before[2], pools[0], pools[2]),
                                            (value, before[1], before[3], pools[1], pools[3])):
        codes, byte = ref.quantise(x.double().cpu().numpy())
        for i, s in enumerate(at):
            if 0 <= s < nb * bs:
                payload[s // bs, s % bs] = codes[i]
                scale[s // bs, :, s % bs] = byte[i]
        np.testing.assert_array_equal(got_s.cpu().numpy(), scale)
        np.testing.assert_array_equal(got_p.view(torch.uint8).cpu().numpy(), payload)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,hkv,d,bs", [(1, 1, 64, 16), (3, 2, 128, 16), (37, 12, 64, 32), (130, 8, 128, 16),
                                        (5, 3, 128, 48)])
def test_append_is_bit_exact(pkg, dtype, t, hkv, d, bs):
    g = torch.Generator().manual_seed(t + d)
    kv = torch.randn(t, 2 * hkv, d, generator=g) * torch.exp(2.5 * torch.randn(t, 2 * hkv, 1, generator=g))
    kv = kv.to(dtype).to(DEV)
    nb = t // bs + 4
    slots = torch.randperm(nb * bs, generator=g)[:t].to(DEV)
    _check_append(pkg, kv[:, :hkv], kv[:, hkv:], nb, bs, slots)


def test_append_of_special_rows(pkg):
    """Zero rows, largest magnitudes on the scale's steps and one unit past them, rounding
    ties, subnormals, values past the range, infinities and NaN."""
    d = 64
    rows = [torch.zeros(d), torch.full((d,), -0.0), torch.full((d,), 448.0), torch.full((d,), 448.0 * 2 ** -14),
            torch.full((d,), 2.0 ** -24), torch.full((d,), 57344.0), torch.full((d,), -65504.0)]
    for k in (-16, -14, -3, 0, 1, 7):
        for top in (1.75, 1.7509765625, 1.0, 1.9990234375):
            r = torch.linspace(-1, 1, d) * top * 2.0 ** (k + 8)
            r[0], r[1] = top * 2.0 ** (k + 8), 0.0
            rows.append(r.clamp(-65504, 65504))
    ties = (torch.arange(d) * 0.0625 + 1.0) * 16.0                     # midpoints between e4m3 values
    ties[0] = 448.0
    rows.append(ties)
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = torch.linspace(-3, 3, d)
        r[d // 2 + 1] = bad
        rows.append(r)
    x = torch.stack(rows)[:, None]
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        y = x.to(dtype).to(DEV)
        _check_append(pkg, y, y.flip(0).contiguous(), 8, 16, torch.arange(3, 3 + len(rows), device=DEV))
    wide = torch.tensor([1e30, -3e38, 1e-38, 1.0]).repeat(16)[None, None].to(DEV)
    _check_append(pkg, wide, wide, 1, 16, torch.tensor([5], device=DEV))
    _check_append(pkg, wide.bfloat16(), wide.bfloat16(), 1, 16, torch.tensor([5], device=DEV))


def test_append_passes_over_slots_outside_the_pool(pkg):
    x = torch.randn(6, 2, 64, device=DEV)
    _check_append(pkg, x, -x, 2, 16, torch.tensor([-1, 31, 32, 0, 1 << 30, -7], device=DEV))


def test_append_odd_strides(pkg):
    base = torch.randn(9, 3, 131, device=DEV).half()
    _check_append(pkg, base[:, :, 1:129], base[:, :, 3:131], 3, 16, torch.arange(9, device=DEV) * 4)
    cross = torch.randn(2, 128, 11, device=DEV).bfloat16().permute(2, 0, 1)     # no unit stride
    _check_append(pkg, cross, cross * 2, 3, 16, torch.arange(11, device=DEV) * 4)
    _check_append(pkg, base[:0, :, :64], base[:0, :, :64], 1, 16, torch.zeros(0, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------ attention
def _batch(lengths, hq, hkv, d, bs, dtype, seed=0, spread=1.0, pad_tokens=0, extra_width=0):
    """Pools of random bytes (NaN codes and wild scales among them) with valid rows at the
    contexts' slots only."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // bs) for c, _ in lengths]
    nb = sum(need) + 3
    pools = _pools(nb, bs, hkv, d, seed)
    perm = torch.randperm(nb, generator=g)
    w = max(need + [1]) + extra_width
    tables = torch.randint(0, nb, (len(lengths), w), generator=g, dtype=torch.int32)
    at, slots = 0, []
    for i, (n, (c, _)) in enumerate(zip(need, lengths)):
        tables[i, :n] = perm[at:at + n]
        at += n
        p = torch.arange(c)
        slots.append(tables[i].long()[p // bs] * bs + p % bs)
    slots = torch.cat(slots).to(DEV)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    total = slots.numel()
    for pool, scale in ((pools[0], pools[2]), (pools[1], pools[3])):
        x = torch.randn(total, hkv, d, generator=gd, device=DEV) * spread
        x *= torch.exp(0.7 * torch.randn(total, hkv, 1, generator=gd, device=DEV))
        big = x.abs().amax(-1)
        e = torch.ceil(torch.log2(big / 448.0)).clamp(-14, 7)          # any scale will do here
        raw = (x * torch.exp2(-e)[..., None]).clamp(-448, 448).to(ref.E4M3)
        pool.view(torch.uint8).view(-1, hkv, d)[slots] = raw.view(torch.uint8)
        scale[slots // bs, :, slots % bs] = (e + 127).to(torch.uint8)
    t = sum(q for _, q in lengths) + pad_tokens
    query = torch.randn(t, hq, d, generator=gd, device=DEV).to(dtype)
    ctx, ql = _i32([c for c, _ in lengths]), _i32([q for _, q in lengths])
    return query, pools, tables.to(DEV), ctx, ql


def _check_attention(pkg, query, pools, tables, ctx, ql, scale, most=None, out=None):
    k, v = (ref.dequantise(pools[i].view(torch.uint8), pools[i + 2]) for i in (0, 1))
    got = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, scale, max_query_len=most, out=out)
    c, q = ctx.tolist(), ql.tolist()
    want, mean, slip = ref.attention(query, k, v, tables, c, q, scale)
    tol = ref.tolerance(want, mean, slip, query.dtype, query.shape[2], max(c + [1]))
    n = sum(q)
    assert not got[:n].isnan().any()
    worst = ((got[:n].double() - want[:n]).abs() / tol[:n]).max().item() if n else 0.0
    assert worst <= 1.0, worst
    return got


LENGTHS = {
    "one": [(1, 1)],
    "decode": [(517, 1), (1, 1), (16, 1), (17, 1), (300, 1), (15, 1)],
    "long": [(9000, 1), (33, 1)],
    "verify": [(600, 5), (5, 5), (40, 1), (17, 3), (2100, 4)],
    "empty rows": [(0, 0), (100, 1), (64, 0), (48, 2), (0, 0)],
    "chunks": [(333, 77), (130, 130), (64, 1), (500, 33)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (12, 12, 64), (8, 1, 128), (16, 1, 64), (6, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("which", list(LENGTHS))
def test_attention_matches_64_bits(pkg, dtype, hq, hkv, d, which):
    batch = _batch(LENGTHS[which], hq, hkv, d, 16, dtype, seed=hq + d, extra_width=2)
    _check_attention(pkg, *batch, d ** -0.5, most=max(q for _, q in LENGTHS[which]))


@pytest.mark.parametrize("bs", [32, 64, 256])
def test_attention_other_block_sizes(pkg, bs):
    batch = _batch([(517, 1), (70, 3), (1, 1), (2000, 2)], 8, 2, 128, bs, torch.bfloat16, seed=bs)
    _check_attention(pkg, *batch, 0.1, most=3)


def test_attention_splits_and_many_sequences(pkg):
    """More sequences than the grid has slices, so that a CTA walks several; then few and
    long ones, which several CTAs share."""
    rng = np.random.default_rng(0)
    many = [(int(c), 1) for c in rng.integers(1, 200, size=700)]
    _check_attention(pkg, *_batch(many, 8, 2, 64, 16, torch.bfloat16, seed=3), 0.125, most=1)
    mixed = [(int(c), min(int(c), int(q))) for c, q in zip(rng.integers(1, 3000, size=60), rng.integers(1, 9, size=60))]
    _check_attention(pkg, *_batch(mixed, 8, 8, 128, 16, torch.float16, seed=4), 0.09, most=8)
    _check_attention(pkg, *_batch([(40000, 2)], 16, 4, 128, 16, torch.bfloat16, seed=5), 0.09, most=2)


def test_attention_default_bound_and_padding_tokens(pkg):
    """max_query_len left out; rows of `out` past the last sequence stay as they were."""
    query, pools, tables, ctx, ql = _batch([(90, 2), (40, 7)], 8, 2, 128, 16, torch.bfloat16, seed=8, pad_tokens=6)
    out = torch.full_like(query, 7.0)
    got = _check_attention(pkg, query, pools, tables, ctx, ql, 0.1, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (got[9:] == 7.0).all()


def test_attention_strided_queries(pkg):
    query, pools, tables, ctx, ql = _batch([(90, 2), (40, 1)], 8, 2, 128, 16, torch.bfloat16, seed=9)
    wide = torch.randn(3, 24, 128, device=DEV).bfloat16()
    wide[:, 5:13] = query
    _check_attention(pkg, wide[:, 5:13], pools, tables, ctx, ql, 0.1, most=2)
    odd = torch.randn(3, 8, 131, device=DEV).bfloat16()
    odd[:, :, 1:129] = query
    _check_attention(pkg, odd[:, :, 1:129], pools, tables, ctx, ql, 0.1, most=2)
    turned = query.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    _check_attention(pkg, turned, pools, tables, ctx, ql, 0.1, most=2)


@pytest.mark.parametrize("factor", [2.0 ** -100, 2.0 ** -20, 2.0 ** 20, 2.0 ** 100])
def test_attention_queries_far_outside_fp16(pkg, factor):
    """bf16 queries of any magnitude, with the softmax scale that brings the scores back."""
    query, pools, tables, ctx, ql = _batch([(300, 1), (40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=10)
    _check_attention(pkg, query * factor, pools, tables, ctx, ql, 0.1 / factor, most=3)


def test_attention_steep_scores(pkg):
    """Softmax far from uniform: maxima that keep moving, weights down to nothing."""
    query, pools, tables, ctx, ql = _batch([(2000, 1), (900, 5)], 8, 2, 128, 16, torch.float16, seed=12, spread=2.0)
    _check_attention(pkg, query * 8, pools, tables, ctx, ql, 0.3, most=5)


def test_attention_small_and_mixed_value_scales(pkg):
    """V rows whose scale is the smallest beside ordinary ones: the weights carry the scale."""
    query, pools, tables, ctx, ql = _batch([(700, 2)], 8, 2, 128, 16, torch.float16, seed=13)
    pools[3][pools[3] <= 134] = 113
    _check_attention(pkg, query, pools, tables, ctx, ql, 0.1, most=2)
    pools[3][::2] = torch.where(pools[3][::2] == 113, 134, pools[3][::2])
    _check_attention(pkg, query, pools, tables, ctx, ql, 0.1, most=2)


def test_a_nan_row_reaches_only_the_tokens_that_see_it(pkg):
    lengths = [(40, 6), (30, 2)]
    query, pools, tables, ctx, ql = _batch(lengths, 8, 2, 128, 16, torch.bfloat16, seed=14)
    clean = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=6)
    for which in (0, 1):                              # a K row, then a V row
        p = [x.clone() for x in pools]
        pos = 37                                      # seen by the tokens at 37, 38, 39 of the first sequence
        slot = int(tables[0, pos // 16]) * 16 + pos % 16
        p[which].view(torch.uint8).view(-1, 2, 128)[slot] = 0
        p[which + 2][slot // 16, 1, slot % 16] = 255
        got = pkg.paged_attention_kv8(query, *p, tables, ctx, ql, 0.1, max_query_len=6)
        assert got[3:6, 4:].isnan().all()
        got[3:6, 4:] = clean[3:6, 4:]
        got[3:6, :4], clean2 = clean[3:6, :4], clean
        assert torch.equal(got, clean2)


TILES = {
    "one tile": [(64, 64)],
    "prompt": [(333, 333)],
    "prompts": [(700, 700), (65, 65), (129, 129), (1, 1), (2, 2)],
    "chunk over a prefix": [(3000, 100)],
    "split along the context": [(9000, 40), (700, 90)],
    "mixed with decodes": [(500, 1), (1200, 150), (64, 2), (900, 33), (0, 0), (77, 70)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (12, 12, 64), (14, 2, 128), (16, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("which", list(TILES))
def test_attention_of_long_chunks(pkg, dtype, hq, hkv, d, which):
    lengths = TILES[which]
    batch = _batch(lengths, hq, hkv, d, 16, dtype, seed=hq * d, extra_width=1)
    _check_attention(pkg, *batch, d ** -0.5, most=max(q for _, q in lengths))
    assert "kv8_tiles" in pkg._lib.last_launches()


@pytest.mark.parametrize("bs", [32, 128])
def test_long_chunks_other_block_sizes(pkg, bs):
    batch = _batch([(517, 100), (70, 3), (1000, 64)], 8, 2, 128, bs, torch.bfloat16, seed=bs)
    _check_attention(pkg, *batch, 0.1, most=100)


def test_long_chunks_steep_scores_and_signs(pkg):
    """Maxima that move past the headroom, a negative and a zero softmax scale, queries far
    outside fp16."""
    lengths = [(1500, 70), (400, 400)]
    for dtype, q_factor, scale in ((torch.float16, 8.0, 0.3), (torch.bfloat16, 1.0, -0.2), (torch.bfloat16, 1.0, 0.0),
                                   (torch.bfloat16, 2.0 ** -90, 0.1 * 2.0 ** 90), (torch.bfloat16, 2.0 ** 80, 2.0 ** -83)):
        query, pools, tables, ctx, ql = _batch(lengths, 8, 2, 128, 16, dtype, seed=21, spread=2.0)
        _check_attention(pkg, query * q_factor, pools, tables, ctx, ql, scale, most=400)


@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_few_rows_negative_and_zero_scale(pkg, scale):
    query, pools, tables, ctx, ql = _batch([(700, 2), (33, 1)], 8, 2, 128, 16, torch.bfloat16, seed=22)
    _check_attention(pkg, query, pools, tables, ctx, ql, scale, most=2)


def test_long_chunks_ascending_scores(pkg):
    """Scores that grow along the context: the running maximum rises in every tile."""
    query, pools, tables, ctx, ql = _batch([(2000, 64)], 4, 1, 128, 16, torch.bfloat16, seed=23)
    pools[2].fill_(120)
    k = pools[0].view(torch.uint8)
    pos = torch.arange(2000, device=DEV)
    slots = tables[0].long()[pos // 16] * 16 + pos % 16
    ramp = (pos.float() / 2000 * 400).to(ref.E4M3).view(torch.uint8)
    k.view(-1, 1, 128)[slots] = ramp[:, None, None]
    _check_attention(pkg, query.abs(), pools, tables, ctx, ql, 0.09, most=64)


def test_a_nan_row_in_a_long_chunk_reaches_only_the_tokens_that_see_it(pkg):
    query, pools, tables, ctx, ql = _batch([(300, 100), (90, 80)], 8, 2, 128, 16, torch.bfloat16, seed=24)
    clean = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=100)
    for which in (0, 1):
        p = [x.clone() for x in pools]
        pos = 237                                     # token 37 of the first sequence
        slot = int(tables[0, pos // 16]) * 16 + pos % 16
        p[which].view(torch.uint8).view(-1, 2, 128)[slot] = 0
        p[which + 2][slot // 16, 0, slot % 16] = 255
        got = pkg.paged_attention_kv8(query, *p, tables, ctx, ql, 0.1, max_query_len=100)
        assert got[37:100, :4].isnan().all() and not got[37:100, 4:].isnan().any()
        got[37:100] = clean[37:100]                   # the other head's row there was zeroed with it
        assert torch.equal(got, clean)


def test_attention_is_deterministic_and_independent_of_neighbours(pkg):
    lengths = [(700, 2), (33, 1), (1500, 3)]
    query, pools, tables, ctx, ql = _batch(lengths, 8, 2, 128, 16, torch.bfloat16, seed=15)
    a = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=3)
    for _ in range(3):
        assert torch.equal(a, pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=3))


def test_attention_with_an_attached_step(pkg):
    lengths = [(700, 2), (33, 1), (1500, 3)]
    query, pools, tables, ctx, ql = _batch(lengths, 8, 2, 128, 16, torch.bfloat16, seed=16)
    a = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=3)
    step = pkg.device_step(tables, ctx, ql, num_tokens=6, max_query_len=3, num_blocks=pools[0].shape[0], block_size=16,
                           group=4)
    riding = pkg.kv8.attach_step(torch.empty(0, dtype=torch.int32, device=DEV), step)
    assert torch.equal(a, pkg.paged_attention_kv8(query, *pools, riding, None, None, 0.1))


def test_an_emptied_step_leaves_the_output_alone_and_reports(pkg):
    query, pools, tables, ctx, ql = _batch([(40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=17)
    out = torch.full_like(query, 3.0)
    pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=2, out=out)     # the chunk is longer
    assert (out == 3.0).all()
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_attention_checks_block_ids_and_reports(pkg):
    query, pools, tables, ctx, ql = _batch([(40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=18)
    tables[0, 1] = pools[0].shape[0]
    pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=3)
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_BLOCK


def test_refusals(pkg):
    query, pools, tables, ctx, ql = _batch([(40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=19)
    k, v, ks, vs = pools
    call = pkg.paged_attention_kv8
    with pytest.raises(NotImplementedError, match="float16 and bfloat16"):
        call(query.float(), *pools, tables, ctx, ql, 0.1)
    with pytest.raises(ValueError, match="k_pool must be"):
        call(query, k.view(torch.uint8), v, ks, vs, tables, ctx, ql, 0.1)
    with pytest.raises(ValueError, match="k_scale must be contiguous"):
        call(query, k, v, ks[:, :1], vs, tables, ctx, ql, 0.1)
    with pytest.raises(ValueError, match="not divisible"):
        call(query[:, :7], *pools, tables, ctx, ql, 0.1)
    with pytest.raises(ValueError, match="head_dim"):
        call(query[..., :64], *pools, tables, ctx, ql, 0.1)
    with pytest.raises(ValueError, match="match block_tables"):
        call(query, *pools, tables, ctx[:0], ql, 0.1)
    with pytest.raises(ValueError, match="expected"):
        call(query, *pools, tables, ctx.cpu(), ql, 0.1)
    with pytest.raises(ValueError, match="out must be"):
        call(query, *pools, tables, ctx, ql, 0.1, out=torch.empty(3, 8, 64, device=DEV))
    with pytest.raises(ValueError, match="int32 or int64"):
        pkg.device_step(tables, ctx.float(), ql, num_tokens=3, max_query_len=3, num_blocks=9, block_size=16)
    with pytest.raises(ValueError, match="key rows"):
        pkg.reshape_and_cache_kv8(query, query, *pools, torch.zeros(3, dtype=torch.int32, device=DEV))
    bt = pkg.DeviceBlockTables(4, 4, 20, 16, DEV)
    with pytest.raises(ValueError, match="made by reserve"):
        bt.commit(pkg.device_step(tables, ctx, ql, num_tokens=3, max_query_len=3, num_blocks=9, block_size=16))
    with pytest.raises(ValueError, match="contiguous int32"):
        pkg.DeviceBlockTables.adopt(bt.tables.long(), bt.lens, bt.held, bt.free, bt.num_free, num_blocks=20, block_size=16)


# ------------------------------------------------------------------ together
def _decode_loop(pkg, steps, stream=None, graph=False):
    """A decode loop that lives on the GPU: reserve, append, attend, commit; new K/V rows are
    made from the positions, queries from the step's number."""
    hq, hkv, d, bs, nb, r, w = 8, 2, 128, 16, 64, 4, 12
    pool = pkg.KV8Pool(1, nb, bs, hkv, d, DEV)
    bt = pkg.DeviceBlockTables(r, w, nb, bs, DEV)
    ids, one = _i32([2, 0, 3]), _i32([1, 1, 1])
    g = torch.Generator(device=DEV).manual_seed(1)
    feed = torch.randn(steps, 3, hq + 2 * hkv, d, generator=g, device=DEV).bfloat16()
    x = torch.zeros(3, hq + 2 * hkv, d, device=DEV).bfloat16()
    outs = []

    def prompt():
        q = _i32([21, 5, 40])
        t = 66
        kv = torch.randn(t, 2 * hkv, d, generator=g, device=DEV).bfloat16()
        step = bt.reserve(ids, q, num_tokens=t, max_query_len=40, group=4)
        pkg.reshape_and_cache_kv8(kv[:, :hkv], kv[:, hkv:], pool.k[0], pool.v[0], pool.k_scale[0], pool.v_scale[0],
                                  step.slot_mapping)
        bt.commit(step)

    def decode():
        step = bt.reserve(ids, one, num_tokens=3, max_query_len=1, group=4)
        pkg.reshape_and_cache_kv8(x[:, hq:hq + hkv], x[:, hq + hkv:], pool.k[0], pool.v[0], pool.k_scale[0],
                                  pool.v_scale[0], step.slot_mapping)
        out = pkg.paged_attention_kv8(x[:, :hq], pool.k[0], pool.v[0], pool.k_scale[0], pool.v_scale[0],
                                      pkg.kv8.attach_step(step.block_tables, step), None, None, d ** -0.5)
        bt.commit(step)
        return out

    prompt()
    replay = None
    for i in range(steps):
        x.copy_(feed[i])
        if graph and i == 2:
            torch.cuda.synchronize()
            replay = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(replay, stream=side):
                captured = decode()
            torch.cuda.current_stream().wait_stream(side)
        if replay is not None:
            replay.replay()
            outs.append(captured.clone())
        else:
            outs.append(decode())
    torch.cuda.synchronize()
    return torch.stack(outs), pool, bt, feed


def test_a_decode_loop_on_the_gpu(pkg):
    """The operators together; the attention is checked against 64 bits over the cache's own
    values at the last step, and the captured loop and one on another stream give the same."""
    steps = 30
    outs, pool, bt, feed = _decode_loop(pkg, steps)
    assert bt.lens.tolist() == [5 + steps, 0, 21 + steps, 40 + steps]
    k, v = (ref.dequantise(a.view(torch.uint8), s) for a, s in ((pool.k[0], pool.k_scale[0]), (pool.v[0], pool.v_scale[0])))
    order = [2, 0, 3]
    ctx = [int(bt.lens[i]) for i in order]
    want, mean, slip = ref.attention(feed[-1][:, :8], k, v, bt.tables[order], ctx, [1, 1, 1], 128 ** -0.5)
    tol = ref.tolerance(want, mean, slip, torch.bfloat16, 128, max(ctx))
    assert ((outs[-1].double() - want).abs() <= tol).all()
    again, pool2, bt2, _ = _decode_loop(pkg, steps, graph=True)
    assert torch.equal(outs, again)
    assert torch.equal(bt.tables, bt2.tables) and torch.equal(bt.lens, bt2.lens)
    assert torch.equal(pool.k[0].view(torch.uint8), pool2.k[0].view(torch.uint8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third, *_ = _decode_loop(pkg, steps)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(outs, third)


def test_a_captured_call_follows_the_lengths(pkg):
    """One captured call over both kernels, replayed with other lengths (other splits, other
    classes of chunks, an empty sequence), on either way of making the sums."""
    lengths = [[(40, 3), (700, 60), (5, 5)], [(2000, 2), (65, 65), (1, 1)], [(0, 0), (4000, 68), (0, 0)],
               [(300, 20), (300, 20), (300, 28)]]
    for extra in (0, 40, 80):                              # 83 sequences: the sums take a launch
        hq, hkv, d = 8, 2, 128
        pad = [(0, 0)] * extra
        query, pools, tables, _, _ = _batch([(4200, 68)] * 3 + pad, hq, hkv, d, 16, torch.bfloat16, seed=31)
        query = query[:68].contiguous()
        k, v = (ref.dequantise(pools[i].view(torch.uint8), pools[i + 2]) for i in (0, 1))
        ctx, ql = _i32([40, 700, 5] + [0] * extra), _i32([3, 60, 5] + [0] * extra)
        out = torch.zeros_like(query)
        call = lambda: pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=68, out=out)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        for pairs in lengths:
            ctx.copy_(_i32([c for c, _ in pairs] + [0] * extra))
            ql.copy_(_i32([q for _, q in pairs] + [0] * extra))
            out.fill_(9.0)
            graph.replay()
            n = sum(q for _, q in pairs)
            want, mean, slip = ref.attention(query[:n], k, v, tables, ctx.tolist(), ql.tolist(), 0.1)
            tol = ref.tolerance(want, mean, slip, torch.bfloat16, d, 4200)
            assert ((out[:n].double() - want).abs() <= tol).all()
            assert (out[n:] == 9.0).all()
            eager = torch.full_like(out, 9.0)
            pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=68, out=eager)
            assert torch.equal(out, eager)


@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65])
def test_attention_at_the_counts_where_the_sums_change_hands(pkg, n):
    """One scan, two, a launch: single tokens, chunks for both kernels and empty sequences."""
    lengths = [[(300, 1), (0, 0), (70, 40), (33, 2), (1, 1), (0, 0), (129, 7)][i % 7] for i in range(n)]
    query, pools, tables, ctx, ql = _batch(lengths, 8, 2, 128, 16, torch.bfloat16, seed=60 + n)
    got = _check_attention(pkg, query, pools, tables, ctx, ql, 0.1, most=40)
    step = pkg.device_step(tables, ctx, ql, num_tokens=query.shape[0], max_query_len=40, num_blocks=pools[0].shape[0],
                           block_size=16, group=4)
    own = pkg.paged_attention_kv8(query, *pools, pkg.attach_step(tables.view_as(tables), step), ctx, ql, 0.1)
    assert torch.equal(got, own)


@pytest.mark.parametrize("n,at", [(40, 5), (40, 38), (64, 63)])
def test_a_bad_sequence_anywhere_empties_the_call_and_reports(pkg, n, at):
    query, pools, tables, ctx, ql = _batch([(50, 1)] * n, 8, 2, 128, 16, torch.bfloat16, seed=71)
    out = torch.full_like(query, 9.0)
    ctx[at] = 0                                            # a token of a sequence without context
    pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=1, out=out)
    assert (out == 9.0).all()
    assert pkg.read_kv8_error() == pkg._lib.PA_KV8_ERR_STEP


@pytest.mark.parametrize("n,most,hq,hkv,d", [(1, 300, 8, 2, 128), (3, 70, 4, 4, 64), (40, 33, 6, 2, 128)])
@pytest.mark.parametrize("attached", [False, True])
def test_a_captured_call_without_room_for_short_chunks_gets_some(pkg, n, most, hq, hkv, d, attached):
    """Sizes that leave the kernel for few rows out, then lengths below them: single tokens,
    empty sequences, contexts that several CTAs share, twins of one key tile."""
    assert pkg.kv8._tiling(hq // hkv, most, n, n * most).small_max == 0
    query, pools, tables, _, _ = _batch([(3000, most)] * n, hq, hkv, d, 16, torch.float16, seed=51)
    k, v = (ref.dequantise(pools[i].view(torch.uint8), pools[i + 2]) for i in (0, 1))
    ctx, ql = _i32([3000] * n), _i32([most] * n)
    out = torch.zeros_like(query)
    step = pkg.device_step(tables, ctx, ql, num_tokens=n * most, max_query_len=most, num_blocks=pools[0].shape[0],
                           block_size=16, group=hq // hkv)

    def call():
        if attached:
            pkg.device_step(tables, ctx, ql, num_tokens=n * most, max_query_len=most, num_blocks=pools[0].shape[0],
                            block_size=16, group=hq // hkv, out=step)
        return pkg.paged_attention_kv8(query, *pools, pkg.attach_step(tables.view_as(tables), step) if attached else tables,
                                       ctx, ql, 0.1, max_query_len=most, out=out)

    call()
    torch.cuda.synchronize()
    assert "kv8_rows" not in pkg._lib.last_launches()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    cycle = [[(3000, most)], [(1, 1), (2999, 1), (0, 0)], [(most + 40, most), (64, 2), (130, 17), (0, 0)], [(1500, most), (65, 1)]]
    for pairs in cycle:
        pairs = (pairs * n)[:n]
        ctx.copy_(_i32([c for c, _ in pairs]))
        ql.copy_(_i32([q for _, q in pairs]))
        out.fill_(9.0)
        graph.replay()
        t = sum(q for _, q in pairs)
        want, mean, slip = ref.attention(query[:t], k, v, tables, ctx.tolist(), ql.tolist(), 0.1)
        tol = ref.tolerance(want, mean, slip, torch.float16, d, 3000)
        assert ((out[:t].double() - want).abs() <= tol).all()
        assert (out[t:] == 9.0).all()


def test_calls_on_two_streams_at_once(pkg):
    a = _batch([(900, 2), (4000, 1)], 8, 2, 128, 16, torch.bfloat16, seed=41)
    b = _batch([(700, 90), (33, 33)], 8, 2, 128, 16, torch.float16, seed=42)
    run = lambda x, most: pkg.paged_attention_kv8(x[0], *x[1], *x[2:], 0.1, max_query_len=most)  # noqa: E731
    want = run(a, 2), run(b, 90)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, (x, most) in enumerate(((a, 2), (b, 90))):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(x, most))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], g) for g in got[i])


def test_pools_past_four_gigabytes(pkg):
    """Blocks whose bytes lie past 2^32 in the pool: append and both attention kernels."""
    hkv, d, bs, nb = 8, 128, 16, 290_000
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=DEV)  # noqa: E731
    payload = [zeros(nb, bs, hkv, d) for _ in range(2)]
    scale = [zeros(nb, hkv, bs) for _ in range(2)]
    pools = [payload[0].view(ref.E4M3), payload[1].view(ref.E4M3), *scale]
    tables = _i32([[nb - 1, nb - 7, 3, nb - 2], [nb - 5, nb - 4, nb - 3, 0]])
    ctx, ql = _i32([60, 40]), _i32([3, 30])
    step = pkg.device_step(tables, ctx, ctx, num_tokens=100, max_query_len=60, num_blocks=nb, block_size=bs, group=2)
    kv = torch.randn(100, 2 * hkv, d, device=DEV).bfloat16()
    pkg.reshape_and_cache_kv8(kv[:, :hkv], kv[:, hkv:], *pools, step.slot_mapping)
    used = tables.flatten().long()
    local = _i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    k, v = (ref.dequantise(payload[i][used], scale[i][used]) for i in (0, 1))
    codes, byte = ref.quantise(kv[:, :hkv].double().cpu().numpy())
    assert np.array_equal(k.view(2, 64, hkv, d)[0, :60].cpu().numpy(),
                          ref.e4m3_table()[codes[:60]] * 2.0 ** (byte[:60].astype(int) - 127)[..., None])
    query = torch.randn(33, 2 * hkv, d, device=DEV).bfloat16()
    got = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.09, max_query_len=30)
    want, mean, slip = ref.attention(query, k, v, local, [60, 40], [3, 30], 0.09)
    assert ((got.double() - want).abs() <= ref.tolerance(want, mean, slip, torch.bfloat16, d, 60)).all()
    assert {"kv8_rows", "kv8_tiles"} <= pkg._lib.last_launches()


def test_the_most_rows_and_request_slots(pkg):
    """4,096 rows over 131,072 slots, one token each; every eighth slot needs a block."""
    r, b, w, bs = 131072, 4096, 2, 16
    nb = 2 * r
    bt = pkg.DeviceBlockTables(r, w, nb, bs, DEV)
    ids = torch.randperm(r, generator=torch.Generator().manual_seed(0))[:b].to(DEV)
    bt.lens[ids[::8]] = 16
    bt.held[ids] = 1
    step = bt.reserve(ids, torch.ones(b, dtype=torch.int32, device=DEV), num_tokens=b, max_query_len=1)
    assert int(step.num_free) == nb - b // 8
    assert torch.equal(step.cu_query_lens, torch.arange(b + 1, dtype=torch.int32, device=DEV))
    assert torch.equal(step.q_pos, bt.lens[ids])
    new = step.block_tables[::8, 1]
    assert torch.equal(new, torch.arange(b // 8, dtype=torch.int32, device=DEV))   # from the list's end, in row order
    assert torch.equal(step.slot_mapping[::8], new * bs)
    with pytest.raises(NotImplementedError, match="at most 4096"):
        more = torch.arange(b + 1, device=DEV)
        bt.reserve(more, torch.ones_like(more), num_tokens=b + 1, max_query_len=1)


def test_a_step_counts_once(pkg):
    bt = pkg.DeviceBlockTables(4, 4, 20, 16, DEV)
    step = bt.reserve(_i32([0]), _i32([3]), num_tokens=3, max_query_len=3)
    bt.commit(step)
    with pytest.raises(ValueError, match="committed before"):
        bt.commit(step)
    bt.commit(bt.reserve(_i32([0]), _i32([3]), num_tokens=3, max_query_len=3, out=step))
    assert int(bt.lens[0]) == 6


def test_an_attached_step_of_other_sizes_is_refused(pkg):
    query, pools, tables, ctx, ql = _batch([(40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=43)
    step = pkg.device_step(tables, ctx, ql, num_tokens=3, max_query_len=3, num_blocks=pools[0].shape[0], block_size=16,
                           group=2)
    with pytest.raises(ValueError, match="attached step"):
        pkg.paged_attention_kv8(query, *pools, pkg.kv8.attach_step(tables, step), ctx, ql, 0.1)


def test_empty_calls(pkg):
    query, pools, tables, ctx, ql = _batch([(40, 3)], 8, 2, 128, 16, torch.bfloat16, seed=44)
    assert pkg.paged_attention_kv8(query[:0], *pools, tables[:0], ctx[:0], ql[:0], 0.1).shape == (0, 8, 128)
    out = torch.full_like(query, 2.0)
    pkg.paged_attention_kv8(query, *pools, tables[:0], ctx[:0], ql[:0], 0.1, out=out)
    assert (out == 2.0).all()
    step = pkg.device_step(tables[:0], ctx[:0], ql[:0], num_tokens=2, max_query_len=1, num_blocks=3, block_size=16)
    assert step.slot_mapping.tolist() == [-1, -1] and step.cu_query_lens.tolist() == [0]
    bt = pkg.DeviceBlockTables(4, 4, 20, 16, DEV)
    step = bt.reserve(_i32([]), _i32([]), num_tokens=0, max_query_len=1)
    bt.commit(step)
    bt.release(_i32([]))
    assert int(bt.num_free) == 20


@pytest.fixture(scope="module")
def small_llama():
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=512, intermediate_size=512, num_attention_heads=8, num_key_value_heads=2,
                      head_dim=64, num_hidden_layers=2, vocab_size=1024, max_position_embeddings=2048)
    return LlamaForCausalLM(cfg).to(DEV, torch.bfloat16).eval()


def test_the_executor_over_an_8_bit_pool(pkg, small_llama):
    """The executor's passes (mixed prefill and decode, then decode) over the 8-bit cache: layer
    0's K/V depend on the embeddings only, so its cache is the quantised form of what the
    16-bit pool holds; captured decode passes give the eager ones' tokens and cache."""
    import importlib

    from _engine import generate

    mod = importlib.import_module(f"{pkg.__name__}.executor")
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 1024, size=n).tolist() for n in (40, 7, 130, 16)]
    nb, steps, join = 64, 12, {3: [3]}
    wide = pkg.KVPool.from_model(small_llama, num_blocks=nb)
    generate(mod.CudaPagedExecutor(small_llama, None, wide), prompts, 1, nb)
    pools = [pkg.KV8Pool.from_model(small_llama, num_blocks=nb) for _ in range(2)]
    generate(mod.CudaPagedExecutor(small_llama, None, pools[0]), prompts, 1, nb)
    for x, payload, scale in ((wide.k[0], pools[0].k[0], pools[0].k_scale[0]),
                              (wide.v[0], pools[0].v[0], pools[0].v_scale[0])):
        codes, byte = ref.quantise(x.double().cpu().numpy())
        written = byte[..., 0] != 113                      # the smallest scale: a row of zeros, never written
        assert written.sum() == sum(len(p) for p in prompts)
        np.testing.assert_array_equal(payload.view(torch.uint8).cpu().numpy(), codes)
        np.testing.assert_array_equal(scale.transpose(1, 2).cpu().numpy()[written], byte[written])
    pools = [pkg.KV8Pool.from_model(small_llama, num_blocks=nb) for _ in range(2)]
    eager = generate(mod.CudaPagedExecutor(small_llama, None, pools[0]), prompts, steps, nb, join_at=join)
    graph = generate(mod.CudaPagedExecutor(small_llama, None, pools[1], decode_graphs=True), prompts, steps, nb,
                     join_at=join)
    assert [len(t) for t in eager] == [len(t) for t in graph] and eager == graph
    assert "kv8_rows" in pkg._lib.last_launches()


def test_the_executor_refuses_a_float32_model(pkg, small_llama):
    import copy
    import importlib

    mod = importlib.import_module(f"{pkg.__name__}.executor")
    with pytest.raises(NotImplementedError, match="float32"):
        mod.CudaPagedExecutor(copy.deepcopy(small_llama).float(), None, pkg.KV8Pool.from_model(small_llama, 4))


def test_pool_block_moves(pkg):
    pool = pkg.KV8Pool(3, 12, 16, 2, 64, DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    every = [t.view(torch.uint8) for t in pool.k + pool.v + pool.k_scale + pool.v_scale]
    for t in every:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8, device=DEV))
    before = [t.clone() for t in every]
    host = pool.swap_out([4, 1, 7])
    assert len(host) == 3 and torch.equal(host.k[2].view(-1), before[2][[4, 1, 7]].cpu().view(-1))
    pool.copy_blocks([(2, 0), (3, 11)])
    pool.swap_in(host, [9, 8, 5])
    torch.cuda.synchronize()
    for t, b in zip(every, before):
        b[[0, 11]] = b[[2, 3]].clone()
        b[[9, 8, 5]] = b[[4, 1, 7]].clone()
        assert torch.equal(t, b)
    assert pool.read_error() == 0
    with pytest.raises(ValueError, match="swap_in"):
        pool.swap_in(host, [1])
