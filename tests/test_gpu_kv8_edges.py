"""The 8-bit paged cache where it can go wrong: weights far below the maximum, steps that went
stale, ids that the GPU has to refuse, views at odd offsets (tests/_kv8_ref.py has the plain
64-bit forms)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import _kv8_ref as ref
from test_gpu_kv8 import DEV, _batch, _i32, _no_device_error  # noqa: F401  (the fixture reads the error word)

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


ROWS, TILES = 2.0 ** -40, 2.0 ** -32     # of the largest weight: half of fp16's least step under the kernels' shifts


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
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (8, 1, 64), (6, 3, 128)])
@pytest.mark.parametrize("drop,v_bytes", [(9.0, (113,)), (13.0, (113,)), (13.0, (113, 114, 120)), (18.0, (119,)),
                                          (18.0, (134,)), (13.0, (113, 134))])
def test_few_rows_keep_small_weights_of_any_value_scale(pkg, dtype, hq, hkv, d, drop, v_bytes):
    """Weights carry 11 bits down to 2^-29 of the maximum, whatever the V rows' scales are; one
    token, and chunks that take two and three groups of rows (with eight heads a chunk of four
    has 32 rows, which the tiles take)."""
    for lengths, most in (([(2000, 1), (300, 1)], 1), ([(1500, 3), (700, 2), (64, 4)], 4)):
        batch = _peaked(lengths, hq, hkv, d, dtype, 32, drop, v_bytes, seed=d + hq)
        tiles = most * hq // hkv > 24
        _check_tight(pkg, *batch, 1.0, most, TILES if tiles else ROWS)
        assert ("kv8_tiles" in pkg._lib.last_launches()) == tiles


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("lengths", [[(700, 300)], [(2000, 60), (130, 30)]])
def test_long_chunks_keep_small_weights(pkg, dtype, hq, hkv, d, lengths):
    """Weights of e^-15 of the maximum, which was five steps of fp16's least number."""
    batch = _peaked(lengths, hq, hkv, d, dtype, 64, 15.0, (113, 120), seed=d)
    _check_tight(pkg, *batch, 1.0, max(q for _, q in lengths), TILES)
    assert "kv8_tiles" in pkg._lib.last_launches()


def test_few_rows_of_one_cta_over_a_long_context(pkg):
    """As many KV heads as there are CTAs, so that each walks a whole context."""
    hq = hkv = 446
    batch = _peaked([(6000, 1)], hq, hkv, 64, torch.bfloat16, 2048, 13.0, (113,), seed=3)
    _check_tight(pkg, *batch, 1.0, 1, ROWS)


def test_few_rows_nan_value_rows_among_small_weights(pkg):
    """A V row that stands for NaN reaches every token that sees it, even where its weight has
    vanished, and no other token or head."""
    for hq, hkv, d in ((8, 2, 128), (4, 4, 64)):
        query, pools, tables, ctx, ql = _peaked([(90, 4), (40, 2)], hq, hkv, d, torch.bfloat16, 32, 120.0, (113,), seed=6)
        clean = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 1.0, max_query_len=4)
        slot = int(tables[0, 88 // 16]) * 16 + 88 % 16         # seen by the tokens at 88 and 89
        pools[1].view(torch.uint8).view(-1, hkv, d)[slot, 1] = 0
        pools[3][slot // 16, 1, slot % 16] = 255
        got = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 1.0, max_query_len=4)
        g = hq // hkv
        assert got[2:4, g:2 * g].isnan().all()
        got[2:4, g:2 * g] = clean[2:4, g:2 * g]
        assert torch.equal(got, clean)


# ------------------------------------------------------------------ steps that went stale
def _tables(pkg, lens=(20, 5, 40, 0), nb=24, width=6, bs=16):
    """Four slots with some tokens in them, 24 blocks."""
    bt = pkg.DeviceBlockTables(len(lens), width, nb, bs, DEV)
    step = bt.reserve(_i32(range(len(lens))), _i32(lens), num_tokens=sum(lens), max_query_len=max(lens))
    bt.commit(step)
    return bt


def _owned(bt):
    """Every block of the pool by its holder: the slots' blocks, then the free list's."""
    held, tables = bt.held.tolist(), bt.tables.tolist()
    return [b for row, n in zip(tables, held) for b in row[:n]] + bt.free[:int(bt.num_free)].tolist()


def _state_of(bt):
    n = int(bt.num_free)
    return [bt.lens.tolist(), bt.held.tolist(), [r[:h] for r, h in zip(bt.tables.tolist(), bt.held.tolist())],
            bt.free[:n].tolist()]


def _reserve(bt, ids, ql):
    return bt.reserve(_i32(ids), _i32(ql), num_tokens=sum(ql), max_query_len=max(ql))


def test_a_step_under_released_blocks_is_not_committed_and_reports(pkg):
    """Blocks that came back after the step took its own lie over them on the list: committing
    it set the list's length back and lost them."""
    bt = _tables(pkg)
    step = _reserve(bt, [0, 1], [13, 1])                       # slot 0 needs a block
    bt.release(_i32([2]))
    before = _state_of(bt)
    bt.commit(step)
    assert _state_of(bt) == before and sorted(_owned(bt)) == list(range(24))
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP
    bt.commit(_reserve(bt, [0, 1], [13, 1]))                   # made again, it counts
    assert bt.lens.tolist() == [33, 6, 0, 0] and sorted(_owned(bt)) == list(range(24))


def test_a_step_without_new_blocks_survives_a_release(pkg):
    bt = _tables(pkg)
    step = _reserve(bt, [0, 1], [2, 1])
    bt.release(_i32([2]))
    free = int(bt.num_free)
    bt.commit(step)
    assert int(bt.num_free) == free and bt.lens.tolist() == [22, 6, 0, 0]
    assert sorted(_owned(bt)) == list(range(24))


def test_two_steps_with_the_same_free_blocks_do_not_both_count_and_reports(pkg):
    bt = _tables(pkg)
    a, b = _reserve(bt, [0], [13]), _reserve(bt, [3], [1])     # both plan with the list's last block
    assert int(a.block_tables[0, 2]) == int(b.block_tables[0, 0])
    bt.commit(a)
    before = _state_of(bt)
    bt.commit(b)
    assert _state_of(bt) == before and sorted(_owned(bt)) == list(range(24))
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_two_steps_of_which_one_needs_no_block_both_count(pkg):
    bt = _tables(pkg)
    a, b = _reserve(bt, [0], [13]), _reserve(bt, [1], [1])
    bt.commit(a)
    bt.commit(b)
    assert bt.lens.tolist() == [33, 6, 40, 0] and sorted(_owned(bt)) == list(range(24))


@pytest.mark.parametrize("ids,ql", [([2], [1]), ([2], [9]), ([0, 2], [13, 3])])
def test_a_step_of_a_released_slot_is_not_committed_and_reports(pkg, ids, ql):
    bt = _tables(pkg)
    step = _reserve(bt, ids, ql)
    bt.release(_i32([2]))
    before = _state_of(bt)
    bt.commit(step)
    assert _state_of(bt) == before and sorted(_owned(bt)) == list(range(24))
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_a_slot_that_was_filled_again_elsewhere_is_not_committed_and_reports(pkg):
    """The same slot with the same length, in other blocks: the step's K and V went into the old ones."""
    bt = _tables(pkg)
    step = _reserve(bt, [2], [1])
    bt.release(_i32([2]))
    bt.commit(_reserve(bt, [3, 2], [3, 40]))
    before = _state_of(bt)
    bt.commit(step)
    assert _state_of(bt) == before and sorted(_owned(bt)) == list(range(24))
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_a_slot_that_was_filled_again_up_to_a_block_is_not_committed_and_reports(pkg):
    """The step's token starts a block of its own, so only the block before it tells."""
    bt = _tables(pkg, lens=(20, 5, 32, 0))
    step = _reserve(bt, [0, 2], [1, 1])
    want = int(step.block_tables[1, 2])
    bt.release(_i32([2]))
    bt.commit(_reserve(bt, [3], [1]))
    bt.commit(_reserve(bt, [2], [32]))
    bt.free[int(bt.num_free) - 1] = want                       # as if it had come back on top of the list
    before = _state_of(bt)
    bt.commit(step)
    assert _state_of(bt) == before
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_a_dropped_step_leaves_no_trace_in_one_that_counts(pkg):
    """The dropped one planned the same free blocks for other rows and wrote them into the tables."""
    bt = _tables(pkg)
    a = _reserve(bt, [0, 3], [30, 20])
    want = a.block_tables.tolist()
    _reserve(bt, [3, 0], [20, 30])
    bt.commit(a)
    assert [bt.tables[0].tolist()[:4], bt.tables[3].tolist()[:2]] == [want[0][:4], want[1][:2]]
    assert sorted(_owned(bt)) == list(range(24))


def test_a_step_of_other_tables_is_refused(pkg):
    bt, other = _tables(pkg), _tables(pkg)
    with pytest.raises(ValueError, match="other tables"):
        other.commit(_reserve(bt, [0], [1]))


def test_a_step_of_many_rows_counts(pkg):
    """More rows than a CTA has threads, some of them padding, several new blocks a row."""
    rows, bs, width = 1300, 16, 9
    rng = np.random.default_rng(2)
    bt = pkg.DeviceBlockTables(rows, width, rows * width, bs, DEV)
    ids = rng.permutation(rows).astype(np.int32)
    ids[::7] = -1
    lens = np.zeros(rows, int)
    for most in (50, 3, 70):
        ql = rng.integers(0, most + 1, size=rows)
        step = bt.reserve(_i32(ids), _i32(ql), num_tokens=int(ql.sum()), max_query_len=most)
        want = step.block_tables.tolist()
        bt.commit(step)
        live = ids >= 0
        lens[ids[live]] += ql[live]
        np.testing.assert_array_equal(bt.lens.cpu().numpy(), lens)
        np.testing.assert_array_equal(bt.held.cpu().numpy()[ids[live]], -(-lens[ids[live]] // bs))
        tables, held = bt.tables.tolist(), bt.held.tolist()
        assert all(tables[r][:held[r]] == want[i][:held[r]] for i, r in enumerate(ids) if r >= 0)
        assert sorted(_owned(bt)) == list(range(rows * width))


def test_a_captured_commit_counts_its_step_once_and_reports(pkg):
    """Replayed without the reserve before it, a commit meets lengths that have moved on."""
    bt = _tables(pkg)
    step = _reserve(bt, [0, 1], [2, 1])
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        bt.commit(step)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert bt.lens.tolist() == [22, 6, 40, 0]
    graph.replay()
    assert bt.lens.tolist() == [22, 6, 40, 0]
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_request_ids_may_be_filled_anew_before_the_commit(pkg):
    """The step keeps its rows' slots: the caller's tensor is the next step's by then."""
    bt = _tables(pkg)
    ids = _i32([0, 1])
    step = bt.reserve(ids, _i32([13, 1]), num_tokens=14, max_query_len=13)
    ids.copy_(_i32([1, 2]))
    bt.commit(step)
    assert bt.lens.tolist() == [33, 6, 40, 0] and bt.held.tolist() == [3, 1, 3, 0]
    assert sorted(_owned(bt)) == list(range(24))


@pytest.mark.parametrize("bad", [24, -1, 1 << 30])
@pytest.mark.parametrize("where", ["list", "held", "row of many"])
def test_a_step_whose_new_tokens_have_a_bad_block_is_emptied_and_reports(pkg, where, bad):
    """A block id outside the pool, new or held before: no token of the step counts and the id
    does not reach the slots' tables."""
    bt = _tables(pkg)
    ids, ql = [0, 1, 3], [13, 1, 2]                            # slots 0 and 3 need a block, slot 1 has room
    if where == "list":
        bt.free[int(bt.num_free) - 2] = bad                    # slot 3's
    elif where == "held":
        bt.tables[1, 0] = bad
    else:                                                      # a chunk over blocks that were held for it
        bt.held[2] = 5
        bt.tables[2, 3:5] = _i32([7, bad])
        ids, ql = [1, 2], [1, 33]
    before = _state_of(bt)
    step = _reserve(bt, ids, ql)
    assert int(step.num_free) == -1 and not step.context_lens.any() and not step.block_tables.any()
    assert (step.slot_mapping == -1).all()
    bt.commit(step)
    assert _state_of(bt) == before
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_BLOCK


@pytest.mark.parametrize("rows", [2380, 2400, 2430, 2440, 2460, 4070, 4085, 4095])
def test_reserve_and_commit_of_any_row_count(pkg, rows):
    """Among them the counts whose sums fill the shared memory that a launch has without asking."""
    bt = pkg.DeviceBlockTables(rows, 2, 2 * rows, 16, DEV)
    ids = torch.arange(rows, dtype=torch.int32, device=DEV)
    step = bt.reserve(ids, torch.ones_like(ids), num_tokens=rows, max_query_len=1)
    assert torch.equal(step.slot_mapping, 16 * ids)
    bt.commit(step)
    assert bool((bt.lens == 1).all()) and int(bt.num_free) == rows
    bt.release(ids)
    assert int(bt.num_free) == 2 * rows


def test_reserve_on_two_host_threads(pkg):
    """Steps of different sizes, whose shared memory has to be asked for, side by side."""
    import threading

    failed = []

    def work(rows):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                bt = pkg.DeviceBlockTables(rows, 2, rows, 16, DEV)
                ids = torch.arange(rows, dtype=torch.int32, device=DEV)
                one = torch.ones_like(ids)
                step = None
                for _ in range(2000):
                    step = bt.reserve(ids, one, num_tokens=rows, max_query_len=1, out=step)
                assert torch.equal(step.slot_mapping, 16 * ids)
        except BaseException as e:  # noqa: BLE001  (to the test's own thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in (4096, 2700, 3300)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


# ------------------------------------------------------------------ views, ids and sizes of any kind
@pytest.mark.parametrize("tokens", [1, 3])
def test_queries_at_odd_offsets(pkg, tokens):
    """Contiguous queries that do not start on 16 bytes, and one token whose token stride (which no
    address depends on) is odd."""
    query, pools, tables, ctx, ql = _batch([(90, tokens)], 8, 2, 128, 16, torch.bfloat16, seed=9)
    want = pkg.paged_attention_kv8(query, *pools, tables, ctx, ql, 0.1, max_query_len=tokens)
    for off in (1, 4):
        flat = torch.zeros(query.numel() + off, dtype=query.dtype, device=DEV)
        view = flat[off:].view_as(query)
        view.copy_(query)
        assert view.is_contiguous() and view.data_ptr() % 16
        assert torch.equal(want, pkg.paged_attention_kv8(view, *pools, tables, ctx, ql, 0.1, max_query_len=tokens))
    view = torch.zeros(tokens * 1027, dtype=query.dtype, device=DEV).as_strided((tokens, 8, 128), (1027, 128, 1))
    view.copy_(query)
    assert torch.equal(want, pkg.paged_attention_kv8(view, *pools, tables, ctx, ql, 0.1, max_query_len=tokens))


def test_wide_ids_are_not_wrapped_and_reports(pkg):
    """64-bit slots, ids and lengths past 32 bits are out of range, not their low halves."""
    nb, hkv, d = 4, 2, 64
    pools = [torch.zeros(nb, 16, hkv, d, dtype=torch.uint8, device=DEV).view(ref.E4M3) for _ in range(2)]
    pools += [torch.zeros(nb, hkv, 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
    rows = torch.ones(3, hkv, d, device=DEV)
    pkg.reshape_and_cache_kv8(rows, rows, *pools, torch.tensor([(1 << 32) + 5, 7, -(1 << 32) + 9], device=DEV))
    assert pools[2][0, 0].nonzero().flatten().tolist() == [7]
    bt = _tables(pkg)
    step = bt.reserve(torch.tensor([1 << 32], device=DEV), _i32([1]), num_tokens=1, max_query_len=1)
    assert int(step.num_free) == -1 and pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP
    step = pkg.device_step(_i32([[0, 1]]), torch.tensor([(1 << 32) + 3], device=DEV), _i32([1]), num_tokens=1,
                           max_query_len=1, num_blocks=4, block_size=16)
    assert step.slot_mapping.tolist() == [-1] and pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP
    step = pkg.device_step(torch.tensor([[1 << 32, 1]], device=DEV), _i32([3]), _i32([1]), num_tokens=1,
                           max_query_len=1, num_blocks=4, block_size=16)
    assert step.slot_mapping.tolist() == [-1] and pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_BLOCK


def test_a_replayed_reserve_may_be_committed_outside_the_graph_and_reports(pkg):
    """A captured step with the commit outside: the accepted counts come from somewhere else."""
    bt = _tables(pkg)
    ids, ql = _i32([0, 1]), _i32([4, 4])
    step = bt.reserve(ids, ql, num_tokens=8, max_query_len=4)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        bt.reserve(ids, ql, num_tokens=8, max_query_len=4, out=step)
    torch.cuda.current_stream().wait_stream(side)
    want = [20, 5]
    for accepted in ([1, 4], [0, 3], [4, 2]):
        graph.replay()
        bt.commit(step, _i32(accepted))
        want = [a + b for a, b in zip(want, accepted)]
        assert bt.lens.tolist()[:2] == want
    bt.commit(step)                                            # without a replay: the lengths have moved on
    assert bt.lens.tolist()[:2] == want
    assert pkg.read_kv8_error(DEV) == pkg._lib.PA_KV8_ERR_STEP


def test_the_executor_refuses_too_many_query_heads_at_once(pkg):
    import importlib
    from types import SimpleNamespace

    mod = importlib.import_module(f"{pkg.__name__}.executor")
    model = SimpleNamespace(config=SimpleNamespace(num_attention_heads=34),
                            parameters=lambda: iter([torch.zeros(1, dtype=torch.bfloat16)]))
    with pytest.raises(NotImplementedError, match="17 query heads per KV head: at most 16"):
        mod.CudaPagedExecutor(model, None, pkg.KV8Pool(1, 4, 16, 2, 64, DEV))


def test_decode_step_graphs_refuse_8_bit_pools(pkg):
    import importlib

    mod = importlib.import_module(f"{pkg.__name__}.graphs")
    pool = pkg.KV8Pool(1, 4, 16, 2, 64, DEV)
    with pytest.raises(NotImplementedError, match="float32, float16 or bfloat16"):
        mod.DecodeStepGraph(pool.k, pool.v, num_heads=4, scale=0.1, batch=1, width=2)


# ------------------------------------------------------------------ neighbours
@pytest.mark.parametrize("own", [(700, 2), (1500, 3), (517, 1), (600, 70), (130, 130), (2000, 300)])
def test_a_sequence_among_neighbours(pkg, own):
    """A sequence alone and first, between and last among others, whose keys move the cuts that fall
    into its own: each time as near to 64 bits as alone."""
    hq, hkv, d = 8, 2, 128
    around = [(90, 1), (4000, 2), (33, 33), (0, 0), (900, 64), (5, 5)]
    query, pools, tables, ctx, ql = _batch([own] + around, hq, hkv, d, 16, torch.bfloat16, seed=own[0])
    k, v = (ref.dequantise(pools[i].view(torch.uint8), pools[i + 2]) for i in (0, 1))
    starts = torch.cat([ql.new_zeros(1), ql.cumsum(0)]).tolist()
    for order in ([0], [0, 1, 2], [2, 0, 4], [1, 4, 0], [3, 2, 1, 0, 5, 4], [5, 4, 3, 2, 1, 0]):
        q = torch.cat([query[starts[i]:starts[i + 1]] for i in order])
        c, n, t = ctx[order], ql[order], tables[order]
        got = pkg.paged_attention_kv8(q, *pools, t, c, n, 0.09, max_query_len=int(n.max()))
        want, mean, slip = ref.attention(q, k, v, t, c.tolist(), n.tolist(), 0.09)
        lost = ref.lost_weight(t, c.tolist(), n.tolist(), v, hq, TILES)
        assert ((got.double() - want).abs() <= ref.tight_tolerance(want, mean, slip, lost, torch.bfloat16, d)).all(), order


def test_few_rows_keep_small_weights_over_a_long_context(pkg):
    """131,071 keys of which all but every 32nd have a weight of 2^-18.8 of the maximum and V rows
    of the smallest scale, cut over many CTAs and joined."""
    batch = _peaked([(131071, 1), (40, 1)], 8, 2, 128, torch.bfloat16, 32, 13.0, (113,), seed=5)
    _check_tight(pkg, *batch, 1.0, 1, ROWS)


def test_long_chunks_keep_small_weights_over_a_long_context(pkg):
    batch = _peaked([(60001, 40)], 8, 2, 128, torch.float16, 64, 13.0, (113, 116), seed=7)
    _check_tight(pkg, *batch, 1.0, 40, TILES)
