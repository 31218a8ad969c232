"""The 8-bit paged KV cache, driven from the GPU.

Half the bytes of a 16-bit pool per cached token, so about twice the decode rate where HBM
bounds it and twice the tokens a pool holds.  Three operators that work together:

* :class:`DeviceBlockTables` / :func:`device_step` — a step's block tables, slot map and
  work sums built on the GPU from request lengths (blocks taken from a free list there), so
  a decode loop needs no host plan;
* :func:`reshape_and_cache_kv8` — the fused K+V append, quantising each row;
* :func:`paged_attention_kv8` — causal attention of a chunk of new tokens (one and more)
  over the 8-bit pools.

Format: a row (one token of one KV head) is e4m3 payload ``[NB, BS, Hkv, D]`` and a scale
byte ``[NB, Hkv, BS]`` that stands for ``2^(byte - 127)`` (``torch.float8_e8m0fnu``): the least
exponent in [-14, 7] that brings the row's largest magnitude to 448.  Every cached value is
exactly an fp16 number; magnitudes past 57,344 saturate; rows below 448 * 2^-15 are kept in steps
of 2^-23; a row with a NaN reads as NaN.

Lengths and ids that only the GPU sees are checked there: a bad step is emptied and leaves
a bit in the device's error word, which :func:`read_kv8_error` returns.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _DTYPE_CODE
from .kv_cache import HostBlocks, _error_word, copy_blocks, gather_blocks, scatter_blocks

_PAYLOAD = torch.float8_e4m3fn


def _launch(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` with ``device`` current and its current stream."""
    index, current = device.index, torch._C._cuda_getDevice()
    if index == current:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _need_cuda(device: torch.device, what: str) -> None:
    if device.type != "cuda":
        raise NotImplementedError(f"ATTENTION=cuda: {what} needs a CUDA device, got {device}. There is no CPU fallback.")


def _int32(name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype is torch.int32 and t.device == device and t.is_contiguous():
        return t
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != torch.int32:   # what 32 bits do not hold stays out of range, not its low half
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def read_kv8_error(device=None, clear: bool = True) -> int:
    """The KV8 error word of ``device`` (0: nothing reported; else ``_lib.PA_KV8_ERR_*``
    bits).  Synchronises the current stream."""
    device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    word = ctypes.c_int32(0)
    torch.cuda.init()
    _launch(device, _lib.lib().pa_kv8_read_error, int(clear), ctypes.byref(word))
    return int(word.value)


# ---------------------------------------------------------------------------- steps
_TILINGS: dict[tuple[int, int, int, int], _lib.Kv8Tiling] = {}


def _tiling(group: int, max_query_len: int, num_seqs: int, num_tokens: int) -> _lib.Kv8Tiling:
    key = (group, max_query_len, num_seqs, num_tokens)
    t = _TILINGS.get(key)
    if t is None:
        t = _lib.Kv8Tiling()
        _lib.check(_lib.lib().pa_kv8_choose_tiling(*key, ctypes.byref(t)))
        if len(_TILINGS) > 1024:
            _TILINGS.clear()
        _TILINGS[key] = t
    return t


def check_group(group: int) -> None:
    """Refuses what the attention kernels do not take of query heads per KV head."""
    _tiling(group, 1, 1, 1)


# The step's arrays in one int32 buffer: num_free with the rest of what a commit has to know (8-byte
# words and the rows' slots among it), work (int64), context_lens, query_lens, held, cu_query_lens,
# seq_idx, q_pos, slot_mapping, block_tables.
_FREE, _WORK, _CTX, _QL, _HELD, _CU, _SEQ, _POS, _SLOT, _TABLES = range(10)


_LAYOUTS: dict[tuple[int, int, int], tuple[tuple[int, ...], tuple[int, ...], int]] = {}


def _layout(b: int, t: int, cells: int) -> tuple[tuple[int, ...], tuple[int, ...], int]:
    """(words of each array, their byte offsets, words in all); work's words have the rest of the
    commit's record before them."""
    got = _LAYOUTS.get((b, t, cells))
    if got is None:
        record = (_lib.PA_KV8_STEP_WORDS + b + 1) // 2 * 2
        sizes = (1, record - 1 + 4 * (b + 1), b, b, b, b + 1, t, t, t, cells)
        offsets = [4 * sum(sizes[:i]) for i in range(len(sizes))]
        offsets[_WORK] = 4 * record
        got = (sizes, tuple(offsets), sum(sizes))
        if len(_LAYOUTS) > 1024:
            _LAYOUTS.clear()
        _LAYOUTS[(b, t, cells)] = got
    return got


class DeviceStep:
    """One step's metadata on the GPU, shared by every layer: ``block_tables [B, W]``,
    ``context_lens`` / ``query_lens [B]``, ``cu_query_lens [B + 1]``, per token ``seq_idx``,
    ``q_pos`` and ``slot_mapping [T]`` (-1 past the step's last token), ``held [B]`` (blocks of
    each row's slot), ``num_free [1]`` (the free list's length once the step counts; -1: the
    step was emptied)."""

    def __init__(self, num_rows: int, num_tokens: int, width: int, max_query_len: int, block_size: int,
                 num_blocks: int, group: int, device: torch.device, own_tables: bool):
        self.num_seqs, self.num_tokens, self.width, self.max_query_len = num_rows, num_tokens, width, max_query_len
        self.block_size, self.num_blocks, self.group, self.device = block_size, num_blocks, group, device
        self._sizes, offsets, words = _layout(num_rows, num_tokens, num_rows * width if own_tables else 0)
        self.buffer = torch.empty(words, dtype=torch.int32, device=device)
        at = self.buffer.data_ptr()
        self._ptr = [at + o for o in offsets]
        self._views: tuple[torch.Tensor, ...] | None = None
        self._tables: torch.Tensor | None = None      # the caller's, when the step has none of its own
        self._counted = False
        self._captured = False                        # a graph's replays make it again, unseen here
        self._home = 0                                # the address of the num_free it was reserved against, if any

    @property
    def _arrays(self) -> tuple[torch.Tensor, ...]:
        if self._views is None:
            self._views = torch.unsafe_split_with_sizes(self.buffer, self._sizes)  # int32: autograd has no say
        return self._views

    work = property(lambda self: self._arrays[_WORK][-4 * (self.num_seqs + 1):].view(torch.int64)
                    .view(2, self.num_seqs + 1))
    context_lens = property(lambda self: self._arrays[_CTX])
    query_lens = property(lambda self: self._arrays[_QL])
    held = property(lambda self: self._arrays[_HELD])
    cu_query_lens = property(lambda self: self._arrays[_CU])
    seq_idx = property(lambda self: self._arrays[_SEQ])
    q_pos = property(lambda self: self._arrays[_POS])
    slot_mapping = property(lambda self: self._arrays[_SLOT])
    num_free = property(lambda self: self._arrays[_FREE])

    @property
    def block_tables(self) -> torch.Tensor:
        return self._tables if self._tables is not None else self._arrays[_TABLES].view(self.num_seqs, self.width)

    def matches(self, num_tokens: int, block_size: int, num_blocks: int, group: int) -> bool:
        """Whether this step can drive an attention call of these sizes."""
        return (self.num_tokens == num_tokens and self.block_size == block_size and self.num_blocks == num_blocks
                and self.group == group)


def _check_step_sizes(num_tokens: int, max_query_len: int, block_size: int, num_blocks: int) -> None:
    if num_tokens < 0 or max_query_len < 0:
        raise ValueError("num_tokens and max_query_len must be non-negative")
    if block_size <= 0 or num_blocks < 0:
        raise ValueError("block_size must be positive and the pool's block count non-negative")


def _table_rows(tables: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Block tables as int32 rows of any stride (a slice of a wider table stays in place)."""
    if tables.device != device:
        raise ValueError(f"block_tables is on {tables.device}, expected {device}")
    b, w = tables.shape
    if tables.dtype is torch.int32 and (w < 2 or tables.stride(1) == 1) and (b < 2 or tables.stride(0) >= w):
        return tables
    return _int32("block_tables", tables, device)


def _reusable(out: DeviceStep | None, like: tuple, device) -> DeviceStep | None:
    if out is None:
        return None
    have = (out.num_seqs, out.num_tokens, out.width, out.max_query_len, out.block_size, out.num_blocks, out.group)
    if have != like or out.device != device:
        raise ValueError(f"out was made for a step of other sizes: {have}, this one needs {like}")
    return out


def device_step(block_tables: torch.Tensor, context_lens: torch.Tensor, query_lens: torch.Tensor, *, num_tokens: int,
                max_query_len: int, num_blocks: int, block_size: int, group: int = 1,
                out: DeviceStep | None = None) -> DeviceStep:
    """Prefix sums, per-token positions and the slot map of a step whose block tables are
    already on the GPU (``block_tables [B, W]``, ``context_lens [B]`` with this step's tokens,
    ``query_lens [B]``), in one launch and without the host reading a length.  ``num_tokens``
    is the packed token count (tokens past ``sum(query_lens)`` get -1), ``max_query_len`` a
    bound on the chunks, ``group`` the query heads per KV head of the attention that will use
    the step.  ``out``: a step of the same sizes whose buffers are written again (for captured
    graphs)."""
    dev = block_tables.device
    _need_cuda(dev, "device_step")
    _check_step_sizes(num_tokens, max_query_len, block_size, num_blocks)
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [batch, max_blocks]")
    b, w = block_tables.shape
    if tuple(context_lens.shape) != (b,) or tuple(query_lens.shape) != (b,):
        raise ValueError("context_lens and query_lens must be [batch] to match block_tables")
    tables = _table_rows(block_tables, dev)
    ctx, ql = _int32("context_lens", context_lens, dev), _int32("query_lens", query_lens, dev)
    tiling = _tiling(group, max_query_len, b, num_tokens)
    step = _reusable(out, (b, num_tokens, w, max_query_len, block_size, num_blocks, group), dev)
    if step is None:
        step = DeviceStep(b, num_tokens, w, max_query_len, block_size, num_blocks, group, dev, own_tables=False)
    elif step._sizes[_TABLES]:
        raise ValueError("out was made by DeviceBlockTables.reserve")
    step._tables = tables
    p = step._ptr
    _launch(dev, _lib.lib().pa_kv8_build_step, None, ctx.data_ptr(), ql.data_ptr(), tables.data_ptr(),
            max(tables.stride(0), w), None, None, None, 0, b, b, w, block_size, num_blocks, num_tokens, max_query_len,
            ctypes.byref(tiling), None, p[_CTX], p[_QL], p[_HELD], p[_CU], p[_SEQ], p[_POS], p[_SLOT], p[_FREE], p[_WORK])
    return step


def step_of_metadata(meta, group: int) -> DeviceStep:
    """The step of host-planned metadata (:class:`~.metadata.StepMetadata`, uploaded): its
    tables and lengths are read where they lie."""
    plan, buf = meta.plan, meta.device_buffer
    n = plan.num_seqs
    return device_step(meta.block_tables(), buf[plan.off_context_lens:plan.off_context_lens + n],
                       buf[plan.off_query_lens:plan.off_query_lens + n], num_tokens=plan.num_tokens,
                       max_query_len=max(1, plan.max_query_len), num_blocks=meta.pool_num_blocks,
                       block_size=plan.block_size, group=group)


class DeviceBlockTables:
    """Block tables that live and grow on the GPU: per request slot a row of block ids, the
    tokens cached and the blocks held, and one free list for the pool.

    A step is ``reserve`` (blocks for the new tokens, the step's metadata), then the layers,
    then ``commit`` — with the accepted counts, where a chunk of speculated tokens was only
    partly accepted.  Until ``commit``, a step can be reserved again or dropped; one that no
    longer fits when it is committed (its slots moved on, its blocks went to another step, blocks
    were released after it took its own) changes nothing and leaves an error bit.  ``release``
    returns a finished request's blocks.  Nothing here reads the GPU from the host, so the
    whole loop can be captured in a CUDA graph.  Prefix sharing stays with the host allocator:
    a block is held by one slot."""

    def __init__(self, max_requests: int, width: int, num_blocks: int, block_size: int, device) -> None:
        device = torch.device(device)
        _need_cuda(device, "DeviceBlockTables")
        if max_requests <= 0 or width <= 0 or num_blocks < 0 or block_size <= 0:
            raise ValueError("max_requests, width and block_size must be positive, num_blocks non-negative")
        zeros = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
        # Taken from the end of the list: block 0 first.
        free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self._set(zeros(max_requests, width), zeros(max_requests), zeros(max_requests), free,
                  torch.full((1,), num_blocks, dtype=torch.int32, device=device), num_blocks, block_size)

    @classmethod
    def adopt(cls, tables: torch.Tensor, lens: torch.Tensor, held: torch.Tensor, free: torch.Tensor,
              num_free: torch.Tensor, *, num_blocks: int, block_size: int) -> "DeviceBlockTables":
        """Over tensors the caller already keeps (all int32, contiguous, on one GPU): ``tables
        [R, W]``, ``lens [R]``, ``held [R]``, ``free`` with its first ``num_free [1]`` entries
        valid.  They are updated in place."""
        dev, i32 = tables.device, torch.int32
        if not (tables.dtype is i32 and lens.dtype is i32 and held.dtype is i32 and free.dtype is i32
                and num_free.dtype is i32 and dev == lens.device and dev == held.device and dev == free.device
                and dev == num_free.device and tables.is_contiguous() and lens.is_contiguous()
                and held.is_contiguous() and free.is_contiguous()):
            _need_cuda(dev, "DeviceBlockTables")
            for name, t in (("tables", tables), ("lens", lens), ("held", held), ("free", free), ("num_free", num_free)):
                if t.dtype != i32 or t.device != dev or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous int32 on {dev}")
        shape = tables.shape
        if len(shape) != 2 or lens.shape != shape[:1] or held.shape != shape[:1]:
            raise ValueError("tables must be [requests, width], lens and held [requests]")
        if free.dim() != 1 or num_free.numel() != 1:
            raise ValueError("free must be [capacity] and num_free [1]")
        _need_cuda(dev, "DeviceBlockTables")
        self = cls.__new__(cls)
        self._set(tables, lens, held, free, num_free, num_blocks, block_size)
        return self

    def _set(self, tables, lens, held, free, num_free, num_blocks, block_size) -> None:
        _check_step_sizes(0, 0, block_size, num_blocks)
        self.tables, self.lens, self.held, self.free, self.num_free = tables, lens, held, free, num_free
        self.num_blocks, self.block_size, self.device = int(num_blocks), int(block_size), tables.device
        self.max_requests, self.width = tables.shape

    def reserve(self, request_ids: torch.Tensor, query_lens: torch.Tensor, *, num_tokens: int, max_query_len: int,
                group: int = 1, out: DeviceStep | None = None) -> DeviceStep:
        """The step that appends ``query_lens[i]`` tokens to request slot ``request_ids[i]``
        (-1: a padding row; a slot at most once), in one launch.  A slot that needs more blocks
        than it holds takes them from the free list, rows in order.  When the list is too short,
        a new token's block is outside the pool or the arguments do not fit together, the step
        is emptied (``num_free`` -1, an error bit) and no table changes."""
        dev = self.device
        _check_step_sizes(num_tokens, max_query_len, self.block_size, self.num_blocks)
        if request_ids.dim() != 1 or query_lens.shape != request_ids.shape:
            raise ValueError("request_ids and query_lens must both be [rows]")
        ids, ql = _int32("request_ids", request_ids, dev), _int32("query_lens", query_lens, dev)
        b = ids.shape[0]
        tiling = _tiling(group, max_query_len, b, num_tokens)
        step = _reusable(out, (b, num_tokens, self.width, max_query_len, self.block_size, self.num_blocks, group), dev)
        if step is None:
            step = DeviceStep(b, num_tokens, self.width, max_query_len, self.block_size, self.num_blocks, group, dev,
                              own_tables=True)
        elif step._tables is not None:
            raise ValueError("out was made by device_step")
        home = self.num_free.data_ptr()
        step._counted, step._home = False, home
        step._captured |= torch._C._cuda_isCurrentStreamCapturing()
        p = step._ptr
        _launch(dev, _lib.lib().pa_kv8_build_step, ids.data_ptr(), self.lens.data_ptr(), ql.data_ptr(),
                self.tables.data_ptr(), self.width, self.held.data_ptr(), self.free.data_ptr(),
                home, self.free.shape[0], b, self.max_requests, self.width, self.block_size,
                self.num_blocks, num_tokens, max_query_len, ctypes.byref(tiling), p[_TABLES], p[_CTX], p[_QL], p[_HELD],
                p[_CU], p[_SEQ], p[_POS], p[_SLOT], p[_FREE], p[_WORK])
        return step

    def commit(self, step: DeviceStep, accepted: torch.Tensor | None = None) -> None:
        """Make a reserved step count: its tokens (or the ``accepted[i]`` first of row i) are
        cached now and its blocks are held.  An emptied step changes nothing; nor does one that
        no longer fits the slots and the free list, which :func:`read_kv8_error` reports.  A
        step counts once (one whose ``reserve`` was captured, once a replay)."""
        if not step._home:
            raise ValueError("commit needs a step made by reserve")
        if step._home != self.num_free.data_ptr():
            raise ValueError("this step was reserved in other tables")
        if step._counted and not step._captured:
            raise ValueError("this step was committed before")
        acc = None
        if accepted is not None:
            if tuple(accepted.shape) != (step.num_seqs,):
                raise ValueError(f"accepted must be [{step.num_seqs}], got {tuple(accepted.shape)}")
            acc = _int32("accepted", accepted, self.device)
        p = step._ptr
        _launch(self.device, _lib.lib().pa_kv8_commit, None, p[_QL],
                acc.data_ptr() if acc is not None else None, p[_HELD], p[_FREE], step.num_seqs, self.max_requests,
                self.lens.data_ptr(), self.held.data_ptr(), self.num_free.data_ptr())
        step._counted = True

    def release(self, request_ids: torch.Tensor) -> None:
        """Return the blocks of these request slots (-1 is passed over; a slot at most once) to
        the free list and empty the slots."""
        if request_ids.dim() != 1:
            raise ValueError("request_ids must be [count]")
        ids = _int32("request_ids", request_ids, self.device)
        _launch(self.device, _lib.lib().pa_kv8_release, ids.data_ptr(), ids.shape[0], self.tables.data_ptr(), self.width,
                self.width, self.max_requests, self.lens.data_ptr(), self.held.data_ptr(), self.free.data_ptr(),
                self.free.shape[0], self.num_free.data_ptr())


# ---------------------------------------------------------------------------- the pools
def _check_pools(k_pool, v_pool, k_scale, v_scale, device) -> tuple[int, int, int, int]:
    if k_pool.dim() != 4 or k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool must both be [blocks, block_size, kv_heads, dim]")
    nb, bs, hkv, dim = k_pool.shape
    side = (nb, hkv, bs)
    if (k_pool.dtype is _PAYLOAD and v_pool.dtype is _PAYLOAD and k_scale.dtype is torch.uint8
            and v_scale.dtype is torch.uint8 and k_scale.shape == side and v_scale.shape == side
            and k_pool.device == device and v_pool.device == device and k_scale.device == device
            and v_scale.device == device and k_pool.is_contiguous() and v_pool.is_contiguous()
            and k_scale.is_contiguous() and v_scale.is_contiguous()):
        return nb, bs, hkv, dim
    for name, t, shape in (("k_pool", k_pool, k_pool.shape), ("v_pool", v_pool, k_pool.shape),
                           ("k_scale", k_scale, (nb, hkv, bs)), ("v_scale", v_scale, (nb, hkv, bs))):
        want = _PAYLOAD if name.endswith("pool") else torch.uint8
        if t.dtype != want:
            raise ValueError(f"{name} must be {want}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")
        if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {tuple(shape)}, got {tuple(t.shape)}")
    return nb, bs, hkv, dim


def reshape_and_cache_kv8(key: torch.Tensor, value: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                          k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantise ``key``/``value`` ``[T, Hkv, D]`` (float32, float16 or bfloat16; D 64 or 128;
    any token and head strides) and write them into the 8-bit pools at flat slots
    ``slot_mapping [T]``; one launch for K and V.  Slots outside the pool (the -1 of padding
    tokens) are passed over; a slot named twice must get the same row."""
    dev = key.device
    _need_cuda(dev, "the 8-bit KV append")
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError(f"key/value must both be [tokens, kv_heads, dim], got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")
    nb, bs, hkv, dim = _check_pools(k_pool, v_pool, k_scale, v_scale, dev)
    if key.shape[1:] != (hkv, dim):
        raise ValueError(f"key rows {tuple(key.shape[1:])} do not match the pool's {(hkv, dim)}")
    if value.dtype != key.dtype or value.device != dev:
        raise ValueError("key and value must share dtype and device")
    if key.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"ATTENTION=cuda: dtype {key.dtype} is not float32, float16 or bfloat16")
    if key.stride(2) != 1 or value.stride(2) != 1:
        key, value = key.contiguous(), value.contiguous()
    if slot_mapping.shape != (key.shape[0],):
        raise ValueError(f"slot_mapping must be [{key.shape[0]}], got {tuple(slot_mapping.shape)}")
    slots = _int32("slot_mapping", slot_mapping, dev)
    ks, vs = key.stride(), value.stride()
    _launch(dev, _lib.lib().pa_kv8_append, key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], key.shape[0],
            hkv, dim, _DTYPE_CODE[key.dtype], k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), nb, bs, slots.data_ptr())


def attach_step(block_tables: torch.Tensor, step: DeviceStep) -> torch.Tensor:
    """Let a step ride on its block-table tensor (as ``metadata.attach`` does for host plans),
    so that every layer's :func:`paged_attention_kv8` uses it instead of building its own."""
    block_tables._kv8_step = step
    return block_tables


_SCRATCH_BYTES: dict[tuple[int, ...], int] = {}


def _scratch(device: torch.device, *sizes: int) -> torch.Tensor:
    """Scratch of one call, from the caching allocator: calls on two streams and captured
    graphs each have their own."""
    n = _SCRATCH_BYTES.get(sizes)
    if n is None:
        n = int(_lib.lib().pa_kv8_workspace_bytes(*sizes))
        if len(_SCRATCH_BYTES) > 1024:
            _SCRATCH_BYTES.clear()
        _SCRATCH_BYTES[sizes] = n
    return torch.empty(max(n, 1), dtype=torch.uint8, device=device)


def paged_attention_kv8(query: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                        query_lens: torch.Tensor, scale: float, *, max_query_len: int | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal paged attention over the 8-bit pools: :func:`paged_attention_cuda`'s arguments
    and rule with the pools' scales.  Lengths and tables are device tensors that the host never
    reads; ``max_query_len`` bounds the chunks (default: the token count).  Sums the step up by
    itself (past 64 sequences in a launch of its own) unless ``block_tables`` carries one
    (:func:`attach_step`).  Sums are float32; softmax weights are rounded to fp16 for the product
    with V (11 bits; of a key far below the maximum at most 2^-32 of the largest weight is lost).

    query ``[T, Hq, D]``, float16 or bfloat16, any strides and offset (rows that are not 16-byte
    aligned are copied first), D 64 or 128, at most 16 query heads per KV head; ``out``
    contiguous and 16-byte aligned; pools' block size a power of two times 16.  Rows past the
    last sequence's are left as they were in ``out`` (undefined without ``out``)."""
    if query.dim() != 3:
        raise ValueError(f"query must be [num_tokens, heads, dim], got {tuple(query.shape)}")
    dev = query.device
    _need_cuda(dev, "attention over the 8-bit pools")
    nb, bs, hkv, dim = _check_pools(k_pool, v_pool, k_scale, v_scale, dev)
    tokens, heads, qdim = query.shape
    if qdim != dim:
        raise ValueError(f"query head_dim {qdim} != pool head_dim {dim}")
    if heads == 0 or hkv == 0 or heads % hkv:
        raise ValueError(f"{heads} query heads not divisible by {hkv} kv heads")
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"ATTENTION=cuda: the 8-bit cache takes float16 and bfloat16 queries, not {query.dtype}")
    if out is None:
        out = (torch.empty_like(query) if query.is_contiguous() else
               torch.empty((tokens, heads, dim), dtype=query.dtype, device=dev))
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous with the query's shape, dtype and device")
    group = heads // hkv
    step = getattr(block_tables, "_kv8_step", None)
    if step is not None:
        if step.device != dev or not step.matches(tokens, bs, nb, group):
            raise ValueError(f"the attached step is for {step.num_tokens} tokens, {step.group} heads per KV head and "
                             f"{step.num_blocks} blocks of {step.block_size} on {step.device}; the call has {tokens}, "
                             f"{group}, {nb} of {bs} on {dev}")
        tables, p = step.block_tables, step._ptr
        b, w, most = step.num_seqs, step.width, step.max_query_len
        ctx, lens, cu, work = p[_CTX], None, p[_CU], p[_WORK]
    else:
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be [batch, max_blocks]")
        b, w = block_tables.shape
        if tuple(context_lens.shape) != (b,) or tuple(query_lens.shape) != (b,):
            raise ValueError("context_lens and query_lens must be [batch] to match block_tables")
        tables = _table_rows(block_tables, dev)
        context_lens, query_lens = _int32("context_lens", context_lens, dev), _int32("query_lens", query_lens, dev)
        most = tokens if max_query_len is None else min(int(max_query_len), tokens)
        _check_step_sizes(tokens, most, bs, nb)
        ctx, lens, cu, work = context_lens.data_ptr(), query_lens.data_ptr(), None, None
    _tiling(group, most, b, tokens)                   # refuses what has no kernel, also for empty calls
    if tokens == 0:
        return out
    qs = query.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)   # rows of 16 bytes, contiguous before or not
        qs = query.stride()
    scratch = _scratch(dev, b, tokens, heads, hkv, dim, most)
    _launch(dev, _lib.lib().pa_kv8_attention, query.data_ptr(), qs[0], qs[1], tokens, heads, dim, k_pool.data_ptr(),
            v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), nb, bs, hkv, _DTYPE_CODE[query.dtype], scale, b,
            most, tables.data_ptr(), max(tables.stride(0), w), w, ctx, lens, cu, work, out.data_ptr(), heads * dim, dim,
            scratch.data_ptr(), scratch.shape[0])
    return out


class KV8Pool:
    """Per-layer 8-bit K and V pools with :class:`KVPool`'s attributes and block moves: ``k`` /
    ``v`` lists of e4m3 ``[num_blocks, block_size, Hkv, D]`` and ``k_scale`` / ``v_scale`` lists
    of bytes ``[num_blocks, Hkv, block_size]``, all zero-initialised.  ``dtype`` is the
    payload's."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device) -> None:
        if head_dim not in (64, 128):
            raise NotImplementedError(f"ATTENTION=cuda: head_dim {head_dim}: the 8-bit cache supports 64 and 128")
        if block_size < 16 or block_size & (block_size - 1) or block_size > 4096:
            raise NotImplementedError(f"ATTENTION=cuda: block_size {block_size}: the 8-bit cache supports 16, 32, ... 4096")
        self.num_blocks, self.block_size = num_blocks, block_size
        self.num_kv_heads, self.head_dim, self.dtype = num_kv_heads, head_dim, _PAYLOAD
        shape, sshape = (num_blocks, block_size, num_kv_heads, head_dim), (num_blocks, num_kv_heads, block_size)

        def payload():
            return torch.zeros(shape, dtype=torch.uint8, device=device).view(_PAYLOAD)

        def scales():
            return torch.zeros(sshape, dtype=torch.uint8, device=device)

        layers = range(num_layers)
        self.k, self.v = [payload() for _ in layers], [payload() for _ in layers]
        self.k_scale, self.v_scale = [scales() for _ in layers], [scales() for _ in layers]

    @classmethod
    def from_model(cls, model, num_blocks: int, block_size: int = 16, device=None) -> "KV8Pool":
        """Sizes off the model config as :meth:`KVPool.from_model` reads them."""
        cfg = model.config
        heads = getattr(cfg, "num_attention_heads", None) or cfg.n_head
        hidden = getattr(cfg, "hidden_size", None) or cfg.n_embd
        layers = getattr(cfg, "num_hidden_layers", None) or cfg.n_layer
        kv_heads = getattr(cfg, "num_key_value_heads", None) or heads
        head_dim = getattr(cfg, "head_dim", None) or hidden // heads
        return cls(layers, num_blocks, block_size, kv_heads, head_dim, device or next(model.parameters()).device)

    @property
    def num_slots(self) -> int:
        return self.num_blocks * self.block_size

    @property
    def nbytes(self) -> int:
        return sum(t.numel() for t in self.k + self.v + self.k_scale + self.v_scale)

    # ------------------------------------------------------------ block moves
    def _bytes(self):
        """The pools as byte tensors: payload lists, scale lists ``[blocks, 1, Hkv, BS]``."""
        u8 = torch.uint8
        return ([t.view(u8) for t in self.k], [t.view(u8) for t in self.v],
                [t.unsqueeze(1) for t in self.k_scale], [t.unsqueeze(1) for t in self.v_scale])

    def _err(self) -> torch.Tensor:
        if getattr(self, "_err_word", None) is None:
            self._err_word = _error_word(self.k[0].device)
        return self._err_word

    def read_error(self, clear: bool = True) -> int:
        """Error bits block moves reported since the last clear (1 = a bad block id).
        Synchronises the device."""
        word = int(self._err().item())
        if clear and word:
            self._err().zero_()
        return word

    def copy_blocks(self, pairs) -> None:
        """Copy-on-write moves ``pool[dst] = pool[src]`` for every layer, payload and scales."""
        k, v, ks, vs = self._bytes()
        pairs = list(pairs)
        copy_blocks(k, v, pairs, self._err())
        copy_blocks(ks, vs, pairs, self._err())

    def _block_bytes(self) -> tuple[int, int]:
        n = self.block_size * self.num_kv_heads
        return n * self.head_dim, n

    def swap_out(self, blocks) -> HostBlocks:
        """Copy the named blocks of every layer to pinned host memory: ``k`` / ``v`` are byte
        views per layer, ``flat`` holds [payload | scales], each [layer][K, V][n][block]."""
        n, layers = len(blocks), len(self.k)
        pb, sb = self._block_bytes()
        split = layers * 2 * n * pb
        flat = torch.empty(split + layers * 2 * n * sb, dtype=torch.uint8, pin_memory=True)
        if n:
            stage = torch.empty(flat.numel(), dtype=torch.uint8, device=self.k[0].device)
            k, v, ks, vs = self._bytes()
            gather_blocks(k, v, blocks, stage[:split], self._err())
            gather_blocks(ks, vs, blocks, stage[split:], self._err())
            flat.copy_(stage)
            if self.read_error():
                raise RuntimeError("swap_out: the gather kernel met a block id outside the pool")
        view = flat[:split].view(layers, 2, n, self.block_size, self.num_kv_heads, self.head_dim)
        return HostBlocks(k=[view[l, 0] for l in range(layers)], v=[view[l, 1] for l in range(layers)], flat=flat)

    def swap_in(self, host: HostBlocks, blocks) -> None:
        """Copy a host copy made by :meth:`swap_out` back into ``blocks``, which need not be the
        ones it left."""
        if len(blocks) != len(host):
            raise ValueError(f"swap_in: {len(host)} host blocks into {len(blocks)} device blocks")
        n, layers = len(blocks), len(self.k)
        if n == 0:
            return
        pb, sb = self._block_bytes()
        split = layers * 2 * n * pb
        if host.flat is None or host.flat.dtype != torch.uint8 or host.flat.numel() != split + layers * 2 * n * sb:
            raise ValueError("swap_in: the host copy was not made by a KV8Pool of this shape")
        stage = host.flat.to(self.k[0].device, non_blocking=True)
        k, v, ks, vs = self._bytes()
        scatter_blocks(k, v, blocks, stage[:split], self._err())
        scatter_blocks(ks, vs, blocks, stage[split:], self._err())
