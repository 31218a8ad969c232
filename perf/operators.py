"""The 8-bit paged KV cache's operators, as cases that can be timed and compared.

* ``tables``: a step's block tables and slot map built on the GPU from request lengths,
  with the blocks that the step still needs taken from a free list.
* ``append``: new K/V rows quantised into the paged pools (e4m3 payload, one power-of-two
  scale per row).
* ``attend``: attention of a chunk of new tokens (one token and more) over those pools.

``run`` computes each in elementary torch operations, or, where ``own`` is set, through
the package's entry points.  The scale byte b of a row stands for 2^(b - 127), as in
``torch.float8_e8m0fnu``; it lies in [113, 134], so every cached value is an fp16 number.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 16
E_MIN, E_MAX = -14, 7          # exponents of a row's scale
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # A few requests decoding: the call whose latency a small server sees every step.
        {"name": "tables decode 8", "op": "tables", "requests": 64, "rows": 8, "pad_rows": 0, "ctx": 900, "chunk": 1,
         "width": 128},
        # A full decode batch padded to its CUDA-graph bucket, speculative chunks of 4.
        {"name": "tables verify 500", "op": "tables", "requests": 512, "rows": 500, "pad_rows": 12, "ctx": 4096,
         "chunk": 4, "width": 1024},
        # Admission: long prompts packed into one prefill step.
        {"name": "tables prefill 13x2047", "op": "tables", "requests": 256, "rows": 13, "pad_rows": 0, "ctx": 0,
         "chunk": 2047, "width": 2048},
        # One decode step of a small batch.
        {"name": "append decode 32", "op": "append", "tokens": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # GPT-2's heads, an odd chunk, strided keys and values as a fused projection leaves them.
        {"name": "append gpt2 1001", "op": "append", "tokens": 1001, "kv_heads": 12, "dim": 64, "dtype": "f16"},
        # A packed prefill step.
        {"name": "append prefill 16384", "op": "append", "tokens": 16384, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # One request, one token, a short context: latency.
        {"name": "attend one 517", "op": "attend", "seqs": 1, "ctx": 517, "chunk": 1, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # GPT-2's heads, a ragged decode batch.
        {"name": "attend gpt2 decode 48x700", "op": "attend", "seqs": 48, "ctx": 700, "chunk": 1, "ragged": True,
         "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "f16"},
        # A serving decode batch of ragged contexts, grouped heads: the bandwidth-bound case.
        {"name": "attend decode 64x4096", "op": "attend", "seqs": 64, "ctx": 4096, "chunk": 1, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # One long conversation: the work has to be split along the context.
        {"name": "attend long 131071", "op": "attend", "seqs": 1, "ctx": 131071, "chunk": 1, "ragged": False,
         "heads": 64, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # Verification of speculated tokens.
        {"name": "attend verify 24x5x6000", "op": "attend", "seqs": 24, "ctx": 6000, "chunk": 5, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # A prefill chunk over a long cached prefix: the arithmetic-bound case.
        {"name": "attend chunk 1000x16384", "op": "attend", "seqs": 1, "ctx": 16384, "chunk": 1000, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend"])
    if op == "tables":
        rows = _log(rng, 1, 600)
        chunk = rng.choice([1, _log(rng, 2, 8), max(1, _log(rng, 16, 26000) // rows)])
        ctx = rng.choice([0, _log(rng, 1, 8000)])
        width = -(-(2 * ctx + chunk + 2) // BLOCK) + rng.randrange(0, 9)
        return {"op": op, "requests": rows + rng.randrange(0, 200), "rows": rows, "pad_rows": rng.choice([0, 0, 5]),
                "ctx": ctx, "chunk": chunk, "width": width}
    if op == "append":
        heads, dim = rng.choice([(8, 128), (12, 64), (2, 128), (1, 64), (4, 128)])
        return {"op": op, "tokens": _log(rng, 1, 16000), "kv_heads": heads, "dim": dim,
                "dtype": rng.choice(["bf16", "f16"])}
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (12, 12, 64), (16, 2, 128), (28, 4, 128), (8, 8, 64)])
    chunk = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 17, 800)])
    ctx = _log(rng, max(chunk, 4), 20000)
    most = min(64, max(1, 250000 // ctx), max(1, 8000000 // (chunk * ctx)))
    return {"op": op, "seqs": _log(rng, 1, most), "ctx": ctx, "chunk": chunk, "ragged": rng.random() < 0.7,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "f16"])}


# ------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Contexts and chunk lengths of an ``attend`` case: the same for every seed, so that
    the work is the case's own.  Ragged ones spread around the named length and include
    a chunk of one token."""
    n, ctx, chunk = case["seqs"], case["ctx"], case["chunk"]
    if not case["ragged"] or n == 1:
        return [ctx] * n, [chunk] * n
    g = torch.Generator().manual_seed(n * 1000003 + ctx)
    q = torch.randint(1, chunk + 1, (n,), generator=g)
    q[0] = chunk
    c = (torch.exp(0.4 * torch.randn(n, generator=g)) * ctx).long().clamp(1, 2 * ctx)
    return torch.maximum(c, q).tolist(), q.tolist()


def _rows(g, shape, dtype, device):
    """K/V rows as projections give them: unit spread, some channels and some rows larger."""
    x = torch.randn(shape, generator=g, device=device, dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device=device))
    x *= torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=g, device=device))
    return x.to(dtype)


def _power(byte):
    """2^(byte - 127) as float32, exactly: the byte is the number's exponent field."""
    return (byte.int() << 23).view(torch.float32)


def _quantise(x):
    """Rows [..., D] -> (e4m3 payload, scale bytes [...]).  The scale is the least power of
    two (exponent in [E_MIN, E_MAX]) that brings the row's largest magnitude to 448."""
    x = x.float()
    big = torch.where(x.isnan(), 0.0, x.abs()).amax(-1)
    m, e = torch.frexp(big.clamp(2.0 ** -30, 2.0 ** 30))         # big = m * 2^e, m in [0.5, 1)
    byte = (e - 9 + (m > 0.875).int()).clamp(E_MIN, E_MAX) + 127  # 448 = 0.875 * 2^9
    return (x / _power(byte)[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _pool(g, blocks, kv_heads, dim, device):
    """A pool's payload [blocks, BLOCK, kv_heads, dim] and scale bytes [blocks, kv_heads, BLOCK]."""
    payload = torch.empty(blocks, BLOCK, kv_heads, dim, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(blocks, kv_heads, BLOCK, dtype=torch.uint8, device=device)
    part = max(1, (1 << 26) // (BLOCK * kv_heads * dim))
    for b in range(0, blocks, part):
        n = min(part, blocks - b)
        y, s = _quantise(_rows(g, (n, BLOCK, kv_heads, dim), torch.float32, device))
        payload[b:b + n] = y
        scale[b:b + n] = s.transpose(1, 2)
    return payload, scale


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "tables":
        reqs, rows, width = case["requests"], case["rows"], case["width"]
        order = torch.randperm(reqs, generator=g, device=device)
        lens = torch.zeros(reqs, dtype=torch.int32, device=device)
        if case["ctx"]:
            spread = torch.exp(0.3 * torch.randn(reqs, generator=g, device=device)) * case["ctx"]
            lens = spread.clamp(1, min(2 * case["ctx"], width * BLOCK - case["chunk"])).int()
        held = (lens + BLOCK - 1) // BLOCK
        fresh = -(-case["chunk"] // BLOCK) + 1
        blocks = int(held.sum()) + rows * fresh + 64
        perm = torch.randperm(blocks, generator=g, device=device).int()
        j = torch.arange(width, device=device, dtype=torch.int32)
        first = torch.cumsum(held, 0) - held
        mine = j < held[:, None]
        tables = torch.where(mine, perm[(first[:, None] + j).clamp(max=blocks - 1).long()], 0).int()
        free = perm[int(held.sum()):].contiguous()
        lengths = torch.Generator().manual_seed(rows * 1000003 + case["chunk"])    # the case's own, for every seed
        q = torch.randint(1, case["chunk"] + 1, (rows,), generator=lengths, dtype=torch.int32)
        q[0] = case["chunk"]
        q = q.to(device)
        pad = torch.zeros(case["pad_rows"], dtype=torch.int32, device=device)
        s.update(tables=tables, lens=lens, held=held.int(), free=free,
                 num_free=torch.tensor([free.numel()], dtype=torch.int32, device=device),
                 request_ids=torch.cat([order[:rows].int(), pad - 1]), query_lens=torch.cat([q, pad]),
                 tokens=int(q.sum()) + case["pad_rows"], blocks=blocks)
        return s
    heads, dim, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        t = case["tokens"]
        blocks = -(-t // BLOCK) + 64
        kv = _rows(g, (t, 2 * heads, dim), dtype, device)      # one projection's output: K and V are strided views
        s.update(key=kv[:, :heads], value=kv[:, heads:])
        s["k_pool"], s["k_scale"] = _pool(g, blocks, heads, dim, device)
        s["v_pool"], s["v_scale"] = _pool(g, blocks, heads, dim, device)
        s["slots"] = torch.randperm(blocks * BLOCK, generator=g, device=device)[:t].int()
        return s
    ctx, q = _lengths(case)
    need = [-(-c // BLOCK) for c in ctx]
    blocks = sum(need) + 7
    s["k_pool"], s["k_scale"] = _pool(g, blocks, heads, dim, device)
    s["v_pool"], s["v_scale"] = _pool(g, blocks, heads, dim, device)
    perm = torch.randperm(blocks, generator=g, device=device).int()
    n = torch.tensor(need, device=device)
    j = torch.arange(max(need), device=device)
    at = (torch.cumsum(n, 0) - n)[:, None] + j
    s["tables"] = torch.where(j < n[:, None], perm[at.clamp(max=blocks - 1)], 0).int()
    s["context_lens"] = torch.tensor(ctx, dtype=torch.int32, device=device)
    s["query_lens"] = torch.tensor(q, dtype=torch.int32, device=device)
    s["query"] = torch.randn(sum(q), case["heads"], dim, generator=g, device=device).to(dtype)
    s["softmax_scale"] = dim ** -0.5
    return s


# ------------------------------------------------------------------------------ the plain forms
def _run_tables(s):
    req, width, t = s["request_ids"].long(), s["width"], s["tokens"]
    valid = req >= 0
    row = req.clamp_min(0)
    q = torch.where(valid, s["query_lens"], 0)
    held = torch.where(valid, s["held"][row], 0)
    ctx = torch.where(valid, s["lens"][row], 0) + q
    need = ((ctx + BLOCK - 1) // BLOCK - held).clamp_min(0)
    before = torch.cumsum(need, 0) - need
    j = torch.arange(width, device=req.device)
    k = j - held[:, None]                                              # place among the row's new blocks
    new = (k >= 0) & (k < need[:, None])
    top = (s["num_free"] - 1 - before)[:, None] - k
    ids = torch.where(new, s["free"][top.clamp(0, s["free"].numel() - 1)], s["tables"][row])
    ids = torch.where(j < (held + need)[:, None], ids, 0).int()
    kept = torch.cat([s["tables"], s["tables"][:1]])                   # the last row takes the padding's writes
    at = torch.where(valid, row, s["requests"])
    kept[at] = torch.where(new, ids, kept[at])
    cu = torch.cat([q.new_zeros(1), torch.cumsum(q, 0)]).int()
    tok = torch.arange(t, device=req.device)
    seq = torch.searchsorted(cu[1:].contiguous(), tok.int(), right=True).clamp(max=req.numel() - 1)
    pos = (ctx - q)[seq] + tok - cu[seq]
    slot = ids[seq, (pos // BLOCK).clamp(0, width - 1)] * BLOCK + pos % BLOCK
    real = tok < cu[-1]
    return {"block_tables": ids, "context_lens": ctx.int(), "cu_query_lens": cu,
            "seq_idx": torch.where(real, seq, -1).int(), "q_pos": torch.where(real, pos, -1).int(),
            "slot_mapping": torch.where(real, slot, -1).int(), "tables": kept[:-1],
            "num_free": (s["num_free"] - need.sum()).int()}


def _run_append(s):
    at = s["slots"].long()
    block, offset = at // BLOCK, at % BLOCK
    for rows, pool, scale in ((s["key"], "k_pool", "k_scale"), (s["value"], "v_pool", "v_scale")):
        payload, byte = _quantise(rows)
        raw = s[pool].view(torch.uint8).view(-1, s["kv_heads"], s["dim"])
        raw[at] = payload.view(torch.uint8)
        s[scale][block, :, offset] = byte
    return {k: s[k] for k in ("k_pool", "k_scale", "v_pool", "v_scale")}


def _gather(pool, scale, tables):
    """The pool's values in the order of the tables: [B, W * BLOCK, kv_heads, dim] in 32 bits."""
    b, w = tables.shape
    x = pool.view(torch.uint8)[tables].view(torch.float8_e4m3fn).float()
    x *= _power(scale[tables]).transpose(2, 3)[..., None]
    return x.view(b, w * BLOCK, pool.shape[2], pool.shape[3])


def _run_attend(s):
    tables, ctx, q = s["tables"].long(), s["context_lens"].long(), s["query_lens"].long()
    b, most, heads, group = q.numel(), s["chunk"], s["kv_heads"], s["heads"] // s["kv_heads"]
    k, v = _gather(s["k_pool"], s["k_scale"], tables), _gather(s["v_pool"], s["v_scale"], tables)
    key = torch.arange(k.shape[1], device=q.device)
    v = torch.where((key < ctx[:, None])[..., None, None], v, 0.0)     # what lies behind a context is not read
    first = torch.cumsum(q, 0) - q
    t = torch.arange(most, device=q.device)
    there = t < q[:, None]
    query = s["query"].float()[(first[:, None] + t).clamp(max=s["query"].shape[0] - 1)]
    query = query.view(b, most, heads, group, s["dim"])
    score = torch.einsum("bthgd,bkhd->bhgtk", query, k) * s["softmax_scale"]
    seen = key <= ((ctx - q)[:, None] + t)[..., None]
    score = torch.where(seen[:, None, None], score, -torch.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.einsum("bhgtk,bkhd->bthgd", weight / weight.sum(-1, keepdim=True), v)
    out = out.reshape(b * most, s["heads"], s["dim"])
    # Packed order: token i of the call is row seq * most + place of the padded batch.
    tok = torch.arange(s["query"].shape[0], device=q.device)
    seq = torch.searchsorted(torch.cumsum(q, 0), tok, right=True)
    return out[seq * most + tok - first[seq]].to(s["query"].dtype)


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _run_tables, "append": _run_append, "attend": _run_attend}[s["op"]](s)


# ------------------------------------------------------------------------------ the package's calls
def _run_own(s):
    from __graft_entry__ import import_package

    pkg = import_package()
    if s["op"] == "tables":
        bt = pkg.DeviceBlockTables.adopt(s["tables"], s["lens"], s["held"], s["free"], s["num_free"],
                                         num_blocks=s["blocks"], block_size=BLOCK)
        step = bt.reserve(s["request_ids"], s["query_lens"], num_tokens=s["tokens"], max_query_len=s["chunk"])
        return {"block_tables": step.block_tables, "context_lens": step.context_lens,
                "cu_query_lens": step.cu_query_lens, "seq_idx": step.seq_idx, "q_pos": step.q_pos,
                "slot_mapping": step.slot_mapping, "tables": bt.tables, "num_free": step.num_free}
    if s["op"] == "append":
        pkg.reshape_and_cache_kv8(s["key"], s["value"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"],
                                  s["slots"])
        return {k: s[k] for k in ("k_pool", "k_scale", "v_pool", "v_scale")}
    return pkg.paged_attention_kv8(s["query"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["tables"],
                                   s["context_lens"], s["query_lens"], s["softmax_scale"], max_query_len=s["chunk"])


# ------------------------------------------------------------------------------ work and the definition in 64 bits
def work(case):
    if case["op"] == "tables":
        rows, tokens = case["rows"] + case["pad_rows"], case["rows"] * (case["chunk"] + 1) // 2
        held = min(case["width"], -(-(case["ctx"] + case["chunk"]) // BLOCK))
        return {"bytes": 4 * (case["rows"] * held + rows * case["width"] + 3 * tokens + 6 * rows), "flops": 0}
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return {"bytes": case["tokens"] * (2 * heads * (2 * dim + dim + 1) + 4),
                "flops": case["tokens"] * 2 * heads * dim * 2}
    ctx, q = _lengths(case)
    pairs = sum(t * (c - t) + t * (t + 1) // 2 for c, t in zip(ctx, q))
    return {"bytes": sum(ctx) * heads * 2 * (dim + 1) + 4 * sum(-(-c // BLOCK) for c in ctx)
            + 2 * 2 * sum(q) * case["heads"] * dim,
            "flops": 4 * case["heads"] * dim * pairs}


def _two_to(e):
    """2^e in 64 bits for whole e within +-64, exactly."""
    return torch.tensor([2.0 ** k for k in range(-64, 65)], dtype=torch.float64, device=e.device)[e.long() + 64]


def _to_e4m3(y):
    """The nearest e4m3 value (ties to the even one) of a float64 tensor within +-448."""
    step = _two_to(torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent - 4)    # 2^(e-1) <= |y|: three bits behind it
    return torch.round(y / step) * step


def exact(case, seed):
    if case["op"] == "tables":
        return None                                                    # whole numbers: they are compared as such
    s = prepare(case, seed)
    if case["op"] == "append":
        at = s["slots"].long()
        for rows, pool, scale in ((s["key"], "k_pool", "k_scale"), (s["value"], "v_pool", "v_scale")):
            x = rows.double()
            m, e = torch.frexp(x.abs().amax(-1).clamp_min(1e-30) / 448.0)
            e = (e - (m == 0.5).int()).clamp(E_MIN, E_MAX)              # the least e with 2^e >= amax / 448
            s[pool] = s[pool].double()
            s[pool].view(-1, case["kv_heads"], case["dim"])[at] = _to_e4m3(x * _two_to(-e)[..., None])
            s[scale][at // BLOCK, :, at % BLOCK] = (e + 127).to(torch.uint8)
        return {k: s[k] for k in ("k_pool", "k_scale", "v_pool", "v_scale")}
    ctx, lens = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out, first = torch.empty(s["query"].shape, dtype=torch.float64, device=s["query"].device), 0
    for i, (c, n) in enumerate(zip(ctx, lens)):
        ids = s["tables"][i, :-(-c // BLOCK)].long()
        for h in range(case["kv_heads"]):
            k, v = (s[p].view(torch.uint8)[ids, :, h].view(torch.float8_e4m3fn).double()
                    * _two_to(s[e][ids, h].int() - 127)[..., None] for p, e in
                    (("k_pool", "k_scale"), ("v_pool", "v_scale")))
            k, v = k.reshape(-1, case["dim"])[:c], v.reshape(-1, case["dim"])[:c]
            q = s["query"][first:first + n, h * group:(h + 1) * group].double().transpose(0, 1)
            a = q @ k.T * s["softmax_scale"]
            hidden = torch.ones(n, c, dtype=torch.bool, device=a.device).triu(c - n + 1)
            a = torch.softmax(a.masked_fill(hidden, -torch.inf), -1)
            out[first:first + n, h * group:(h + 1) * group] = (a @ v).transpose(0, 1)
        first += n
    return out
