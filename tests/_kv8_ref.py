"""Plain 64-bit forms of the 8-bit cache's operators, for the tests."""

from __future__ import annotations

import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def e4m3_table() -> np.ndarray:
    """The value of each of the 256 e4m3 codes (1 sign, 4 exponent, 3 mantissa bits; bias 7)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = (-1.0 if c & 128 else 1.0), (c >> 3) & 15, c & 7
        out[c] = s * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        if e == 15 and m == 7:
            out[c] = math.nan
    return out


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Rows [..., D] -> (codes uint8 [..., D], scale bytes uint8 [...])."""
    x = np.asarray(x, dtype=np.float64)
    flat = x.reshape(-1, x.shape[-1])
    codes, bytes_ = np.zeros(flat.shape, np.uint8), np.zeros(flat.shape[0], np.uint8)
    grid = e4m3_table()[:127]                      # non-negative finite values, ascending
    mids = (grid[1:] + grid[:-1]) / 2
    for i, row in enumerate(flat):
        if np.isnan(row).any():
            bytes_[i] = 255
            continue
        e = -14
        while e < 7 and np.abs(row).max() > 448.0 * 2.0 ** e:
            e += 1
        y = np.minimum(np.abs(row) * 2.0 ** -e, 448.0)
        k = np.searchsorted(mids, y, side="left")  # index of the nearest, a midpoint going down
        tie = (k < len(mids)) & (y == mids[np.minimum(k, len(mids) - 1)])
        k = np.where(tie & (k % 2 == 1), k + 1, k)  # ties to the even code
        codes[i] = k.astype(np.uint8) | np.where(np.signbit(row), 128, 0).astype(np.uint8)
        bytes_[i] = e + 127
    return codes.reshape(x.shape), bytes_.reshape(x.shape[:-1])


def dequantise(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Pool codes uint8 [NB, BS, Hkv, D] and bytes [NB, Hkv, BS] -> float64 values."""
    table = torch.from_numpy(e4m3_table()).to(codes.device)
    power = torch.tensor([2.0 ** (b - 127) if b < 255 else math.nan for b in range(256)], dtype=torch.float64,
                         device=codes.device)
    return table[codes.long()] * power[scale.long()].transpose(1, 2)[..., None]


def attention(query, k, v, tables, ctx, ql, scale):
    """(out, weight-averaged |v|, bound on the scores' float32 error) in 64 bits; k, v are
    dequantised pools [NB, BS, Hkv, D]; only keys inside each context are read."""
    t, hq, d = query.shape
    hkv, bs = k.shape[2], k.shape[1]
    g = hq // hkv
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=query.device)
    mean = torch.zeros_like(out)
    slip = torch.zeros(t, hq, dtype=torch.float64, device=query.device)
    at = 0
    for i, (c, n) in enumerate(zip(ctx, ql)):
        if n == 0:
            continue
        ids = tables[i, :-(-c // bs)].long()
        kk = k[ids].reshape(-1, hkv, d)[:c]
        vv = v[ids].reshape(-1, hkv, d)[:c]
        q = query[at:at + n].double().view(n, hkv, g, d)
        s = torch.einsum("thgd,khd->thgk", q, kk) * scale
        big = torch.einsum("thgd,khd->thgk", q.abs(), kk.abs()) * abs(scale)
        seen = torch.arange(c, device=q.device)[None] <= (c - n + torch.arange(n, device=q.device))[:, None]
        seen = seen[:, None, None]
        s = torch.where(seen, s, -torch.inf)
        p = torch.softmax(s, -1)
        vz = torch.nan_to_num(vv, nan=0.0)
        out[at:at + n] = torch.einsum("thgk,khd->thgd", p, vz).reshape(n, hq, d)
        mean[at:at + n] = torch.einsum("thgk,khd->thgd", p, vz.abs()).reshape(n, hq, d)
        slip[at:at + n] = torch.where(seen, big, 0.0).amax(-1).reshape(n, hq)
        at += n
    return out, mean, slip


def tolerance(ref, mean, slip, dtype, d, keys):
    """How far the kernel's output may be from 64 bits, elementwise.

    * its own rounding: eps / 2 of the value;
    * each weight rounded to fp16, 2^-11 of it, so 2^-11 of sum p |v| (the float32
      exponential, sums and products add 2^-20: inside the 2^-12 allowed on top);
    * weights below fp16's normal range are off by 2^-25 absolute, times a payload of up to
      448 and the shift back by 2^-8, at every key (the denominator is at least 1);
    * a score is a float32 sum of d products: off by (d + 8) 2^-24 of sum |q||k| scale, in
      the exponent, numerator and denominator alike: twice that of sum p |v|."""
    eps = torch.finfo(dtype).eps
    score = (d + 8) * 2.0 ** -24 * slip[..., None]
    return eps / 2 * ref.abs() + (2.0 ** -11 + 2.0 ** -12 + 2 * score) * mean + keys * 448 * 2.0 ** -33 + 1e-30


def step_tables(request_ids, query_lens, tables, lens, held, free, num_free, width, bs, tokens):
    """The step that DeviceBlockTables.reserve builds, by loops over Python integers."""
    b = len(request_ids)
    out = {"block_tables": np.zeros((b, width), np.int32), "context_lens": np.zeros(b, np.int32),
           "query_lens": np.zeros(b, np.int32), "held": np.zeros(b, np.int32),
           "cu_query_lens": np.zeros(b + 1, np.int32), "seq_idx": np.full(tokens, -1, np.int32),
           "q_pos": np.full(tokens, -1, np.int32), "slot_mapping": np.full(tokens, -1, np.int32),
           "tables": np.array(tables)}
    left, at = int(num_free), 0
    for i in range(b):
        r = int(request_ids[i])
        if r >= 0:
            q = int(query_lens[i])
            ctx = int(lens[r]) + q
            row = [int(x) for x in tables[r][:held[r]]]
            while len(row) * bs < ctx:
                left -= 1
                row.append(int(free[left]))
            out["tables"][r, :len(row)] = row
            out["block_tables"][i, :len(row)] = row
            out["context_lens"][i], out["query_lens"][i], out["held"][i] = ctx, q, len(row)
            for t in range(q):
                pos = ctx - q + t
                out["seq_idx"][at], out["q_pos"][at] = i, pos
                out["slot_mapping"][at] = row[pos // bs] * bs + pos % bs
                at += 1
        out["cu_query_lens"][i + 1] = at
    out["num_free"] = np.array([left], np.int32)
    return out


def lost_weight(tables, ctx, ql, v, hq, floor):
    """What a row may lose to weights below fp16's normal range: each of its keys is off by at
    most ``floor`` of the largest weight, times the largest |v| that the row's head sees."""
    bs, hkv = v.shape[1], v.shape[2]
    rows = []
    for i, (c, n) in enumerate(zip(ctx, ql)):
        if n == 0:
            continue
        vv = torch.nan_to_num(v[tables[i, :-(-c // bs)].long()].reshape(-1, hkv, v.shape[3])[:c], nan=0.0)
        rows.append((c * floor * vv.abs().amax((0, 2))).repeat_interleave(hq // hkv).expand(n, hq))
    return torch.cat(rows)[..., None]


def tight_tolerance(want, mean, slip, lost, dtype, d):
    """``tolerance`` with what small weights lose counted per row and relative to its values:
    output's rounding, 2^-11 and 2^-12 of sum p |v| for the weights' rounding and the float32
    arithmetic, the scores' error, and ``lost``.  The rounding is half a step: eps / 2 of the
    value, and below the type's least normal number, where steps no longer shrink, eps / 2 of
    that one (fp16: 2^-25)."""
    score = (d + 8) * 2.0 ** -24 * slip[..., None]
    n = lost.shape[0]
    info = torch.finfo(dtype)
    return info.eps / 2 * want[:n].abs().clamp_min(info.tiny) + (2.0 ** -11 + 2.0 ** -12 + 2 * score[:n]) * mean[:n] + lost
