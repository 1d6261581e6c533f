"""Plain 64-bit forms of the 8-bit paged cache's operators, on the CPU, one block or row at a time."""
from __future__ import annotations

import math

import numpy as np
import torch

HQ, HKV, GROUP, D, BLOCK = 32, 8, 4, 128, 16
THETA = 500000.0
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}


def plan(cached, n_new, free, n_free, table, n_rows):
    """paged_plan by a loop over requests.  -> table, seq_len, cu_new, slots, positions, n_free."""
    table = [list(r) for r in table]
    cap = BLOCK * (len(table[0]) if table else 0)
    n_free = max(0, min(n_free, len(free)))
    cu, need_sum, used = [0], 0, 0
    seq_len, slots, positions = [], [-1] * n_rows, [0] * n_rows
    for b, (c, n) in enumerate(zip(cached, n_new)):
        cu.append(cu[-1] + max(n, 0))
        valid = n >= 0 and c >= 0 and c + n <= cap and cu[-1] <= n_rows
        had = -(-c // BLOCK) if valid else 0
        need = -(-(c + n) // BLOCK) - had if valid else 0
        need_sum += need
        if not valid or (need and need_sum > n_free):
            seq_len.append(0)
            continue
        if need_sum <= n_free:
            used = need_sum
        for k in range(need):
            table[b][had + k] = free[n_free - 1 - (need_sum - need + k)]
        seq_len.append(c + n)
        for i in range(n):
            p = c + i
            slots[cu[b] + i] = table[b][p // BLOCK] * BLOCK + p % BLOCK
            positions[cu[b] + i] = p
    return table, seq_len, cu, slots, positions, n_free - used


def rope(x, pos, theta=THETA):
    """rotate_half in float64: x [n, heads, 128], pos n ints."""
    x = x.double()
    f = torch.tensor([theta ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64)
    ang = torch.as_tensor(pos, dtype=torch.float64)[:, None] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., : D // 2], x[..., D // 2:]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def nearest(x, fmt):
    """float64 code units -> the nearest value of the format (ties to even), saturating; NaN: NaN
    (e4m3) or 0 (int8)."""
    if fmt == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 448.0))) - 3)
    y = ((x.clamp(-448, 448) / step).round() * step).clamp(-448, 448)
    return torch.where(x.isnan(), x, y)


def scale_for(a, fmt):
    """The smallest power of two s with s * qmax >= a, at least 2^-126."""
    if a == 0.0:
        return 2.0 ** -126
    m, e = math.frexp(a / QMAX[fmt])                   # (one rounding: put right below)
    s = math.ldexp(1.0, e)
    while s * QMAX[fmt] < a:
        s *= 2
    while s / 2 * QMAX[fmt] >= a:
        s /= 2
    return max(s, 2.0 ** -126)


def append(codes, scales, x, slots, fmt):
    """One of K and V: rows x [n, 8, 128] (float64 holding float32 values) into codes [n_blocks, 8, 16,
    128] and scales [n_blocks, 8], both float64, in place."""
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= codes.shape[0] * BLOCK:
            t += 1
            continue
        run, e = [t], t + 1                            # skipped tokens end no run
        while e < len(slots) and not (0 <= slots[e] < codes.shape[0] * BLOCK and slots[e] // BLOCK != slots[t] // BLOCK):
            if 0 <= slots[e] < codes.shape[0] * BLOCK:
                run.append(e)
            e += 1
        blk, row = divmod(slots[t], BLOCK)
        rows = x[run]
        for h in range(HKV):
            a = torch.where(rows[:, h].isfinite(), rows[:, h].abs(), 0.0).max().item()
            s = scale_for(a, fmt)
            if row:
                old = scales[blk, h].item()
                old = old if 0.0 < old < math.inf else 0.0
                if s > old:
                    ratio = np.float32(np.float32(old) / np.float32(s))
                    moved = (codes[blk, h, :row].float() * float(ratio)).double()
                    codes[blk, h, :row] = nearest(moved, fmt)
                s = max(s, old)
            scales[blk, h] = s
            units = (rows[:, h].float() / torch.tensor(s, dtype=torch.float32)).double()
            codes[blk, h, row:row + len(run)] = nearest(units, fmt)
        t = e


def attend(q, codes_k, codes_v, scale_k, scale_v, table, seq_len, cu, *, rope_q=True, scale=None, theta=THETA):
    """-> (out, bound) float64 [N, 32, 128]: the definition's value of every row, and how far fp16
    operands and one BF16 rounding may take an output from it, from the arithmetic alone:

      * |q_i| is rounded by 2^-12 of itself at most (fp16's half step; elements far below their
        row's largest lose up to 2^-25 of that), so a score moves by at most
        ds = scale sum_i (2^-12 |q_i| + 2^-25 max|q|) |k_i| + fp32's 2^-17 of sum |q_i k_i| scale (128
        products, sums, exponent arithmetic and sines rounded to fp32), and p by expm1(2 ds);
      * a weight is rounded by 2^-12 of itself, or 2^-25 of the column's largest p sv;
      * fp32 sums over n keys: (n + 8) 2^-24 of sum p |v|;
      * BF16: 2^-8 of the value, and of what the others moved it to."""
    n_rows = q.shape[0]
    out = torch.full((n_rows, HQ, D), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(out)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    for b, length in enumerate(seq_len):
        lo, hi = cu[b], cu[b + 1]
        n = hi - lo
        if n <= 0 or length < n:
            continue
        pos = list(range(length - n, length))
        qr = rope(q[lo:hi], pos, theta) if rope_q else q[lo:hi].double()
        ids = list(table[b][: -(-length // BLOCK)])
        for h in range(HKV):
            sk = scale_k[ids, h].double().repeat_interleave(BLOCK)[:length]
            sv = scale_v[ids, h].double().repeat_interleave(BLOCK)[:length]
            k = codes_k[ids, h].double().reshape(-1, D)[:length] * sk[:, None]
            v = codes_v[ids, h].double().reshape(-1, D)[:length] * sv[:, None]
            for t in range(n):
                see = pos[t] + 1
                qt = qr[t, GROUP * h: GROUP * h + GROUP]                    # [4, 128]
                s = scale * (qt @ k[:see].T)
                p = torch.softmax(s, dim=-1)
                o = p @ v[:see]
                out[lo + t, GROUP * h: GROUP * h + GROUP] = o
                qa, ka, va = qt.abs(), k[:see].abs(), v[:see].abs()
                top = qa.amax(-1, keepdim=True)
                ds = abs(scale) * ((2.0 ** -12 * qa + 2.0 ** -25 * top) @ ka.T + 2.0 ** -17 * (qa @ ka.T))
                ds = ds.amax(-1, keepdim=True) + 2.0 ** -17 * s.abs().amax(-1, keepdim=True)
                rel = torch.expm1(2 * ds) + 2.0 ** -12 + (see + 8) * 2.0 ** -24
                floor = 2.0 ** -25 * (p * sv[:see]).amax(-1, keepdim=True)
                units = codes_v[ids, h].double().reshape(-1, D)[:see].abs().sum(0)
                err = rel * (p @ va) + floor * units
                bound[lo + t, GROUP * h: GROUP * h + GROUP] = 2.0 ** -8 * (o.abs() + err) + err
    return out, bound


def codes64(t):
    """A pool's codes as float64 on the CPU."""
    return t.detach().cpu().double() if t.dtype == torch.int8 else t.detach().cpu().float().double()
