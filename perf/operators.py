"""The operators of a serving step over an 8-bit paged cache, as measurable cases.

listed()          the named cases: smallest to largest calls of every operator
draw(rng)         one more case of the same ranges
prepare(case, s)  what a program holds before the call, on the GPU, values from seed s
run(state)        one pass: the plain form in torch, or (own) the framework's entry points
exact(case, s)    the floating outputs from the definition in float64
work(case)        the bytes and flops a pass cannot do without

Kinds of case (field "kind"):
  plan    paged_plan: block table entries, slots, positions and lengths of a step's tokens
  append  kv_append_q8: new K (rotated) and V rows quantised into the blocks of a pool
  attend  gqa_attention_q8: the step's ragged query rows over that pool

A case's sizes and lengths follow from the case alone (field "lengths" seeds the ragged draws);
a seed changes values, block ids and, for plan, nothing that a size depends on.
"""
import math
import random

import torch

own = False

HQ, HKV, D, BLOCK = 32, 8, 128, 16
GROUP = HQ // HKV
THETA = 500000.0
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -126


def listed():
    return [
        # The bookkeeping of a serving batch's decode step: latency.
        {"name": "plan_decode_b64", "kind": "plan", "batch": 64, "long": 0, "chunk": 1, "high": 8191,
         "max_blocks": 512, "free": 1.0, "pad": 0, "lengths": 11},
        # A busy server's mixed step: decodes beside chunks of prompts, rows padded for a graph.
        {"name": "plan_mixed_b256_8x500", "kind": "plan", "batch": 256, "long": 8, "chunk": 500, "high": 8191,
         "max_blocks": 576, "free": 1.0, "pad": 77, "lengths": 12},
        # Prompts of a whole large batch, more than the pool still holds.
        {"name": "plan_prompts_b2048_131072", "kind": "plan", "batch": 2048, "long": 2048, "chunk": 64,
         "high": 1000, "max_blocks": 128, "free": 0.9, "pad": 0, "lengths": 13},
        # One token each of a serving batch, most of them inside a block that others fill already.
        {"name": "append_b64_e4m3", "kind": "append", "format": "e4m3", "batch": 64, "long": 0, "chunk": 1,
         "high": 4000, "pad": 0, "lengths": 21},
        # A ragged mixed step: chunks that start and end inside a block, decodes, padded rows.
        {"name": "append_b24_4x333_int8", "kind": "append", "format": "int8", "batch": 24, "long": 4, "chunk": 333,
         "high": 2000, "pad": 9, "lengths": 22},
        # A large prefill step.
        {"name": "append_b8_8x2048_e4m3", "kind": "append", "format": "e4m3", "batch": 8, "long": 8, "chunk": 2048,
         "high": 4096, "pad": 0, "lengths": 23},
        # One user's decode step at a medium context: latency.
        {"name": "decode_b1_4096_e4m3", "kind": "attend", "format": "e4m3", "batch": 1, "long": 0, "chunk": 1,
         "short": 1, "low": 4096, "high": 4096, "q_scale": 1.0, "lengths": 31},
        # A serving batch with ragged contexts: the headline workload on the 8-bit cache.
        {"name": "decode_b64_512_8192_e4m3", "kind": "attend", "format": "e4m3", "batch": 64, "long": 0, "chunk": 1,
         "short": 1, "low": 512, "high": 8192, "q_scale": 1.0, "lengths": 20260805},
        # Long-context decode, the largest memory-bound call.
        {"name": "decode_b8_131072_int8", "kind": "attend", "format": "int8", "batch": 8, "long": 0, "chunk": 1,
         "short": 1, "low": 131072, "high": 131072, "q_scale": 1.0, "lengths": 33},
        # Drafted tokens of a serving batch checked at once, 1 to 8 of them for each sequence.
        {"name": "verify_b64_t8_512_8192_int8", "kind": "attend", "format": "int8", "batch": 64, "long": 0, "chunk": 1,
         "short": 8, "low": 512, "high": 8192, "q_scale": 1.0, "lengths": 34},
        # Chunked prefill of four users over long contexts: the matrix-core workload.
        {"name": "chunk_b4_512_over_8192_e4m3", "kind": "attend", "format": "e4m3", "batch": 4, "long": 4, "chunk": 512,
         "short": 1, "low": 8704, "high": 8704, "q_scale": 1.0, "lengths": 35},
        # A mixed step: two chunks of odd length beside decodes, sharper scores than N(0,1) gives.
        {"name": "mixed_b24_2x301_int8", "kind": "attend", "format": "int8", "batch": 24, "long": 2, "chunk": 301,
         "short": 1, "low": 400, "high": 4000, "q_scale": 4.0, "lengths": 36},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their ranges, no more work than the
    largest listed call of its kind."""
    kind = rng.choice(["plan", "append", "attend", "attend", "attend"])
    case = {"kind": kind, "lengths": rng.randrange(1, 1 << 30)}
    if kind == "plan":
        batch = _log_int(rng, 1, 2048)
        long = rng.choice([0, rng.randint(0, batch)])
        chunk = _log_int(rng, 2, max(2, min(4096, 120000 // max(1, long))))
        high = _log_int(rng, 16, 16384)
        case.update(batch=batch, long=long, chunk=chunk, high=high, max_blocks=(high + chunk) // BLOCK + 1,
                    free=rng.choice([1.0, 1.0, 0.5]), pad=rng.choice([0, rng.randint(1, 300)]))
        return case
    case["format"] = rng.choice(["int8", "e4m3"])
    if kind == "append":
        batch = _log_int(rng, 1, 256)
        long = rng.choice([0, 0, rng.randint(0, min(batch, 16))])
        chunk = _log_int(rng, 2, max(2, min(4096, 15000 // max(1, long))))
        case.update(batch=batch, long=long, chunk=chunk, high=_log_int(rng, 1, 4096),
                    pad=rng.choice([0, rng.randint(1, 40)]))
        return case
    case["q_scale"] = rng.choice([1.0, 1.0, 4.0])
    shape = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    if shape in ("decode", "verify"):
        batch = _log_int(rng, 1, 96)
        high = _log_int(rng, 16, min(131072, 900000 // batch))
        short = 1 if shape == "decode" else rng.randint(2, 16)
        if shape == "verify":
            high = min(high, 300000 // batch)
        case.update(batch=batch, long=0, chunk=1, short=short, low=rng.choice([1, max(1, high // 8), high]), high=high)
        return case
    long = _log_int(rng, 1, 4)
    batch = long if shape == "chunk" else long + _log_int(rng, 1, 24)
    chunk = _log_int(rng, 17, 1024 // long)
    most = min(8192, 2_000_000 // (batch * chunk))
    high = chunk + _log_int(rng, 1, max(2, most))
    case.update(batch=batch, long=long, chunk=chunk, short=1, low=rng.choice([1, high]), high=high)
    return case


# ---------------------------------------------------------------------------- inputs


def _news(case):
    """New tokens of each sequence: `long` of them have about `chunk`, the others up to `short`."""
    r = random.Random(case["lengths"] * 3 + 1)
    batch, long, chunk, short = case["batch"], case["long"], case["chunk"], case.get("short", 1)
    at = set(r.sample(range(batch), long))
    news = []
    for b in range(batch):
        if b in at:
            news.append(chunk if long == batch else r.randint((chunk + 1) // 2, chunk))
        elif short > 1:
            news.append(r.randint(1, short))
        else:                                  # a few requests of a plan or an append rest this step
            news.append(0 if case["kind"] != "attend" and batch > 8 and r.random() < 0.05 else 1)
    return news


def _lens(case, news):
    """Positions of each sequence: with the new ones (attend), before them (plan, append)."""
    r = random.Random(case["lengths"])
    if case["kind"] == "attend":
        return [max(n, r.randint(case["low"], case["high"])) for n in news]
    return [r.randint(0, case["high"]) for _ in news]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _shuffled_table(counts, width, gen):
    """A block table of `width` entries a row: counts[b] ids of a shuffled pool each, -1 behind;
    and how many blocks that pool has (a few more than are used)."""
    n_blocks = sum(counts) + 3
    ids = torch.randperm(n_blocks, generator=gen, device="cuda").to(torch.int32)
    have = _i32(counts).long()
    first = have.cumsum(0) - have
    j = torch.arange(width, device="cuda")
    flat = torch.where(j < have[:, None], first[:, None] + j, -1)
    return torch.where(flat >= 0, ids[flat.clamp(min=0)], -1).to(torch.int32), n_blocks


def _codes(n_blocks, fmt, gen):
    """A pool's codes and scales as appends of N(0,1) rows leave them: a block's largest
    magnitude a factor 1 to 2 below what its scale reaches, scales of powers of two."""
    x = torch.randn((n_blocks, HKV, BLOCK, D), generator=gen, device="cuda")
    scale = torch.exp2(torch.randint(-1, 2, (n_blocks, HKV), generator=gen, device="cuda").float())
    if fmt == "int8":
        return (x * 30.0).round_().clamp_(-127, 127).to(torch.int8), scale / 32
    x = (x * 90.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return x, scale / 128


def _spoil_behind(pool, table, lens, fmt):
    """NaN codes (e4m3: 127) in the rows of each sequence's last block behind its end."""
    if fmt != "e4m3":
        return
    rows = pool.view(torch.uint8)
    n = _i32(lens).long()
    last = torch.gather(table, 1, ((n - 1) // BLOCK)[:, None]).long()[:, 0]
    behind = torch.arange(BLOCK, device="cuda")[None, :] > ((n - 1) % BLOCK)[:, None]
    rows[last] = torch.where(behind[:, None, :, None], 127, rows[last])


def _prepare_plan(case, seed):
    news = _news(case)
    cached = _lens(case, news)
    cached = [min(c, BLOCK * case["max_blocks"] - n) for c, n in zip(cached, news)]
    gen = torch.Generator("cuda").manual_seed(1000003 * int(seed) + case["lengths"] % 1000003)
    need = sum(_blocks(c + n) - _blocks(c) for c, n in zip(cached, news))
    table, used = _shuffled_table([_blocks(c) for c in cached], case["max_blocks"], gen)
    spare = max(1, int(need * case["free"]) + (5 if case["free"] == 1.0 else 0))
    free = (used + torch.randperm(spare + 8, generator=gen, device="cuda")).to(torch.int32)
    return {"kind": "plan", "cached": _i32(cached), "news": _i32(news), "table": table, "free": free,
            "n_free": _i32([spare]), "rows": sum(news) + case["pad"]}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda").to(torch.bfloat16)


def _prepare_append(case, seed):
    news = _news(case)
    cached = _lens(case, news)
    gen = torch.Generator("cuda").manual_seed(1000003 * int(seed) + case["lengths"] % 1000003)
    total = [c + n for c, n in zip(cached, news)]
    table, n_blocks = _shuffled_table([_blocks(t) for t in total], _blocks(max(total)) + 1, gen)
    k, k_scale = _codes(n_blocks, case["format"], gen)
    v, v_scale = _codes(n_blocks, case["format"], gen)
    seq = torch.repeat_interleave(torch.arange(len(news), device="cuda"), _i32(news).long())
    cu = torch.tensor([0] + news, device="cuda").cumsum(0)
    pos = torch.arange(sum(news), device="cuda") - cu[seq] + _i32(cached).long()[seq]
    slots = table[seq, pos // BLOCK].long() * BLOCK + pos % BLOCK
    pad = torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")
    slots = torch.cat((slots, pad)).to(torch.int32)
    pos = torch.cat((pos, pad * 0)).to(torch.int32)
    rows = sum(news) + case["pad"]
    # K and V rows are the tail of the fused projection's rows, as a model hands them over
    qkv = _randn(gen, rows, HQ + 2 * HKV, D)
    return {"kind": "append", "format": case["format"], "k_new": qkv[:, HQ:HQ + HKV], "v_new": qkv[:, HQ + HKV:],
            "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "slots": slots, "pos": pos}


def _prepare_attend(case, seed):
    news = _news(case)
    lens = _lens(case, news)
    gen = torch.Generator("cuda").manual_seed(1000003 * int(seed) + case["lengths"] % 1000003)
    table, n_blocks = _shuffled_table([_blocks(n) for n in lens], _blocks(max(lens)), gen)
    k, k_scale = _codes(n_blocks, case["format"], gen)
    v, v_scale = _codes(n_blocks, case["format"], gen)
    _spoil_behind(k, table, lens, case["format"])
    _spoil_behind(v, table, lens, case["format"])
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = (torch.randn((cu[-1], HQ, D), generator=gen, device="cuda") * case["q_scale"]).to(torch.bfloat16)
    s = {"kind": "attend", "format": case["format"], "q": q, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale,
         "table": table, "lens": _i32(lens), "cu": _i32(cu), "max_new": max(news)}
    s["call"] = [None]           # the bound call of a serving loop: made at its first use, then kept
    return s


def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------- plain forms


def _plain_plan(s):
    c, n = s["cached"].long(), s["news"].long()
    rows, f = s["rows"], s["n_free"].long()
    table = s["table"].long()
    cu = torch.cat((c.new_zeros(1), n.clamp(min=0).cumsum(0)))
    valid = (n >= 0) & (c >= 0) & (c + n <= BLOCK * table.shape[1]) & (cu[1:] <= rows)
    had = (c + BLOCK - 1) // BLOCK
    need = torch.where(valid, (c + n + BLOCK - 1) // BLOCK - had, 0)
    upto = need.cumsum(0)
    granted = valid & ((need == 0) | (upto <= f))
    used = torch.where(upto <= f, upto, 0).max()
    j = torch.arange(table.shape[1], device="cuda")
    fresh = granted[:, None] & (j >= had[:, None]) & (j < (had + need)[:, None])
    at = f - 1 - ((upto - need)[:, None] + j - had[:, None])
    table = torch.where(fresh, s["free"].long()[at.clamp(0, s["free"].numel() - 1)], table)
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    inside = b < c.numel()
    b = b.clamp(max=c.numel() - 1)
    ok = inside & granted[b]
    pos = torch.where(ok, c[b] + t - cu[b], 0)
    slot = torch.where(ok, table[b, pos // BLOCK] * BLOCK + pos % BLOCK, -1)
    i = torch.int32
    return {"table": table.to(i), "seq_len": torch.where(granted, c + n, 0).to(i), "cu_new": cu.to(i),
            "slots": slot.to(i), "positions": pos.to(i), "n_free": (f - used).to(i)}


def _rope(x, pos):
    """rotate_half RoPE in float64: x [n, heads, 128], pos [n]."""
    freq = THETA ** (torch.arange(D // 2, dtype=torch.float64, device=x.device) * (-2.0 / D))
    ang = pos.double()[:, None, None] * freq
    c, s = ang.cos(), ang.sin()
    a, b = x.double().split(D // 2, dim=-1)
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _scale_for(a, qmax):
    """The smallest power of two s with s * qmax >= a, at least 2^-126 (a: float32)."""
    m, e = torch.frexp(a)                                         # a = m 2^e, m in [0.5, 1)
    top, te = math.frexp(qmax)
    s = torch.exp2((e - te + (m > top).to(e.dtype)).float().clamp(min=-126))
    return torch.where(a > 0, s, MIN_SCALE)


def _encode(x, fmt):
    """float32 values in code units -> codes, to nearest even, saturating."""
    if fmt == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_quantise(x, codes, scales, slots, fmt):
    """One of K and V: rows x [n, 8, 128] float32 into codes and scales in place."""
    keep = slots >= 0
    x, slots = x[keep], slots[keep].long()
    ids, at = torch.unique_consecutive(slots // BLOCK, return_inverse=True)
    row = slots % BLOCK
    n = ids.numel()
    a = x.new_zeros((n, HKV)).index_reduce_(0, at, x.abs().amax(-1), "amax")
    first = torch.full((n,), BLOCK, dtype=row.dtype, device=row.device).index_reduce_(0, at, row, "amin")
    old = torch.where(first[:, None] > 0, scales[ids], 0.0)
    new = torch.maximum(old, _scale_for(a, QMAX[fmt]))
    held = codes.view(torch.uint8)[ids].view(codes.dtype)
    moved = _encode(held.float() * (old / new)[:, :, None, None], fmt).view(torch.uint8)
    before = torch.arange(BLOCK, device=row.device)[None, :] < first[:, None]
    held = torch.where((before[:, None, :] & (new > old)[:, :, None])[..., None], moved, held.view(torch.uint8))
    codes.view(torch.uint8)[ids] = held
    codes.view(torch.uint8)[ids[at], :, row] = _encode(x / new[at][..., None], fmt).view(torch.uint8)
    scales[ids] = new


def _plain_append(s):
    _plain_quantise(_rope(s["k_new"], s["pos"]).float(), s["k"], s["k_scale"], s["slots"], s["format"])
    _plain_quantise(s["v_new"].float(), s["v"], s["v_scale"], s["slots"], s["format"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _unpaged(codes, scales, table):
    """Pool -> float32 [B, 8, S, 128] by the block table (entries of -1: block 0, masked later)."""
    ids = table.clamp(min=0).long()
    x = codes.view(torch.uint8)[ids].view(codes.dtype).float() * scales[ids][..., None, None]
    b, nb = ids.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, HKV, nb * BLOCK, D)


def _plain_attend(s):
    q, lens, cu = s["q"], s["lens"].long(), s["cu"].long()
    batch, t = lens.numel(), s["max_new"]
    news = cu[1:] - cu[:-1]
    step = torch.arange(t, device="cuda")
    real = step < news[:, None]                                              # [B, T]
    row = torch.where(real, cu[:-1, None] + step, 0)
    pos = torch.where(real, (lens - news)[:, None] + step, 0)
    qr = (_rope(q[row].reshape(batch * t, HQ, D), pos.reshape(-1)) / math.sqrt(D)).float()
    qr = qr.view(batch, t, HKV, GROUP, D).permute(0, 2, 3, 1, 4).reshape(batch, HKV, GROUP * t, D)
    k, v = (_unpaged(s[n], s[n + "_scale"], s["table"]) for n in ("k", "v"))
    key = torch.arange(k.shape[2], device="cuda")
    v = torch.where((key < lens[:, None])[:, None, :, None], v, 0.0)
    w = torch.matmul(qr, k.transpose(2, 3).contiguous()).view(batch, HKV, GROUP, t, -1)
    w = torch.where((key <= pos[..., None])[:, None, None], w, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(batch, HKV, GROUP * t, -1), v).view(batch, HKV, GROUP, t, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, t, HQ, D)
    seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(q.shape[0], device="cuda"), right=True)
    return o[seq, torch.arange(q.shape[0], device="cuda") - cu[seq]].to(torch.bfloat16)


# ---------------------------------------------------------------------------- the framework's calls


def _own_plan(s):
    import attention_accelerator_amd as gqa
    p = gqa.paged_plan(s["cached"], s["news"], s["free"], s["n_free"], s["table"], s["rows"])
    return {"table": s["table"], "seq_len": p.seq_len, "cu_new": p.cu_new, "slots": p.slot_map,
            "positions": p.positions, "n_free": p.n_free}


def _own_append(s):
    import attention_accelerator_amd as gqa
    pool = gqa.Q8Pool(s["k"], s["v"], s["k_scale"], s["v_scale"])
    gqa.kv_append_q8(s["k_new"], s["v_new"], pool, s["slots"], s["pos"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attend(s):
    import attention_accelerator_amd as gqa
    if s["call"][0] is None:
        pool = gqa.Q8Pool(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["call"][0] = gqa.PreparedAttentionQ8(s["q"], pool, s["table"], s["lens"], s["cu"], max_new=s["max_new"])
    return s["call"][0]()


def run(s):
    if own:
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend}[s["kind"]](s)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[s["kind"]](s)


# ---------------------------------------------------------------------------- float64


def _turn(x, pos):
    """RoPE of rows x [n, heads, 128] at pos by complex products in float64."""
    freq = torch.tensor([THETA ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos.double()[:, None] * freq)
    z = torch.complex(x[..., : D // 2].double(), x[..., D // 2:].double()) * turn[:, None, :]
    return torch.cat((z.real, z.imag), dim=-1)


def _nearest(x, fmt):
    """float64 values in code units -> the nearest value a code stands for (ties to even)."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(case, seed):
    """Codes and scales block by block, from a float64 picture of the pool."""
    s = _prepare_append(case, seed)
    fmt, slots = s["format"], s["slots"].tolist()
    got = {}
    runs, begin = [], 0
    for t in range(1, len(slots) + 1):
        if t == len(slots) or slots[t] // BLOCK != slots[begin] // BLOCK:
            if slots[begin] >= 0:
                runs.append((begin, t))
            begin = t
    for name, new in (("k", _turn(s["k_new"], s["pos"])), ("v", s["v_new"].double())):
        new = new.float().double()                      # rows enter as float32
        codes, scales = s[name].double(), s[name + "_scale"].double()
        for lo, hi in runs:
            blk, row = divmod(slots[lo], BLOCK)
            x = new[lo:hi]                              # [rows, 8, 128]
            a = x.abs().amax(dim=(0, 2))
            # the exponent by a logarithm, then put right where the logarithm was rounded
            e = torch.exp2(torch.ceil(torch.log2(a.clamp(min=1e-300) / QMAX[fmt])))
            e = torch.where(e * QMAX[fmt] < a, 2 * e, torch.where(e / 2 * QMAX[fmt] >= a, e / 2, e)).clamp(min=MIN_SCALE)
            if row:
                old = scales[blk]
                e = torch.maximum(old, e)
                held = codes[blk, :, :row]
                codes[blk, :, :row] = torch.where((e > old)[:, None, None],
                                                  _nearest(held * (old / e)[:, None, None], fmt), held)
            scales[blk] = e
            codes[blk, :, row:row + hi - lo] = _nearest(x / e[None, :, None], fmt).transpose(0, 1)
        got[name] = codes if fmt == "e4m3" else None    # int8 codes are whole numbers
        got[name + "_scale"] = scales
    return got


def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b, n in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        ids = s["table"][b, : _blocks(n)].long()
        pos = torch.arange(n - (hi - lo), n, device="cuda")
        q = _turn(s["q"][lo:hi], pos) / math.sqrt(D)                                  # [t, 32, 128]
        hidden = torch.arange(n, device="cuda")[None, :] > pos[:, None]
        for h in range(HKV):
            k, v = ((s[x].view(torch.uint8)[ids, h].view(s[x].dtype).double()
                     * s[x + "_scale"][ids, h].double()[:, None, None]).reshape(-1, D)[:n] for x in ("k", "v"))
            for g in range(GROUP):
                w = q[:, GROUP * h + g].contiguous() @ k.t().contiguous()
                out[lo:hi, GROUP * h + g] = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None                                     # whole numbers
    return _exact_append(case, seed) if case["kind"] == "append" else _exact_attend(case, seed)


def work(case):
    news = _news(case)
    lens = _lens(case, news)
    tokens = sum(news)
    if case["kind"] == "plan":
        fresh = sum(_blocks(c + n) - _blocks(c) for c, n in zip(lens, news))
        # lengths in and out, the table entry a sequence continues in, new entries, token rows
        return {"bytes": 4 * (4 * case["batch"] + 1 + case["batch"] + 2 * fresh + 2 * (tokens + case["pad"])),
                "flops": 0}
    row = HKV * D * 2                                   # one position's K and V codes over all KV heads
    if case["kind"] == "append":
        parts = sum(_blocks(c + n) - c // BLOCK for c, n in zip(lens, news) if n)
        return {"bytes": tokens * (2 * row + row + 8) + parts * HKV * 2 * 4, "flops": 6 * tokens * HKV * D}
    keys = sum(lens)
    blocks = sum(_blocks(n) for n in lens)
    seen = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(news, lens))
    return {"bytes": keys * row + blocks * (4 + HKV * 8) + tokens * HQ * D * 4, "flops": 4 * D * HQ * seen}
