"""paged_plan, kv_append_q8 and gqa_attention_q8 against their plain 64-bit forms (tests/_q8.py).

Plan outputs, codes and scales have to be equal (their definition rounds, and both sides round the same
exact values).  Attention outputs stay within the bound that _q8.attend derives per element."""
from __future__ import annotations

import math
import random
import re

import pytest
import torch

import attention_accelerator_amd as gqa
from attention_accelerator_amd import _lib
from conftest import ROOT
import _q8

pytestmark = pytest.mark.gpu
FORMATS = ("int8", "e4m3")


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------------- plan


def run_plan(dev, cached, n_new, free, n_free, table, n_rows, out=None):
    t = i32(table, dev)
    p = gqa.paged_plan(i32(cached, dev), i32(n_new, dev), i32(free, dev), i32([n_free], dev), t, n_rows, out=out)
    return (t.tolist(), p.seq_len.tolist(), p.cu_new.tolist(), p.slot_map.tolist(), p.positions.tolist(),
            p.n_free.item())


def random_step(seed, batch, most_new, high, free_share=1.0, pad=0, odd=False):
    r = random.Random(seed)
    cached = [r.randint(0, high) for _ in range(batch)]
    n_new = [r.choice([0, 1, 1, r.randint(1, most_new)]) for _ in range(batch)]
    if odd:                                            # values that the plan has to refuse
        for b in r.sample(range(batch), max(1, batch // 8)):
            cached[b], n_new[b] = r.choice([(-1, 2), (3, -2), (2 ** 31 - 1, 1), (high, 2 ** 31 - 1), (high + 1, most_new * 16)])
    width = (high + most_new) // 16 + 2
    ids = list(range(sum(min(max(-(-c // 16), 0), width) for c in cached) + batch * width))
    r.shuffle(ids)
    table = []
    for c in cached:
        have = min(max(-(-c // 16), 0), width)
        table.append([ids.pop() for _ in range(have)] + [-1] * (width - have))
    need = sum(-(-(c + max(n, 0)) // 16) + -(-c // -16) for c, n in zip(cached, n_new) if 0 <= c <= high and 0 <= n <= most_new)
    n_free = int(need * free_share) + (4 if free_share >= 1 else 0)
    free = ids[:n_free + 3]
    rows = sum(n for n in n_new if 0 <= n <= most_new) + pad
    return cached, n_new, free, min(n_free, len(free)), table, rows


@pytest.mark.parametrize("batch,most_new,high,share,pad", [
    (1, 1, 0, 1.0, 0), (1, 40, 33, 1.0, 3), (7, 20, 100, 1.0, 0), (64, 1, 500, 1.0, 5), (63, 90, 200, 0.5, 0),
    (300, 33, 64, 0.9, 100), (1024, 2, 40, 1.0, 0), (1025, 5, 40, 0.7, 1), (2500, 3, 17, 1.0, 2000), (3, 5000, 50, 1.0, 7),
])
def test_plan_matches_plain(dev, batch, most_new, high, share, pad):
    step = random_step(batch * 31 + high, batch, most_new, high, share, pad)
    got, want = run_plan(dev, *step), _q8.plan(*step)
    for name, g, w in zip(("table", "seq_len", "cu", "slots", "positions", "n_free"), got, want):
        assert g == w, name


@pytest.mark.parametrize("batch", [8, 70, 1100])
def test_plan_refuses_odd_requests(dev, batch):
    """Negative values, values near 2^31, requests past the table: refused whole, the others as
    ever (their rows count, so rows behind them may not fit)."""
    step = random_step(batch, batch, 9, 100, 1.0, 50, odd=True)
    got, want = run_plan(dev, *step), _q8.plan(*step)
    assert got[1] == want[1] and got[0] == want[0] and got[3:] == want[3:]
    assert got[2] == [min(c, 2 ** 31 - 1) for c in want[2]]


def test_plan_empty_step(dev):
    """No rows at all: every request rests; and a stack that says more than it holds."""
    got = run_plan(dev, [5, 0, 16], [0, 0, 0], [1, 2], 7, [[3, -1], [-1, -1], [4, -1]], 0)
    assert got == ([[3, -1], [-1, -1], [4, -1]], [5, 0, 16], [0, 0, 0, 0], [], [], 2)
    got = run_plan(dev, [5], [1], [1], -4, [[3, -1]], 1)
    assert got == ([[3, -1]], [6], [0, 1], [3 * 16 + 5], [5], 0)


def test_plan_rows_do_not_fit(dev):
    step = ([0, 16, 3], [5, 4, 1], [9, 8, 7], 3, [[-1, -1], [5, -1], [6, -1]], 7)
    assert run_plan(dev, *step) == tuple(_q8.plan(*step))
    assert run_plan(dev, *step)[1] == [5, 0, 0]


def test_plan_wide_table_and_strides(dev):
    """A table that is a view of a wider one: the entries beside it stay."""
    wide = torch.full((3, 9), -7, dtype=torch.int32, device=dev)
    table = wide[:, 2:6]
    table.fill_(-1)
    p = gqa.paged_plan(i32([0, 0, 0], dev), i32([20, 0, 64], dev), i32([3, 4, 5, 6, 7, 8, 9], dev), i32([7], dev), table, 84)
    assert p.seq_len.tolist() == [20, 0, 64] and p.n_free.item() == 1
    assert table.tolist() == [[9, 8, -1, -1], [-1] * 4, [7, 6, 5, 4]]
    assert (wide[:, :2] == -7).all() and (wide[:, 6:] == -7).all()


def test_plan_python_refusals(dev):
    a, f, n, t = i32([1, 2], dev), i32([3], dev), i32([1], dev), i32([[0, 1], [2, 3]], dev)
    with pytest.raises(ValueError):
        gqa.paged_plan(a.long(), a, f, n, t, 4)
    with pytest.raises(ValueError):
        gqa.paged_plan(a, a[:1], f, n, t, 4)
    with pytest.raises(ValueError):
        gqa.paged_plan(a, a, f, n, t.t(), 4)
    with pytest.raises(ValueError):
        gqa.paged_plan(a, a, f, n, t[:1], 4)
    out = gqa.paged_plan(a, a, f, n, t, 4)
    with pytest.raises(ValueError):
        gqa.paged_plan(a, a, f, n, t, 4, out=out._replace(seq_len=a))
    with pytest.raises(ValueError):
        gqa.paged_plan(a, a, f, n, t, 5, out=out)
    with pytest.raises(gqa.GqaConfigError):
        gqa.paged_plan(a[:0], a[:0], f, n, t[:0], 4)


# ----------------------------------------------------------------------------------------- append


def random_pool(n_blocks, fmt, gen, spread=1):
    k, v = (torch.randn((n_blocks, 8, 16, 128), generator=gen) * (30 if fmt == "int8" else 90) for _ in range(2))
    k, v = ((x.round().clamp(-127, 127) if fmt == "int8" else x.clamp(-448, 448)).to(_q8.DTYPES[fmt]) for x in (k, v))
    ks, vs = (torch.exp2(torch.randint(-spread, spread + 1, (n_blocks, 8), generator=gen).float()) / 64 for _ in range(2))
    return [k, v, ks, vs]


def to_dev(pool, dev):
    return gqa.Q8Pool(*(t.view(torch.uint8).to(dev).view(t.dtype) if t.dtype != torch.float32 else t.to(dev) for t in pool))


def check_append(dev, pool, k_new, v_new, slots, pos, fmt, rope_k=True, device_rows=None):
    """Runs the append on a copy of the pool and compares every code and scale."""
    p = to_dev(pool, dev)
    kd, vd = device_rows or (k_new.to(dev), v_new.to(dev))
    gqa.kv_append_q8(kd, vd, p, i32(slots, dev), i32(pos, dev) if rope_k else None, rope_k=rope_k)
    rows = (_q8.rope(k_new, pos) if rope_k else k_new.double()).float().double(), v_new.double()
    for name, x, codes, scales, gc, gs in zip("kv", rows, pool[:2], pool[2:], p[:2], p[2:]):
        c, s = _q8.codes64(codes), scales.double().clone()
        _q8.append(c, s, x, slots, fmt)
        assert torch.equal(gs.cpu().double().nan_to_num(7.25), s.nan_to_num(7.25)), name + "_scale"
        g = _q8.codes64(gc)
        assert torch.equal(g.isnan(), c.isnan()), name
        assert torch.equal(g.nan_to_num(0.0), c.nan_to_num(0.0)), name


def runs_to_slots(runs):
    """[(block, first row, rows)] -> slots."""
    return [16 * b + r + i for b, r, n in runs for i in range(n)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("runs", [
    [(2, 0, 1)], [(2, 5, 1)], [(2, 15, 1)], [(3, 0, 16)], [(3, 4, 12), (1, 0, 16), (0, 0, 3)],
    [(i, (5 * i) % 16, 1) for i in range(9)], [(0, 13, 3), (1, 0, 16), (2, 0, 16), (3, 0, 1), (4, 7, 9), (5, 0, 11)],
])
def test_append_matches_plain(dev, fmt, runs):
    gen = torch.Generator().manual_seed(len(runs) * 7 + runs[0][1])
    pool = random_pool(10, fmt, gen, spread=3)
    slots = runs_to_slots(runs)
    x = [torch.randn((len(slots), 8, 128), generator=gen).to(torch.bfloat16) for _ in range(2)]
    # rows of very different sizes, so that blocks keep their scale, grow a little and grow much
    x[0] *= torch.exp2(torch.randint(-4, 5, (len(slots), 8, 1), generator=gen).float()).to(torch.bfloat16)
    x[1] *= torch.exp2(torch.randint(-4, 5, (len(slots), 8, 1), generator=gen).float()).to(torch.bfloat16)
    pos = [random.Random(3).randint(0, 200000) + t for t in range(len(slots))]
    check_append(dev, pool, x[0], x[1], slots, pos, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_many_ragged_runs(dev, fmt):
    r = random.Random(11)
    runs = []
    for b in r.sample(range(130), 130):
        first = r.choice([0, 0, r.randint(0, 15)])
        runs.append((b, first, r.randint(1, 16 - first)))
    slots = runs_to_slots(runs)
    for t in sorted(r.sample(range(len(slots)), 20)):
        slots.insert(t, r.choice([-1, -5, 130 * 16, 2 ** 31 - 1]))          # skipped tokens
    gen = torch.Generator().manual_seed(5)
    pool = random_pool(130, fmt, gen, spread=6)
    k, v = (torch.randn((len(slots), 8, 128), generator=gen).to(torch.bfloat16) for _ in range(2))
    check_append(dev, pool, k, v, slots, list(range(len(slots))), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_fused_rows_and_no_rope(dev, fmt):
    """K and V as slices of a fused projection's rows, a pool whose strides are not the natural ones, a
    misaligned slice (copied by the call), and no rotation."""
    gen = torch.Generator().manual_seed(9)
    qkv = torch.randn((37, 48, 128), generator=gen).to(torch.bfloat16)
    slots = runs_to_slots([(1, 3, 13), (0, 0, 16), (4, 0, 8)])
    dq = qkv.to(dev)
    pool = random_pool(6, fmt, gen)
    check_append(dev, pool, qkv[:, 32:40], qkv[:, 40:], slots, None, fmt, rope_k=False, device_rows=(dq[:, 32:40], dq[:, 40:]))
    flat = torch.zeros(37 * 1024 + 1, dtype=torch.bfloat16, device=dev)
    odd = flat[1:].view(37, 8, 128)
    odd.copy_(dq[:, 32:40])
    check_append(dev, pool, qkv[:, 32:40], qkv[:, 40:], slots, None, fmt, rope_k=False, device_rows=(odd, dq[:, 40:]))
    big = torch.zeros((6, 16, 10, 256), dtype=torch.uint8, device=dev).view(_q8.DTYPES[fmt])
    k, v = (b.permute(0, 2, 1, 3)[:, 1:9, :, 128:] for b in (big, big.clone()))
    ks, vs = (torch.zeros((8, 6), device=dev).t() for _ in range(2))
    gqa.kv_append_q8(dq[:, 32:40], dq[:, 40:], gqa.Q8Pool(k, v, ks, vs), i32(slots, dev), rope_k=False)
    c, s = torch.zeros((6, 8, 16, 128), dtype=torch.float64), torch.zeros((6, 8), dtype=torch.float64)
    _q8.append(c, s, qkv[:, 40:].double(), slots, fmt)
    assert torch.equal(_q8.codes64(v.contiguous()), c) and torch.equal(vs.cpu().double(), s)
    assert (big.view(torch.uint8)[..., :128] == 0).all() and (big.view(torch.uint8)[:, :, 0] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_extreme_values(dev, fmt):
    """Zero rows, subnormal and huge ones, infinities and NaN; present scales of 0, NaN, infinity, below
    zero and no power of two."""
    inf, nan = math.inf, math.nan
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((12, 8, 128), generator=gen)
    x[0] = 0.0
    x[1] *= 1e-40
    x[2] *= 1e37
    x[3, :, 5], x[3, :, 70] = inf, -inf
    x[4, :, 9] = nan
    x[5] = nan
    x[6] = inf
    x[7, 0] = torch.where(torch.arange(128) % 2 == 0, 127.0, 448.0)         # border of a power of two
    x[7, 1] = torch.where(torch.arange(128) % 2 == 0, 127.5, 449.0)
    x = x.to(torch.bfloat16)
    pool = random_pool(12, fmt, gen)
    for blk, s in zip(range(6, 12), (0.0, nan, inf, -1.0, 0.013, 2.0 ** -126)):
        pool[2][blk] = pool[3][blk] = s
    slots = [16 * b + (0 if b < 6 else 7) for b in range(12)]
    check_append(dev, pool, x, x.flip(2), slots, None, fmt, rope_k=False)


@pytest.mark.parametrize("fmt", FORMATS)
def test_append_token_by_token(dev, fmt):
    """A block filled one row at a time, its scale growing at several of them; what the codes stand
    for stays within one quantum (int8) or half an e4m3 step plus half a subnormal step."""
    gen = torch.Generator().manual_seed(4)
    v = (torch.randn((16, 8, 128), generator=gen) * torch.exp2(torch.arange(16) / 3.0)[:, None, None]).to(torch.bfloat16)
    pool = gqa.new_q8_pool(2, _q8.DTYPES[fmt], dev)
    c, s = torch.zeros((2, 8, 16, 128), dtype=torch.float64), torch.zeros((2, 8), dtype=torch.float64)
    for t in range(16):
        row = v[t:t + 1].to(dev)
        gqa.kv_append_q8(row, row, pool, i32([16 + t], dev), rope_k=False)
        _q8.append(c, s, v[t:t + 1].double(), [16 + t], fmt)
    assert torch.equal(_q8.codes64(pool.v), c) and torch.equal(pool.v_scale.cpu().double(), s)
    assert torch.equal(pool.k.view(torch.uint8), pool.v.view(torch.uint8))
    off = (c[1] * s[1][:, None, None] - v.double().transpose(0, 1)).abs()
    quantum = s[1][:, None, None]
    step = v.double().transpose(0, 1).abs() * 2.0 ** -4
    # e4m3: its own rounding, and each of at most log2(growth) moves half a subnormal step (2^-10 s')
    # in units that double: less than 2^-9 of the last one's
    assert (off <= (quantum if fmt == "int8" else torch.maximum(step, quantum * 2.0 ** -10) + quantum * 2.0 ** -9)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("gaps", [(0, 20, 40), (3, 530, 1500), (700, 15, 513), (1100, 1, 2000)])
def test_append_long_stretches_of_skipped_tokens(dev, fmt, gaps):
    """Tokens of one block far apart, and skipped ones before and behind them."""
    slots = [-1] * gaps[0] + [19, 20] + [-1] * gaps[1] + [21, 47] + [-1] * gaps[1] + [54, 55] + [-1] * gaps[2]
    gen = torch.Generator().manual_seed(sum(gaps))
    pool = random_pool(4, fmt, gen, spread=4)
    k, v = (torch.randn((len(slots), 8, 128), generator=gen).to(torch.bfloat16) for _ in range(2))
    check_append(dev, pool, k, v, slots, list(range(len(slots))), fmt)


def test_append_nothing(dev):
    pool = gqa.new_q8_pool(2, torch.int8, dev)
    x = torch.zeros((0, 8, 128), dtype=torch.bfloat16, device=dev)
    gqa.kv_append_q8(x, x, pool, i32([], dev), i32([], dev))
    x = torch.ones((3, 8, 128), dtype=torch.bfloat16, device=dev)
    gqa.kv_append_q8(x, x, pool, i32([-1, -1, 32], dev), i32([0, 1, 2], dev))
    assert (pool.k == 0).all() and (pool.k_scale == 0).all() and (pool.v_scale == 0).all()


# -------------------------------------------------------------------------------------- attention


def make_batch(fmt, news, lens, seed, q_scale=1.0, spread=1, spare=2):
    """A shuffled pool holding random rows, stale codes (NaN ones too) behind each sequence's end."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // 16) for n in lens]
    pool = random_pool(sum(need) + spare, fmt, gen, spread)
    ids = torch.randperm(sum(need) + spare, generator=gen).tolist()
    table = []
    for n in need:
        table.append([ids.pop() for _ in range(n)] + [-1] * (max(need) - n))
    for b, n in enumerate(lens):
        if n % 16:
            for codes in pool[:2]:
                codes.view(torch.uint8)[table[b][n // 16], :, n % 16:] = 127
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    q = (torch.randn((cu[-1], 32, 128), generator=gen) * q_scale).to(torch.bfloat16)
    return q, pool, table, cu


def run_attention(dev, q, pool, table, lens, cu, **kw):
    return gqa.gqa_attention_q8(q.to(dev), to_dev(pool, dev), i32(table, dev), i32(lens, dev), i32(cu, dev), **kw).cpu()


def assert_close(got, want, bound, what=""):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    over = ((got - want).abs() - bound).nan_to_num(0.0)
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} elements beyond their bound, the worst by {over.max():.3g}"


BATCHES = [
    # new tokens and lengths of each sequence
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [31]), ([1], [33]), ([1], [700]), ([1, 1, 1], [5, 64, 129]),
    ([2], [2]), ([4, 1, 3], [4, 90, 35]), ([5], [300]), ([8, 1, 7, 2], [8, 65, 40, 100]), ([9], [9]), ([16, 3], [16, 200]),
    ([13, 16, 1], [400, 45, 1]),
    ([17], [17]), ([64], [64]), ([65], [200]), ([100, 1, 33], [100, 77, 161]), ([1, 18, 16, 2], [300, 90, 16, 2]),
    ([130], [601]),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("news,lens", BATCHES)
def test_attention_matches_plain(dev, fmt, news, lens):
    q, pool, table, cu = make_batch(fmt, news, lens, seed=sum(lens) + len(lens))
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news))
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    assert_close(got, want, bound, f"{fmt} {news} {lens}")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("stream_wgs", [4, 64])
def test_attention_few_workgroups(dev, fmt, stream_wgs):
    """Ranges that cover several sequences and heads, and tiles that share a workgroup in turn."""
    news, lens = [1, 3, 40, 1, 16, 70, 1], [3, 70, 45, 130, 48, 90, 400]
    q, pool, table, cu = make_batch(fmt, news, lens, seed=77)
    p = gqa.make_params(stream_wgs=stream_wgs)
    got = run_attention(dev, q, pool, table, lens, cu, max_new=70, params=p)
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    assert_close(got, want, bound, "few workgroups")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("news,lens", [([1, 1], [900, 300]), ([3], [500]), ([40], [520])])
def test_attention_sharp_scores_and_scale_spread(dev, fmt, news, lens):
    """A peaked softmax (Q x 16), block scales spread over 2^24, and a scale of the caller's."""
    q, pool, table, cu = make_batch(fmt, news, lens, seed=5, q_scale=16.0)
    pool[3] *= torch.exp2(torch.randint(-12, 13, pool[3].shape, generator=torch.Generator().manual_seed(1)).float())
    c = [_q8.codes64(t) for t in pool[:2]]
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news))
    assert_close(got, *_q8.attend(q, c[0], c[1], pool[2], pool[3], table, lens, cu), "sharp")
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news), scale=0.01, rope_q=False)
    assert_close(got, *_q8.attend(q, c[0], c[1], pool[2], pool[3], table, lens, cu, scale=0.01, rope_q=False), "own scale")


@pytest.mark.parametrize("news,lens", [([1, 1], [200, 90]), ([2], [66]), ([40], [200])])
def test_attention_zero_values(dev, news, lens):
    """V scales of 0 and 2^-126 (blocks of zero rows): their keys still count in the softmax; all of
    them so: a zero row."""
    q, pool, table, cu = make_batch("int8", news, lens, seed=8)
    pool[3][::2] = 0.0
    pool[3][1::4] = 2.0 ** -126
    c = [_q8.codes64(t) for t in pool[:2]]
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news))
    assert_close(got, *_q8.attend(q, c[0], c[1], pool[2], pool[3], table, lens, cu), "zero scales")
    pool[3][:] = 0.0
    assert (run_attention(dev, q, pool, table, lens, cu, max_new=max(news)) == 0).all()


@pytest.mark.parametrize("news,lens", [([3], [21]), ([16], [40]), ([24], [50]), ([70, 2], [70, 18])])
def test_attention_nan_in_unseen_keys(dev, news, lens):
    """NaN codes in K and V of a sequence's last token reach its row alone; one dimension's NaN in V
    reaches that dimension of the rows that see its key."""
    q, pool, table, cu = make_batch("e4m3", news, lens, seed=12)
    for b, n in enumerate(lens):
        pool[0].view(torch.uint8)[table[b][(n - 1) // 16], 3, (n - 1) % 16, 7] = 127
        pool[1].view(torch.uint8)[table[b][(n - 1) // 16], 5, (n - 1) % 16] = 255
        if n > 2:
            pool[1].view(torch.uint8)[table[b][(n - 2) // 16], 6, (n - 2) % 16, 100] = 127
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news))
    assert_close(got, want, bound.nan_to_num(0.0), "nan")
    assert got.isnan().any() and not got.isnan().all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_bad_lengths_and_blocks(dev, fmt):
    """Lengths that break the rules give NaN rows, ids outside the pool NaN rows for those that read
    them, offsets that break the rules nothing; the other sequences and the rows behind stay."""
    news, lens = [1, 2, 1, 20, 3, 1], [40, 50, 33, 60, 35, 20]
    q, pool, table, cu = make_batch(fmt, news, lens, seed=3)
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    lens = list(lens)
    lens[0] = 16 * len(table[0]) + 1                   # past the table
    lens[1] = 1                                        # fewer positions than rows
    table[4][2] = 999                                  # read by rows at positions 32 .. 34 only
    want[cu[0]:cu[2]] = math.nan
    want[cu[4]:cu[5]] = math.nan
    out = torch.full((q.shape[0] + 3, 32, 128), 7.0, dtype=torch.bfloat16, device=dev)
    more = torch.cat((q, q[:3]))
    got = run_attention(dev, more, pool, table, lens, cu, max_new=20, out=out)
    assert (got[q.shape[0]:] == 7.0).all()
    assert_close(got[:q.shape[0]], want, bound, "bad entries")
    table[4][2] = -1
    assert_close(run_attention(dev, q, pool, table, lens, cu, max_new=20), want, bound, "negative id")
    # more rows than max_new: NaN rows for that sequence; offsets that break the rules: nothing
    got = run_attention(dev, q, pool, table, lens, cu, max_new=4)
    assert got[cu[3]:cu[4]].isnan().all() and not got[cu[5]:].isnan().any()
    out = torch.full((q.shape[0], 32, 128), 7.0, dtype=torch.bfloat16, device=dev)
    for bad in ([-1, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5, q.shape[0] + 1]):
        at = 0 if bad[0] < 0 else 5
        got = run_attention(dev, q, pool, [t for t in table], [40, 50, 33, 60, 35, 20], bad, max_new=4, out=out.clone())
        row = got[0 if at == 0 else 5]
        assert (row == 7.0).all()


def test_attention_scale_not_a_number(dev):
    q, pool, table, cu = make_batch("int8", [1, 1], [40, 40], seed=6)
    pool[2][table[0][1], 2] = math.nan
    pool[3][table[1][0], 5] = -0.5
    got = run_attention(dev, q, pool, table, [40, 40], cu, max_new=1)
    assert got[0, 8:12].isnan().all() and got[1, 20:24].isnan().all()
    assert int(got.isnan().any(-1).sum()) == 8


def test_attention_strides_and_default_arguments(dev):
    """Q as a slice of a fused projection's rows, a pool of other strides, one row per sequence without
    cu_new, and a workspace and output of the caller's."""
    q, pool, table, cu = make_batch("e4m3", [1, 1, 1], [50, 18, 77], seed=21)
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, [50, 18, 77], cu)
    p = to_dev(pool, dev)
    fused = torch.zeros((3, 48, 128), dtype=torch.bfloat16, device=dev)
    fused[:, :32] = q.to(dev)
    wide = [t.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(t.dtype) for t in p[:2]]
    scales = [t.t().contiguous().t() for t in p[2:]]
    ws = gqa.new_attention_q8_workspace(3, 3, 1, dev)
    out = torch.empty((3, 32, 128), dtype=torch.bfloat16, device=dev)
    got = gqa.gqa_attention_q8(fused[:, :32], gqa.Q8Pool(*wide, *scales), i32(table, dev), i32([50, 18, 77], dev),
                               workspace=ws, out=out)
    assert got is out
    assert_close(got.cpu(), want, bound, "strides")
    assert_close(run_attention(dev, q, pool, table, [50, 18, 77], cu), want, bound, "default max_new")
    with pytest.raises(ValueError):
        gqa.gqa_attention_q8(q.to(dev), p, i32(table, dev), i32([50, 18], dev))
    with pytest.raises(ValueError):
        gqa.gqa_attention_q8(q.to(dev), p, i32(table, dev), i32([50, 18, 77], dev), workspace=ws[:1000])
    with pytest.raises(ValueError):
        gqa.gqa_attention_q8(q.to(dev), p._replace(v=p.k.view(torch.int8)), i32(table, dev), i32([50, 18, 77], dev))
    with pytest.raises(gqa.GqaConfigError):
        gqa.gqa_attention_q8(q[:, :16].to(dev), p, i32(table, dev), i32([50, 18, 77], dev))


def test_attention_on_another_stream_and_repeats(dev):
    """Two calls at once on two streams with a workspace each give what one gives, every time."""
    calls, wants = [], []
    for seed, (news, lens) in enumerate([([1, 2], [300, 500]), ([30, 1], [400, 90])]):
        q, pool, table, cu = make_batch("int8", news, lens, seed=seed)
        args = (q.to(dev), to_dev(pool, dev), i32(table, dev), i32(lens, dev), i32(cu, dev))
        calls.append(gqa.PreparedAttentionQ8(*args, max_new=max(news)))
        wants.append(gqa.gqa_attention_q8(*args, max_new=max(news)).clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c in calls:
            c.out.zero_()
        torch.cuda.synchronize()
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c()
        torch.cuda.synchronize()
        for c, w in zip(calls, wants):
            assert torch.equal(c.out, w)


@pytest.mark.parametrize("news,lens,stream_wgs", [
    ([1, 1], [5003, 3100], 0), ([1, 1], [5003, 3100], 16), ([7], [4111], 16), ([2, 16], [2500, 1999], 16),
    ([100], [4500], 16), ([33], [6001], 0),
])
@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_long_ranges(dev, fmt, news, lens, stream_wgs):
    """Ranges and runs of many steps: block ids and scales come in several batches."""
    q, pool, table, cu = make_batch(fmt, news, lens, seed=lens[0])
    got = run_attention(dev, q, pool, table, lens, cu, max_new=max(news), params=gqa.make_params(stream_wgs=stream_wgs))
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    assert_close(got, want, bound, f"{fmt} {news} {lens}")


@pytest.mark.parametrize("most", [1, 2, 20])
def test_attention_many_sequences(dev, most):
    """More sequences than a wave has lanes, some of them empty or without new rows, one odd one."""
    r = random.Random(most)
    news = [r.choice([0, 1, 1, r.randint(1, most)]) if most > 1 else 1 for _ in range(150)]
    lens = [n + r.choice([0, 3, r.randint(0, 70), r.randint(0, 260)]) for n in news]
    q, pool, table, cu = make_batch("int8", news, lens, seed=most)
    bad = news.index(max(news), 70)
    lens[bad] = news[bad] - 1
    got = run_attention(dev, q, pool, table, lens, cu, max_new=most)
    assert got[cu[bad]:cu[bad + 1]].isnan().all()
    lens[bad] = news[bad]
    want, bound = _q8.attend(q, _q8.codes64(pool[0]), _q8.codes64(pool[1]), pool[2], pool[3], table, lens, cu)
    keep = [t for t in range(cu[-1]) if not cu[bad] <= t < cu[bad + 1]]
    assert_close(got[keep], want[keep], bound[keep], str(most))


@pytest.mark.parametrize("most", [1, 700])
def test_attention_refused_sequences(dev, most):
    """Refused sequences (length 0) of one and of many rows between others: NaN rows, all of them, and no other."""
    news = [most, 1, most, 1, 1] if most > 1 else [1] * 200
    lens = [0, 40, 0, 0, 25] if most > 1 else [33 * (b % 3 == 1) for b in range(200)]
    q, pool, table, cu = make_batch("int8", news, [max(n, m) for n, m in zip(news, lens)], seed=most)
    out = torch.full((cu[-1] + 2, 32, 128), 5.0, dtype=torch.bfloat16, device=dev)
    q = torch.cat((q, q[:2]))
    gqa.gqa_attention_q8(q.to(dev), to_dev(pool, dev), i32(table, dev), i32(lens, dev), i32(cu, dev), max_new=most, out=out)
    for b, n in enumerate(lens):
        assert out[cu[b]:cu[b + 1]].isnan().all() if n == 0 else out[cu[b]:cu[b + 1]].isfinite().all(), b
    assert (out[cu[-1]:] == 5).all()


def test_attention_one_workspace_for_all(dev):
    """Calls of every kind in turn on one workspace, and rows behind the last sequence."""
    batches = [([1, 1, 1], [700, 40, 1300]), ([40, 1], [900, 33]), ([8, 3], [500, 777]), ([1], [3000]), ([1] * 70, [90] * 70)]
    ws = gqa.new_attention_q8_workspace(70, 200, 64, dev)
    calls = []
    for i, (news, lens) in enumerate(batches):
        q, pool, table, cu = make_batch("e4m3", news, lens, seed=40 + i)
        q = torch.cat((q, torch.full((3, 32, 128), float("nan"), dtype=torch.bfloat16)))
        out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device=dev)
        args = (q.to(dev), to_dev(pool, dev), i32(table, dev), i32(lens, dev), i32(cu, dev))
        calls.append((gqa.PreparedAttentionQ8(*args, max_new=max(news), workspace=ws, out=out), cu[-1],
                      gqa.gqa_attention_q8(*args, max_new=max(news))[:cu[-1]].clone()))
    for turn in range(3):
        for call, rows, want in calls[turn:] + calls[:turn]:
            call.out[:rows] = 0
            assert torch.equal(call()[:rows], want) and (call.out[rows:] == 5).all()


def test_attention_mixed_step_graph_replays(dev):
    """A mixed step captured with its workspace made inside, replayed with new values and eager calls between."""
    news, lens = [40, 1, 7, 1], [300, 500, 90, 64]
    q, pool, table, cu = make_batch("int8", news, lens, seed=9)
    gen = torch.Generator().manual_seed(10)
    args = [q.to(dev), to_dev(pool, dev), i32(table, dev), i32(lens, dev), i32(cu, dev)]
    gqa.gqa_attention_q8(*args, max_new=40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gqa.gqa_attention_q8(*args, max_new=40)
    for turn in range(5):
        args[0].copy_(torch.randn(q.shape, generator=gen).to(torch.bfloat16))
        args[3].copy_(i32([n - 3 * turn for n in lens], dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gqa.gqa_attention_q8(*args, max_new=40))


# ------------------------------------------------------------------------------------ a serving run


@pytest.mark.parametrize("fmt", FORMATS)
def test_serving_steps(dev, fmt):
    """Plan, append and attend together over steps of prompts, decodes and drafts, from an empty pool:
    the pool's codes equal the plain form's, the outputs lie within their bounds."""
    gen = torch.Generator().manual_seed(31)
    n_blocks, width, batch = 40, 10, 4
    pool = gqa.new_q8_pool(n_blocks, _q8.DTYPES[fmt], dev)
    plain = [torch.zeros((n_blocks, 8, 16, 128), dtype=torch.float64) for _ in range(2)]
    scales = [torch.zeros((n_blocks, 8), dtype=torch.float64) for _ in range(2)]
    free = i32(torch.randperm(n_blocks, generator=gen).tolist(), dev)
    n_free = i32([n_blocks], dev)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
    cached = torch.zeros(batch, dtype=torch.int32, device=dev)
    for news in ([37, 0, 5, 1], [1, 20, 1, 1], [1, 1, 3, 1], [1, 1, 1, 40], [2, 0, 1, 1]):
        rows = sum(news) + 2
        qkv = torch.randn((rows, 48, 128), generator=gen).to(torch.bfloat16)
        d = qkv.to(dev)
        before = cached.tolist(), free.tolist(), n_free.item(), table.tolist()
        plan = gqa.paged_plan(cached, i32(news, dev), free, n_free, table, rows)
        gqa.kv_append_q8(d[:, 32:40], d[:, 40:], pool, plan.slot_map, plan.positions)
        out = gqa.gqa_attention_q8(d[:, :32], pool, table, plan.seq_len, plan.cu_new, max_new=max(news))
        t, lens, cu, slots, pos, left = _q8.plan(before[0], news, before[1], before[2], before[3], rows)
        assert plan.slot_map.tolist() == slots and plan.seq_len.tolist() == lens and plan.n_free.item() == left
        _q8.append(plain[0], scales[0], _q8.rope(qkv[:, 32:40], pos).float().double(), slots, fmt)
        _q8.append(plain[1], scales[1], qkv[:, 40:].double(), slots, fmt)
        for got, want in zip((pool.k, pool.v), plain):
            assert torch.equal(_q8.codes64(got), want)
        for got, want in zip((pool.k_scale, pool.v_scale), scales):
            assert torch.equal(got.cpu().double(), want)
        want, bound = _q8.attend(qkv[:, :32], plain[0], plain[1], scales[0], scales[1], t, lens, cu)
        assert_close(out.cpu()[:cu[-1]], want[:cu[-1]], bound[:cu[-1]], str(news))
        cached, n_free = plan.seq_len, plan.n_free


def test_documented_ctypes_step(dev):
    """The ctypes stub that the integration document gives for a step, run as written, against the
    package's tensor calls, bit for bit."""
    text = (ROOT / "INTEGRATION.md").read_text()
    stub = [re.search(r"```python\n(.*?)```", text[text.index(s):], flags=re.S).group(1) for s in ("## 2.", "## 8.")]
    src = "\n".join(stub).replace('"/path/to/attention_accelerator_amd/libgqa.so"', repr(str(_lib.LIB_PATH)))
    ns: dict = {}
    exec(compile(src, "INTEGRATION.md", "exec"), ns)
    gen = torch.Generator().manual_seed(8)
    ours, theirs = (gqa.new_q8_pool(30, torch.int8, dev) for _ in range(2))
    tables = [torch.full((3, 6), -1, dtype=torch.int32, device=dev) for _ in range(2)]
    free, n_free, cached = i32(list(range(30)), dev), i32([30], dev), i32([0, 0, 0], dev)
    ws = gqa.new_attention_q8_workspace(3, 60, 40, dev)
    for news in ([40, 3, 1], [1, 1, 1], [17, 2, 0]):
        qkv = torch.randn((sum(news), 48, 128), generator=gen).to(torch.bfloat16).to(dev)
        plan = gqa.paged_plan(cached, i32(news, dev), free, n_free, tables[0], sum(news))
        gqa.kv_append_q8(qkv[:, 32:40], qkv[:, 40:], ours, plan.slot_map, plan.positions)
        want = gqa.gqa_attention_q8(qkv[:, :32], ours, tables[0], plan.seq_len, plan.cu_new, max_new=max(news))
        out, lens, left = ns["serving_step"](qkv, *theirs, tables[1], cached, i32(news, dev), free, n_free, max(news), ws)
        assert torch.equal(out, want) and torch.equal(lens, plan.seq_len) and torch.equal(left, plan.n_free)
        assert torch.equal(theirs.k, ours.k) and torch.equal(theirs.v_scale, ours.v_scale)
        cached, n_free = lens, left


def test_serving_step_graph_replays(dev):
    """A captured decode step (plan, append, attend, lengths and stack advanced in the graph) replayed
    over block borders, with eager work between, equals the eager steps."""
    def fresh():
        g = torch.Generator("cuda").manual_seed(3)
        st = {"pool": gqa.new_q8_pool(24, torch.float8_e4m3fn, dev), "table": torch.full((3, 8), -1, dtype=torch.int32, device=dev),
              "free": torch.arange(24, dtype=torch.int32, device=dev).flip(0).contiguous(), "n_free": i32([24], dev),
              "cached": i32([0, 0, 0], dev), "qkv": torch.zeros((4, 48, 128), dtype=torch.bfloat16, device=dev),
              "one": i32([1, 1, 1], dev), "gen": g}
        st["plan"] = gqa.paged_plan(st["cached"], st["one"], st["free"], i32([0], dev), st["table"], 4)
        st["attend"] = gqa.PreparedAttentionQ8(st["qkv"][:, :32], st["pool"], st["table"], st["plan"].seq_len,
                                               st["plan"].cu_new, max_new=1)
        return st

    def step(st):
        p = gqa.paged_plan(st["cached"], st["one"], st["free"], st["n_free"], st["table"], 4, out=st["plan"])
        gqa.kv_append_q8(st["qkv"][:, 32:40], st["qkv"][:, 40:], st["pool"], p.slot_map, p.positions)
        out = st["attend"]()
        st["cached"].copy_(p.seq_len)
        st["n_free"].copy_(p.n_free)
        return out

    eager, graphed = fresh(), fresh()
    warm = fresh()
    step(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed)
    for _ in range(37):
        for st in (eager, graphed):
            st["qkv"].copy_(torch.randn(st["qkv"].shape, generator=st["gen"], device=dev).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out[:3], want[:3])
        assert torch.equal(graphed["pool"].k.view(torch.uint8), eager["pool"].k.view(torch.uint8))
        assert graphed["cached"].tolist() == eager["cached"].tolist() and graphed["n_free"].item() == eager["n_free"].item()
    assert eager["cached"].tolist() == [37, 37, 37] and eager["n_free"].item() == 15
