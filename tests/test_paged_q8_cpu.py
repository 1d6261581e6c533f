"""The 8-bit paged cache's entry points without a GPU: what the C ABI and the Python surface refuse
before any launch, workspace sizes, and the plain forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import attention_accelerator_amd as gqa
from attention_accelerator_amd import _lib
from attention_accelerator_amd._lib import GqaParams, GqaQ8Kv
import _q8

OK, BAD_CFG, BAD_PTR, BAD_WS = 0, 1, 2, 3
A = 1 << 20                  # an aligned address that nothing follows: refused calls launch nothing


def params(**kw):
    p = dict(n_q_heads=32, n_kv_heads=8, head_dim=128, scale=1 / math.sqrt(128), rope_theta=500000.0, flags=0,
             stream_wgs=0)
    p.update(kw)
    return GqaParams(**p)


def layout(**kw):
    d = dict(block_stride=16384, head_stride=2048, pos_stride=128, scale_block_stride=8, scale_head_stride=1,
             block_size=16, max_blocks=4, n_blocks=10, format=1)
    d.update(kw)
    return GqaQ8Kv(**d)


def plan_call(**kw):
    d = dict(cached=A, n_new=2 * A, batch=2, free=3 * A, n_free=4 * A, free_capacity=8, table=5 * A, table_stride=4,
             max_blocks=4, n_rows=8, seq_len=6 * A, cu=7 * A, slots=8 * A, positions=9 * A, n_free_out=10 * A)
    d.update(kw)
    return _lib.lib().gqa_paged_plan(*d.values(), None)


@pytest.mark.parametrize("change,want", [
    (dict(batch=0), BAD_CFG), (dict(batch=-1), BAD_CFG), (dict(n_rows=-1), BAD_CFG), (dict(max_blocks=0), BAD_CFG),
    (dict(max_blocks=1 << 27, table_stride=1 << 27), BAD_CFG), (dict(table_stride=3), BAD_CFG),
    (dict(free_capacity=-1), BAD_CFG), (dict(cached=None), BAD_PTR), (dict(n_new=None), BAD_PTR),
    (dict(free=None), BAD_PTR), (dict(n_free=None), BAD_PTR), (dict(table=None), BAD_PTR),
    (dict(seq_len=None), BAD_PTR), (dict(cu=None), BAD_PTR), (dict(slots=None), BAD_PTR),
    (dict(positions=None), BAD_PTR), (dict(n_free_out=None), BAD_PTR), (dict(cached=A + 2), BAD_PTR),
    (dict(slots=8 * A + 1), BAD_PTR), (dict(seq_len=A), BAD_PTR), (dict(cu=2 * A), BAD_PTR),
    (dict(n_free_out=4 * A), BAD_PTR), (dict(slots=3 * A), BAD_PTR),
])
def test_plan_refusals(change, want):
    assert plan_call(**change) == want


def append_call(p=None, lay=None, **kw):
    d = dict(k_new=A, k_stride=1024, v_new=2 * A, v_stride=1024, k=3 * A, v=4 * A, ks=5 * A, vs=6 * A)
    tail = dict(slots=7 * A, positions=8 * A, n=4)
    d.update({k: v for k, v in kw.items() if k in d})
    tail.update({k: v for k, v in kw.items() if k in tail})
    p = params(flags=2) if p is None else p
    lay = layout() if lay is None else lay
    return _lib.lib().gqa_kv_append_q8(ctypes.byref(p), *d.values(), ctypes.byref(lay), *tail.values(), None)


def attend_call(p=None, lay=None, **kw):
    d = dict(q=A, stride=4096, k=3 * A, v=4 * A, ks=5 * A, vs=6 * A)
    tail = dict(table=7 * A, seq_len=8 * A, cu=9 * A, batch=2, n=4, max_new=2, out=10 * A, ws=11 * A, ws_bytes=1 << 40)
    d.update({k: v for k, v in kw.items() if k in d})
    tail.update({k: v for k, v in kw.items() if k in tail})
    p = params(flags=1) if p is None else p
    lay = layout() if lay is None else lay
    return _lib.lib().gqa_attention_q8(ctypes.byref(p), *d.values(), ctypes.byref(lay), *tail.values(), None)


BAD_LAYOUTS = [
    (dict(block_size=8), BAD_CFG), (dict(n_blocks=0), BAD_CFG), (dict(n_blocks=1 << 27), BAD_CFG),
    (dict(format=2), BAD_CFG), (dict(format=-1), BAD_CFG), (dict(pos_stride=64), BAD_CFG),
    (dict(pos_stride=1 << 27), BAD_CFG), (dict(head_stride=-16), BAD_CFG), (dict(block_stride=-16), BAD_CFG),
    (dict(scale_block_stride=-1), BAD_CFG), (dict(pos_stride=136), BAD_PTR), (dict(head_stride=2056), BAD_PTR),
    (dict(block_stride=16392), BAD_PTR),
]


@pytest.mark.parametrize("change,want", BAD_LAYOUTS)
@pytest.mark.parametrize("call", [append_call, attend_call])
def test_layout_refusals(call, change, want):
    assert call(lay=layout(**change)) == want


@pytest.mark.parametrize("change,want", [
    (dict(k_new=None), BAD_PTR), (dict(v_new=None), BAD_PTR), (dict(k=None), BAD_PTR), (dict(v=None), BAD_PTR),
    (dict(ks=None), BAD_PTR), (dict(vs=None), BAD_PTR), (dict(slots=None), BAD_PTR), (dict(positions=None), BAD_PTR),
    (dict(k_new=A + 2), BAD_PTR), (dict(v_new=2 * A + 4), BAD_PTR), (dict(k_stride=1026), BAD_PTR),
    (dict(v_stride=-4), BAD_CFG), (dict(n=-1), BAD_CFG), (dict(k=3 * A + 8), BAD_PTR), (dict(slots=7 * A + 2), BAD_PTR),
    (dict(n=0), OK),                                           # nothing to do
])
def test_append_refusals(change, want):
    assert append_call(**change) == want


@pytest.mark.parametrize("change", [dict(n_q_heads=31), dict(n_kv_heads=4), dict(head_dim=64), dict(scale=0.0),
                                    dict(flags=64), dict(flags=2, rope_theta=0.0), dict(stream_wgs=-1)])
def test_geometry_refusals(change):
    assert append_call(p=params(**change)) == BAD_CFG
    assert attend_call(p=params(**change)) == BAD_CFG


@pytest.mark.parametrize("change,want", [
    (dict(q=None), BAD_PTR), (dict(k=None), BAD_PTR), (dict(vs=None), BAD_PTR), (dict(table=None), BAD_PTR),
    (dict(seq_len=None), BAD_PTR), (dict(out=None), BAD_PTR), (dict(q=A + 8), BAD_PTR), (dict(stride=4100), BAD_PTR),
    (dict(stride=-8), BAD_CFG), (dict(out=10 * A + 4), BAD_PTR), (dict(batch=0), BAD_CFG), (dict(n=0), BAD_CFG),
    (dict(max_new=0), BAD_CFG), (dict(cu=None, batch=5), BAD_CFG), (dict(ws=None), BAD_WS), (dict(ws=11 * A + 128), BAD_WS),
    (dict(ws_bytes=1024), BAD_WS),
])
def test_attention_refusals(change, want):
    assert attend_call(**change) == want


def test_attention_refuses_rope_k_and_empty_tables():
    assert attend_call(p=params(flags=3)) == BAD_CFG
    assert attend_call(lay=layout(max_blocks=0)) == BAD_CFG
    assert attend_call(lay=layout(max_blocks=1 << 27)) == BAD_CFG


def test_workspace_sizes():
    size = gqa.attention_q8_workspace_bytes
    assert size(0, 1, 1) == 0 and size(1, 0, 1) == 0 and size(1, 1, 0) == 0
    # a size follows from max_new and the device: a call of more sequences or rows needs no more
    assert size(1, 1, 1) == size(500, 900, 1) > 0
    assert size(4, 64, 16) < size(4, 64, 17)
    assert size(1, 1, 1, gqa.make_params(stream_wgs=64)) < size(1, 1, 1, gqa.make_params(stream_wgs=1024))


def test_python_refuses_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        gqa.paged_plan(i, i, i, i[:1], torch.zeros((2, 4), dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        gqa.new_q8_pool(4, torch.float16, "cpu")
    pool = gqa.new_q8_pool(4, torch.int8, "cpu")
    x = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        gqa.kv_append_q8(x, x, pool, i, i)
    with pytest.raises(ValueError):
        gqa.gqa_attention_q8(torch.zeros((2, 32, 128), dtype=torch.bfloat16), pool, torch.zeros((2, 4), dtype=torch.int32), i)


# -- arrays that share a place

@pytest.mark.parametrize("change", [
    dict(cu=6 * A + 4), dict(slots=9 * A + 28), dict(n_free_out=8 * A + 12), dict(seq_len=A + 4), dict(positions=5 * A + 28),
    dict(free=5 * A - 4), dict(n_free=5 * A + 4), dict(table=3 * A + 28), dict(positions=8 * A - 4), dict(n_free_out=10 * A, cu=10 * A - 8),
])
def test_plan_refuses_shared_places(change):
    assert plan_call(**change) == BAD_PTR


@pytest.mark.parametrize("change", [
    dict(block_stride=0), dict(head_stride=0), dict(head_stride=128), dict(block_stride=8192), dict(pos_stride=2048),
    dict(scale_head_stride=0), dict(scale_block_stride=0), dict(scale_block_stride=7), dict(scale_block_stride=1, scale_head_stride=9),
    dict(block_stride=1 << 62, n_blocks=1 << 20),
])
def test_append_refuses_expanded_pools(change):
    assert append_call(lay=layout(**change)) == BAD_CFG


@pytest.mark.parametrize("change", [dict(k=4 * A), dict(ks=6 * A)])
def test_append_refuses_one_pool_for_both(change):
    assert append_call(**change) == BAD_PTR


@pytest.mark.parametrize("out", [A, A + 8192, A + 4 * 8192 - 8, A - 8])
def test_attention_refuses_out_over_q(out):
    assert attend_call(out=out) == BAD_PTR


def test_workspace_init_refusals():
    init = _lib.lib().gqa_attention_q8_workspace_init
    assert init(None, 1 << 30, None) == BAD_WS
    assert init(A + 128, 1 << 30, None) == BAD_WS
    assert init(A, 1024, None) == BAD_WS


def test_batches_beyond_the_counters():
    assert gqa.attention_q8_workspace_bytes(32769, 40000, 1) == 0 < gqa.attention_q8_workspace_bytes(32768, 40000, 1)
    assert attend_call(batch=32769, n=40000) == BAD_CFG


# -- the plain forms themselves, against torch's own conversions and written-out results

def test_plain_e4m3_rounds_as_torch():
    x = torch.cat((torch.linspace(-500, 500, 4001, dtype=torch.float64),
                   torch.tensor([2.0 ** e * m for e in range(-12, 9) for m in (1, 1.0625, 1.125, 1.1875, 1.4375)])))
    want = x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(_q8.nearest(x.float().double(), "e4m3"), want)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_plain_scale_is_the_smallest(fmt):
    top = _q8.QMAX[fmt]
    for a in (1e-30, 0.3, 1.0, top, top * 1.0001, top / 2, 3.0e38, 2.0 ** -140):
        s = _q8.scale_for(a, fmt)
        assert math.frexp(s)[0] == 0.5 and s * top >= a and (s == 2.0 ** -126 or s / 2 * top < a)


def test_plain_plan_by_hand():
    table, seq_len, cu, slots, pos, left = _q8.plan([15, 0, 16], [3, 17, 1], [9, 8, 7, 6], 4,
                                                    [[5, -1], [-1, -1], [4, -1]], 22)
    assert table == [[5, 6], [7, 8], [4, 9]] and seq_len == [18, 17, 17] and cu == [0, 3, 20, 21] and left == 0
    assert slots[:4] == [5 * 16 + 15, 6 * 16, 6 * 16 + 1, 7 * 16] and slots[19:] == [8 * 16, 9 * 16, -1]
    assert pos[:4] == [15, 16, 17, 0] and pos[19:] == [16, 16, 0]
    # the second request does not fit, the third needs a block too, a fourth does not
    _, seq_len, _, slots, _, left = _q8.plan([15, 0, 16, 1], [3, 17, 1, 1], [9, 8], 2,
                                             [[5, -1], [-1, -1], [4, -1], [3, -1]], 22)
    assert seq_len == [18, 0, 0, 2] and left == 1 and slots[3] == -1 and slots[21] == 3 * 16 + 1
