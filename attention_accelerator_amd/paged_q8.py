"""A serving step over an 8-bit paged cache: block plan, quantising append, ragged attention.

paged_plan makes a step's block table entries, slots and positions on the GPU from the requests'
lengths; kv_append_q8 puts the step's new K (rotated) and V rows into their slots; gqa_attention_q8
attends from the step's query rows: single tokens, drafts and prompt chunks in one ragged batch.
A pool keeps one byte an element and a float scale for each (block of 16 positions, KV head).

Every op runs the HIP kernels of libgqa.so on the current torch stream of its tensors' device;
there is no CPU path.  Tensors of a call lie on one device.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import GQA_Q8_E4M3, GQA_Q8_INT8, GqaParams, GqaQ8Kv, check, lib
from .attention import BLOCK_SIZE, HEAD_DIM, N_KV_HEADS, N_Q_HEADS, ROPE_THETA, make_params

Q8_FORMATS = {torch.int8: GQA_Q8_INT8, torch.float8_e4m3fn: GQA_Q8_E4M3}


def _call(fn, device: torch.device, *args) -> int:
    """fn(*args, the current stream of `device`) with that device current.  (The raw handle: a
    torch.cuda.Stream object for it takes 2 us, a small call's kernel 5.)"""
    index = device.index
    if torch.cuda.current_device() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


class Q8Pool(NamedTuple):
    """An 8-bit pool: k, v [n_blocks, 8, 16, 128] int8 or float8_e4m3fn (any strides, multiples of
    16, with contiguous rows), k_scale, v_scale [n_blocks, 8] float32; an element stands for
    code * scale.  k and v share dtype, shape and strides, the scales shape and strides."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new_q8_pool(n_blocks: int, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> Q8Pool:
    """A zeroed pool of n_blocks blocks."""
    if dtype not in Q8_FORMATS:
        raise ValueError("an 8-bit pool is int8 or float8_e4m3fn")
    shape = (int(n_blocks), N_KV_HEADS, BLOCK_SIZE, HEAD_DIM)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return Q8Pool(k, v, ks, vs)


class PagedPlan(NamedTuple):
    """What paged_plan makes: seq_len [B], cu_new [B + 1], slot_map and positions [n_rows],
    n_free [1], all int32 on the device."""

    seq_len: torch.Tensor
    cu_new: torch.Tensor
    slot_map: torch.Tensor
    positions: torch.Tensor
    n_free: torch.Tensor


def _int32(t: torch.Tensor, name: str, device, numel: Optional[int] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on the GPU")
    if device is not None and t.device != device:
        raise ValueError(f"{name} lies on {t.device}, the other tensors on {device}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} entries, {numel} expected")
    return t


def _table(t: torch.Tensor, device, batch: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype != torch.int32 or not t.is_cuda or t.device != device:
        raise ValueError("block_table must be an int32 [B, max_blocks] tensor on the other tensors' device")
    if t.shape[0] != batch:
        raise ValueError("block_table has one row per sequence")
    return t


def _span(t: torch.Tensor):
    """The addresses that an int32 tensor's elements lie in: [first, end)."""
    start = t.data_ptr()
    if t.is_contiguous():
        return start, start + 4 * t.numel()
    return start, start + 4 * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))


def paged_plan(cached: torch.Tensor, n_new: torch.Tensor, free_blocks: torch.Tensor, n_free: torch.Tensor,
               block_table: torch.Tensor, n_rows: int, *, out: Optional[PagedPlan] = None) -> PagedPlan:
    """Block table entries, slots, positions and lengths of a step, from the requests' lengths.

    cached, n_new  [B] int32: positions in the cache, and new tokens of this step (0: at rest)
    free_blocks    int32 stack of free block ids, n_free [1] of them valid: ids are taken from the
                   top (the highest index)
    block_table    [B, max_blocks] int32 (rows contiguous), new blocks' entries written in place
    n_rows         token rows of the step, at least n_new's sum (more: padded rows)
    out            a PagedPlan to write into (for captured graphs); no tensor of it may overlap an
                   input or another one
    Returns the lengths with the new tokens (0: refused), the ragged row offsets, each row's slot (-1:
    refused or padding) and position, and what is left of the stack.  A request is granted whole or
    refused whole, first come, first served; refused are those the stack does not cover, and
    those whose positions or rows do not fit the table or n_rows."""
    _int32(cached, "cached", None)
    device, batch = cached.device, cached.numel()
    _int32(n_new, "n_new", device, batch)
    _int32(free_blocks, "free_blocks", device)
    _int32(n_free, "n_free", device, 1)
    _table(block_table, device, batch)
    if block_table.stride(1) != 1 or block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table rows must be contiguous and not overlap")
    n_rows = int(n_rows)
    sizes = (batch, batch + 1, n_rows, n_rows, 1)
    if out is None:
        if n_rows < 0 or batch == 0:
            check(_lib.GQA_ERR_INVALID_CONFIG, "gqa_paged_plan")
        # (one allocation; the unsafe split keeps no record for autograd, which integers have no use for)
        out = PagedPlan(*torch.empty(sum(sizes), dtype=torch.int32, device=device).unsafe_split_with_sizes(sizes))
    else:
        inputs = [_span(t) for t in (cached, n_new, free_blocks, n_free, block_table)]
        for t, n, name in zip(out, sizes, PagedPlan._fields):
            lo = _int32(t, name, device, n).data_ptr()
            hi = lo + 4 * n
            for first, end in inputs:
                if lo < end and first < hi:
                    raise ValueError(f"out.{name} overlaps an input")
    status = _call(lib().gqa_paged_plan, device, cached.data_ptr(), n_new.data_ptr(), batch, free_blocks.data_ptr(),
                   n_free.data_ptr(), free_blocks.numel(), block_table.data_ptr(), block_table.stride(0),
                   block_table.shape[1], n_rows, *[t.data_ptr() for t in out])
    check(status, "gqa_paged_plan")
    return out


def _q8_layout(pool: Q8Pool, device, max_blocks: int = 1) -> GqaQ8Kv:
    k, v, ks, vs = pool
    shape, strides, dtype = k.shape, k.stride(), k.dtype
    if len(shape) != 4 or v.shape != shape or v.stride() != strides or v.dtype != dtype:
        raise ValueError("k and v of a pool must share dtype, shape [n_blocks,8,16,128] and strides")
    fmt = Q8_FORMATS.get(dtype)
    if fmt is None:
        raise ValueError("an 8-bit pool is int8 or float8_e4m3fn")
    n_blocks, heads, rows, dims = shape
    if heads != N_KV_HEADS or rows != BLOCK_SIZE or dims != HEAD_DIM:
        raise ValueError(f"pools hold {N_KV_HEADS} KV heads of {BLOCK_SIZE} rows of {HEAD_DIM} dimensions per block")
    if strides[3] != 1:
        raise ValueError("pool rows must be contiguous in head_dim")
    scale_strides = ks.stride()
    if ks.shape != shape[:2] or vs.shape != shape[:2] or vs.stride() != scale_strides \
            or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise ValueError("k_scale and v_scale must be float32 [n_blocks, 8] with the same strides")
    if not k.device == v.device == ks.device == vs.device == device:
        raise ValueError("a pool's tensors must be on the GPU, on the other tensors' device")
    return GqaQ8Kv(strides[0], strides[1], strides[2], scale_strides[0], scale_strides[1], BLOCK_SIZE, max_blocks,
                   n_blocks, fmt)


def _rows(t: torch.Tensor, name: str, heads: int, align: int, copy: bool = True) -> torch.Tensor:
    """[N, heads, 128] bfloat16 whose tokens may lie apart (a slice of a fused projection), each one's
    heads together; copied (or refused) where the kernels cannot take it as it lies."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.dtype != torch.bfloat16 or not t.is_cuda:
        raise ValueError(f"{name} must be a bfloat16 [N, {heads}, 128] tensor on the GPU")
    n, h, d = t.shape
    if h != heads or d != HEAD_DIM:
        raise _lib.GqaConfigError(_lib.GQA_ERR_INVALID_CONFIG, f"{name} of {h} heads of {d}")
    token, head, dim = t.stride()
    if dim != 1 or head != HEAD_DIM or token < 0 or (2 * token | t.data_ptr()) % align:
        if not copy:
            raise ValueError(f"{name}: each token's heads must lie together, tokens {align} bytes aligned")
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def kv_append_q8(k_new: torch.Tensor, v_new: torch.Tensor, pool: Q8Pool, slot_map: torch.Tensor,
                 positions: Optional[torch.Tensor] = None, *, rope_k: bool = True, theta: float = ROPE_THETA) -> None:
    """Write k_new / v_new [N, 8, 128] bfloat16 into the pool's slots, K rotated at its position
    (rope_k), quantised with one scale for each (block, KV head).

    slot_map   [N] int32: 16 * block + row, -1 skips the token (paged_plan's slot_map)
    positions  [N] int32 (may be None without rope_k)
    A block's scale is a power of two that covers its rows; where a row appended behind others needs a
    larger one, the rows before it are requantised.  The tokens of one block have to follow each
    other in the call, row after row (skipped ones aside), each slot at most once, and no two sequences may append to one block."""
    k_new, v_new = _rows(k_new, "k_new", N_KV_HEADS, 8), _rows(v_new, "v_new", N_KV_HEADS, 8)
    n, device = k_new.shape[0], k_new.device
    if v_new.shape[0] != n or v_new.device != device:
        raise ValueError("k_new and v_new must have the same tokens on the same device")
    layout = _q8_layout(pool, device)
    _int32(slot_map, "slot_map", device, n)
    if positions is not None:
        _int32(positions, "positions", device, n)
    elif rope_k:
        raise ValueError("rope_k needs positions")
    p = make_params(rope_q=False, rope_k=rope_k, theta=theta)
    status = _call(lib().gqa_kv_append_q8, device, ctypes.byref(p), k_new.data_ptr(), k_new.stride(0),
                   v_new.data_ptr(), v_new.stride(0), *[t.data_ptr() for t in pool], ctypes.byref(layout),
                   slot_map.data_ptr(), None if positions is None else positions.data_ptr(), n)
    check(status, "gqa_kv_append_q8")


def attention_q8_workspace_bytes(batch: int, n_tokens: int, max_new: int, params: Optional[GqaParams] = None) -> int:
    p = params or make_params()
    return int(lib().gqa_attention_q8_workspace_bytes(ctypes.byref(p), int(batch), int(n_tokens), int(max_new)))


def new_attention_q8_workspace(batch: int, n_tokens: int, max_new: int, device="cuda",
                               params: Optional[GqaParams] = None) -> torch.Tensor:
    """A workspace for gqa_attention_q8 calls of at most these sizes, its counters cleared on the
    current stream.  Calls that share it must be ordered (one stream)."""
    device = torch.empty(0, device=device).device              # ("cuda": the current one)
    with torch.cuda.device(device):
        nbytes = attention_q8_workspace_bytes(batch, n_tokens, max_new, params)
    if nbytes == 0:
        check(_lib.GQA_ERR_INVALID_CONFIG, "gqa_attention_q8_workspace_bytes")
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    check(_call(lib().gqa_attention_q8_workspace_init, device, workspace.data_ptr(), nbytes),
          "gqa_attention_q8_workspace_init")
    return workspace


class PreparedAttentionQ8:
    """A gqa_attention_q8 call with every argument bound once, for loops that repeat the same step
    (the tensors' values may change between calls): calling it issues the launches on the current
    stream with no checks or allocation.  The tensors passed in must stay alive while it is used.
    Its workspace is its own, cleared on the stream it is made on: that and the calls of one object
    must be ordered (one stream, or events)."""

    def __init__(self, q: torch.Tensor, pool: Q8Pool, block_table: torch.Tensor, seq_len: torch.Tensor,
                 cu_new: Optional[torch.Tensor] = None, *, max_new: Optional[int] = None, rope_q: bool = True,
                 theta: float = ROPE_THETA, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, params: Optional[GqaParams] = None):
        q = _rows(q, "q", N_Q_HEADS, 16, copy=False)
        device, n = q.device, q.shape[0]
        _int32(seq_len, "seq_len", device)
        batch = seq_len.numel()
        _table(block_table, device, batch)
        if not block_table.is_contiguous():
            raise ValueError("block_table must be contiguous")
        layout = _q8_layout(pool, device, block_table.shape[1])
        if cu_new is not None:
            _int32(cu_new, "cu_new", device, batch + 1)
        elif n != batch:
            raise ValueError(f"without cu_new q has one row per sequence: {n} rows for {batch} sequences")
        max_new = (n if cu_new is not None else 1) if max_new is None else int(max_new)
        p = params or make_params(rope_q=rope_q, rope_k=False, theta=theta, scale=scale)
        if workspace is None:
            workspace = new_attention_q8_workspace(batch, n, max_new, device, p)
        with torch.cuda.device(device):
            nbytes = attention_q8_workspace_bytes(batch, n, max_new, p)
        if nbytes == 0:
            check(_lib.GQA_ERR_INVALID_CONFIG, "gqa_attention_q8_workspace_bytes")
        if workspace.device != device or not workspace.is_contiguous() \
                or workspace.numel() * workspace.element_size() < nbytes:
            raise ValueError(f"workspace must be contiguous, on {device}, of {nbytes} bytes at least")
        if out is None:
            out = torch.empty((n, N_Q_HEADS, HEAD_DIM), dtype=torch.bfloat16, device=device)
        elif out.shape != (n, N_Q_HEADS, HEAD_DIM) or out.dtype != torch.bfloat16 or not out.is_contiguous() \
                or out.device != device:
            raise ValueError("out must be a contiguous bfloat16 [N,32,128] tensor on q's device")
        self.out, self.workspace, self.params, self.layout, self.device = out, workspace, p, layout, device
        self._keep = (q, pool, block_table, seq_len, cu_new)
        self._args = (ctypes.byref(p), q.data_ptr(), q.stride(0), *(t.data_ptr() for t in pool), ctypes.byref(layout),
                      block_table.data_ptr(), seq_len.data_ptr(), None if cu_new is None else cu_new.data_ptr(), batch, n,
                      max_new, out.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size())
        self._fn = lib().gqa_attention_q8

    def __call__(self) -> torch.Tensor:
        status = _call(self._fn, self.device, *self._args)
        if status:
            check(status, "gqa_attention_q8")
        return self.out


def gqa_attention_q8(q: torch.Tensor, pool: Q8Pool, block_table: torch.Tensor, seq_len: torch.Tensor,
                     cu_new: Optional[torch.Tensor] = None, *, max_new: Optional[int] = None, rope_q: bool = True,
                     theta: float = ROPE_THETA, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None, params: Optional[GqaParams] = None) -> torch.Tensor:
    """Ragged causal GQA attention over an 8-bit paged cache.

    q            [N, 32, 128] bfloat16: the query rows of all sequences one after the other
    block_table  [B, max_blocks] int32, seq_len [B] int32 on the device: positions in the cache, the
                 new ones among them (append first)
    cu_new       [B + 1] int32: sequence b has rows cu_new[b] .. cu_new[b+1] - 1, its last positions
                 (None: one row each)
    max_new      a bound on a sequence's rows (a host value; default: N).  Up to 16 rows take the
                 streamed kernel; a tight bound keeps idle launches out
    workspace    from new_attention_q8_workspace, for calls up to its sizes (else one is made for the call);
                 calls that share it must be ordered
    out          may not overlap q
    Returns out [N, 32, 128]; rows behind cu_new[B] are left as they were in `out`."""
    q = _rows(q, "q", N_Q_HEADS, 16)
    if isinstance(block_table, torch.Tensor):
        block_table = block_table.contiguous()
    return PreparedAttentionQ8(q, pool, block_table, seq_len, cu_new, max_new=max_new, rope_q=rope_q, theta=theta,
                               scale=scale, out=out, workspace=workspace, params=params)()
