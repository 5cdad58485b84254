"""An appendable paged KV cache: the tables of a step, new keys and values, and
the pages that a query should read.

A pool of pages holds keys and values of all sequences, (num_blocks,
page_block_size, Hkv, D) bf16 each, as `attention.flash_attn_with_kvcache_dense`
reads them with a block table.  One decode or prefill step is

    plan = plan_paged_step(seqlens, new_lens, block_table, free_pages, num_free, page, max_tokens)
    for every layer:
        append_paged_kv(k, v, k_cache, v_cache, plan.slots, page_bounds)
        pages = select_kv_pages(q, page_bounds, block_table, plan.seqlens, page, top_k)
        out = attention.flash_attn_with_kvcache_sparse(q, k_cache, v_cache, block_table, pages, plan.seqlens)

and the next one goes on with `plan.seqlens` and `plan.num_free`.  Nothing waits
for the GPU, so a step can be captured into a HIP graph; every call has its own
outputs and workspace.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

from ._lib import check, lib
from .codec import _dptr, _stream, _torch


def _here(t):
    """The index of t's device and its current stream, which a call goes to; None
    where another device is the current one."""
    torch = _torch()
    device = t.get_device()
    if device != torch.cuda.current_device():
        return None
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return device, _stream() if raw is None else raw(device)


_MOST = 2 ** 31 - 1  # of a number that goes to the library as a C int (which takes others modulo 2^32)


def _whole(n, name):
    """n as a whole number that a C int holds."""
    n = int(n)
    if not -_MOST <= n <= _MOST:
        raise ValueError(f"{name} must be less than 2^31, got {n}")
    return n


def _check(t, name, dtype, shape, device=None, contiguous=True):
    """Raises where t is not a GPU tensor of these (shape: None where any size that
    a C int holds will do; device: its index)."""
    try:  # (a right tensor takes 0.4 us)
        if t.dtype is dtype and (t.is_cuda if device is None else t.get_device() == device) and \
                (not contiguous or t.is_contiguous()):
            got = t.shape
            if got == shape:
                return
            if len(got) == len(shape):
                for n, m in zip(shape, got):
                    if m > _MOST if n is None else n != m:
                        break
                else:
                    return
    except AttributeError:
        pass
    torch = _torch()
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.shape and max(t.shape) > _MOST:
        raise ValueError(f"{name} must have less than 2^31 entries a dimension, got {tuple(t.shape)}")
    want = ", ".join("*" if n is None else str(n) for n in shape)
    raise ValueError(f"{name} must be ({want}), got {tuple(t.shape)}")


def _rows(t):
    """t (rows, heads, dim) and its strides as the kernels take it: 16-byte pieces
    of contiguous heads at any stride between rows and heads (a slice of a fused
    projection is one), a copy otherwise."""
    s0, s1, s2 = t.stride()
    if s2 != 1 or s0 % 8 or s1 % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=_torch().contiguous_format)
        s0, s1, _ = t.stride()
    return t, s0, s1


def _table(block_table, batch, device):
    """A block table that is read, its row stride and its width."""
    _check(block_table, "block_table", _torch().int32, (batch, None), device, contiguous=False)
    width = block_table.shape[1]
    s0, s1 = block_table.stride()
    if s0 < width or (s1 != 1 and width > 1):
        block_table = block_table.contiguous()
        s0 = max(width, 1)
    return block_table, s0, width


def _lengths(cache_seqlens, batch, device):
    torch = _torch()
    if isinstance(cache_seqlens, int):
        return torch.full((batch,), cache_seqlens, dtype=torch.int32, device=f"cuda:{device}")
    _check(cache_seqlens, "cache_seqlens", torch.int32, (batch,), device)
    return cache_seqlens


def _query(q):
    """(B, 1, H, D) or (B, H, D) -> (B, H, D)."""
    torch = _torch()
    if isinstance(q, torch.Tensor):
        if q.dim() == 4 and q.shape[1] == 1:
            q = q[:, 0]
        if q.dtype is torch.bfloat16 and q.is_cuda and q.dim() == 3 and q.shape[0] <= _MOST and q.shape[1] <= _MOST:
            return q
    _check(q, "q", torch.bfloat16, (None, None, None), contiguous=False)
    return q


def _new_like(q, shape):
    """A contiguous tensor of q's type and place (empty_like takes two thirds of
    the time of empty)."""
    torch = _torch()
    return torch.empty_like(q) if q.shape == shape and q.is_contiguous() else q.new_empty(shape)


@functools.lru_cache(maxsize=4096)
def _bytes(query, *sizes):
    """What a workspace query answers."""
    return int(getattr(lib(), query)(*sizes))


@dataclass(slots=True)
class QuantizedKVCache:
    """A pool of pages held in 4 or 8 bits, as `quantized_kv_cache` makes it: for
    every (page, KV head) page_block_size times 8 bytes with a token's (scale,
    low) of the key and of the value in bf16, then the tokens' rows of key codes,
    then those of value codes; a value is low + code * scale.  (include/zipserv.h
    has the order of the codes.)"""
    data: object         # uint8 (num_blocks, Hkv, page_block_size * (8 + head_dim * bits / 4))
    page_block_size: int
    head_dim: int
    bits: int


@dataclass
class PagedPlan:
    """One step's tables (all int32 on the GPU)."""
    slots: object       # [max_tokens] slot of each new token, -1 without one
    sequences: object   # [max_tokens] its sequence, -1 behind the last token
    positions: object   # [max_tokens] its place in the sequence, -1 behind the last
    seqlens: object     # [batch] cached tokens after the step: the context's and the new ones with a slot
    cu_new: object      # [batch + 1] each sequence's first token of the step
    counts: object      # [4] tokens asked for, pages taken, missing, left

    @property
    def num_free(self):
        """Free pages after the step, [1]: what the next step takes."""
        return self.counts[3:]


def plan_paged_step(context_lens, new_lens, block_table, free_pages, num_free, page_block_size: int,
                    max_tokens: int) -> PagedPlan:
    """The tables of one step from its requests' lengths, on the GPU: sequence b
    has context_lens[b] tokens in its pages and brings new_lens[b] more (int32
    [B], B <= 4096).  New pages come off the end of free_pages[:num_free] (int32,
    num_free [1]) in the order of the sequences and are entered into block_table
    (B, max_blocks) in place.  max_tokens is the size of the step's buffers: new
    tokens past it are left out, entries behind the last one are -1.

    Where pages run out (or a row of the table is full) the tokens that would
    need them get slot -1, and seqlens and counts say so: counts[0] against
    cu_new[-1] shows tokens left out, counts[2] the pages missing.  The context's
    own pages are taken to be in the table: a context that is longer than its row,
    or a negative entry among its pages, is not reported (new tokens there get slot
    -1 and count in seqlens all the same)."""
    torch = _torch()
    i32 = torch.int32
    _check(context_lens, "context_lens", i32, (None,))
    here = _here(context_lens)
    if here is None:
        with torch.cuda.device(context_lens.device):
            return plan_paged_step(context_lens, new_lens, block_table, free_pages, num_free, page_block_size,
                                   max_tokens)
    device, stream = here
    batch = context_lens.shape[0]
    _check(new_lens, "new_lens", i32, (batch,), device)
    _check(block_table, "block_table", i32, (batch, None), device, contiguous=False)
    width = block_table.shape[1]
    stride, inner = block_table.stride()
    if batch == 1:
        stride = max(width, 1)
    if (inner != 1 and width > 1) or stride < width:
        raise ValueError("block_table is written in place: its rows must be contiguous and apart")
    _check(free_pages, "free_pages", i32, (None,), device)
    _check(num_free, "num_free", i32, (1,), device)
    page, most = _whole(page_block_size, "page_block_size"), _whole(max_tokens, "max_tokens")
    if most < 0:
        raise ValueError("max_tokens must not be negative")
    out = torch.empty(3 * most + 2 * batch + 5, dtype=i32, device=context_lens.device)
    at = out.data_ptr()
    check("zs_paged_plan", lib().zs_paged_plan(
        stream, context_lens.data_ptr(), new_lens.data_ptr(), batch, block_table.data_ptr(), stride, width,
        free_pages.data_ptr(), free_pages.shape[0], num_free.data_ptr(), page, most, at,
        at + 4 * most, at + 8 * most, at + 12 * most, at + 12 * most + 4 * batch, at + 12 * most + 8 * batch + 4))
    return PagedPlan(*torch.split_with_sizes(out, (most, most, most, batch, batch + 1, 4)))


def append_paged_kv(k, v, k_cache, v_cache, slots, page_bounds=None) -> None:
    """New keys and values (tokens, Hkv, D) bf16 into their slots (int32
    [tokens], `PagedPlan.slots`; slots outside the pool are skipped).  k and v may
    be slices of a fused projection's output.  page_bounds (num_blocks, Hkv, 2,
    D) bf16, if given, is brought up to date: the smallest and the largest key of
    each channel in the pages written to, NaNs passed over; a page's bounds start
    anew with the token at its offset 0, so they need no first fill.  The tokens
    of one page stand next to one another, as a plan puts them, and no slot
    occurs twice."""
    torch = _torch()
    bf16 = torch.bfloat16
    _check(k_cache, "k_cache", bf16, (None, None, None, None))
    here = _here(k_cache)
    if here is None:
        with torch.cuda.device(k_cache.device):
            return append_paged_kv(k, v, k_cache, v_cache, slots, page_bounds)
    device, stream = here
    blocks, page, heads_k, dim = size = k_cache.shape
    _check(v_cache, "v_cache", bf16, size, device)
    _check(slots, "slots", torch.int32, (None,), device)
    n = slots.shape[0]
    _check(k, "k", bf16, (n, heads_k, dim), device, contiguous=False)
    _check(v, "v", bf16, (n, heads_k, dim), device, contiguous=False)
    if page_bounds is not None:
        _check(page_bounds, "page_bounds", bf16, (blocks, heads_k, 2, dim), device)
    k, k0, k1 = _rows(k)
    v, v0, v1 = _rows(v)
    check("zs_paged_append", lib().zs_paged_append(
        stream, k.data_ptr(), v.data_ptr(), k0, k1, v0, v1, slots.data_ptr(), n, k_cache.data_ptr(),
        v_cache.data_ptr(), _dptr(page_bounds), blocks, page, heads_k, dim))


def select_kv_pages(q, page_bounds, block_table, cache_seqlens, page_block_size: int, top_k: int,
                    sink_pages: int = 1, local_pages: int = 1):
    """The pages that each query's attention should read: (B, Hkv, top_k) int32
    logical pages in ascending order, -1 behind.  q: (B, 1, H, D) or (B, H, D)
    bf16; page_bounds as `append_paged_kv` keeps them; cache_seqlens: int32 [B] or
    an int.

    A page scores the largest q.k that its bounds allow, the most over the heads
    that share the KV head (in 64 bits, so the selection is the definition's;
    scores that are no number count as +inf).  The first sink_pages and the last
    local_pages of a sequence are always taken, the others by score, ties to the
    lowest page; sequences of at most top_k pages keep them all.

    Rows that fp32 cannot settle cost 25 to 50 times as much, as one workgroup
    scores all of their pages in 64 bits (0.25 ms for 2000 pages, 0.8 ms for 8000):
    those with a key that is not finite or a table entry outside the pool among
    their pages, queries with values past 2^60 or (0 aside) below 2^-126, and more than
    4096 pages that score the same (a query or a cache of zeros)."""
    torch = _torch()
    q = _query(q)
    here = _here(q)
    if here is None:
        with torch.cuda.device(q.device):
            return select_kv_pages(q, page_bounds, block_table, cache_seqlens, page_block_size, top_k, sink_pages,
                                   local_pages)
    device, stream = here
    batch, heads, dim = q.shape
    _check(page_bounds, "page_bounds", torch.bfloat16, (None, None, 2, dim), device)
    blocks, heads_k = page_bounds.shape[:2]
    table, row, width = _table(block_table, batch, device)
    lens = _lengths(cache_seqlens, batch, device)
    page, top_k = _whole(page_block_size, "page_block_size"), _whole(top_k, "top_k")
    sink, local = int(sink_pages), int(local_pages)  # (not below 0, and top_k at most together)
    if top_k <= 0 or sink < 0 or local < 0 or sink + local > top_k:
        raise ValueError("top_k must be positive and hold sink_pages and local_pages")
    if heads_k == 0 or heads % heads_k:
        raise ValueError(f"{heads} query heads do not share {heads_k} KV heads evenly")
    q, q0, q1 = _rows(q)
    at = q.device
    pages = torch.empty((batch, heads_k, top_k), dtype=torch.int32, device=at)
    need = _bytes("zs_select_kv_pages_workspace_bytes", batch, heads_k, width)
    ws = torch.empty(need, dtype=torch.uint8, device=at)
    check("zs_select_kv_pages", lib().zs_select_kv_pages(
        stream, q.data_ptr(), q0, q1, page_bounds.data_ptr(), blocks, page, table.data_ptr(),
        row, width, lens.data_ptr(), batch, heads, heads_k, dim, top_k, sink, local, pages.data_ptr(),
        ws.data_ptr(), need))
    return pages


def quantized_kv_cache(num_blocks: int, page_block_size: int, num_heads_k: int, head_dim: int, bits: int = 4,
                       device="cuda") -> QuantizedKVCache:
    """An empty pool of num_blocks pages held in `bits` (4 or 8) bits; head_dim 64
    or 128, pages a multiple of 16 tokens.  With head_dim 128 a token's key and
    value of one KV head take 136 (264) bytes where bf16 takes 512."""
    torch = _torch()
    if bits not in (4, 8) or head_dim not in (64, 128):
        raise ValueError(f"a cache of {bits} bits and head_dim {head_dim}: bits must be 4 or 8, head_dim 64 or 128")
    if page_block_size <= 0 or page_block_size % 16:
        raise ValueError(f"page_block_size must be a positive multiple of 16, got {page_block_size}")
    record = page_block_size * (8 + head_dim * bits // 4)
    data = torch.empty(num_blocks, num_heads_k, record, dtype=torch.uint8, device=device)
    return QuantizedKVCache(data, page_block_size, head_dim, bits)


def _quantized(cache):
    """A QuantizedKVCache's numbers as the library takes them: address, num_blocks,
    page, Hkv, head_dim, bits."""
    if type(cache) is not QuantizedKVCache:
        raise ValueError("cache must be a QuantizedKVCache")
    data, page, dim, bits = cache.data, cache.page_block_size, cache.head_dim, cache.bits
    try:  # (a right one takes 1 us)
        blocks, heads_k, record = data.shape
        if data.is_cuda and data.is_contiguous() and data.dtype is _torch().uint8 and \
                record == page * (8 + dim * bits // 4) and 0 < record <= _MOST and blocks <= _MOST and \
                heads_k <= _MOST and (bits == 4 or bits == 8):
            return data.data_ptr(), blocks, page, heads_k, dim, bits
    except (AttributeError, TypeError, ValueError):
        pass
    if not (isinstance(page, int) and isinstance(dim, int) and page > 0 and dim > 0 and bits in (4, 8)):
        raise ValueError("cache: page_block_size, head_dim or bits is wrong")
    _check(data, "cache.data", _torch().uint8, (None, None, page * (8 + dim * bits // 4)))
    raise ValueError(f"cache: pages of {page} tokens of {dim} channels are too large")


def append_paged_kv_quantized(k, v, cache: QuantizedKVCache, slots) -> None:
    """New keys and values (tokens, Hkv, D) bf16 quantised into their slots of a
    cache held in 4 or 8 bits (slots: int32 [tokens], `PagedPlan.slots`; those
    outside the pool are skipped, none occurs twice).  k and v may be slices of a
    fused projection's output.

    Of a token's row x of one KV head: low = min x, scale = the least bf16 with (2^bits
    - 1) scale >= max x - low, code = (x - low) / scale to the nearest, the even
    one of two; both differences rounded to fp32.  So a value comes back half a
    scale off at most.  A row with a value that is not finite is stored as NaNs."""
    torch = _torch()
    data, blocks, page, heads_k, dim, bits = _quantized(cache)
    here = _here(cache.data)
    if here is None:
        with torch.cuda.device(cache.data.device):
            return append_paged_kv_quantized(k, v, cache, slots)
    device, stream = here
    _check(slots, "slots", torch.int32, (None,), device)
    n = slots.shape[0]
    _check(k, "k", torch.bfloat16, (n, heads_k, dim), device, contiguous=False)
    _check(v, "v", torch.bfloat16, (n, heads_k, dim), device, contiguous=False)
    k, k0, k1 = _rows(k)
    v, v0, v1 = _rows(v)
    check("zs_paged_append_quant", lib().zs_paged_append_quant(
        stream, k.data_ptr(), v.data_ptr(), k0, k1, v0, v1, slots.data_ptr(), n, data, blocks, page, heads_k, dim,
        bits))


def read_paged_kv_quantized(cache: QuantizedKVCache, slots):
    """The keys and values in slots (int32 [tokens], in any order, any number of
    times) of a cache held in 4 or 8 bits: (k, v), (tokens, Hkv, D) bf16 each,
    low + code * scale in fp32, rounded to bf16; zeros for slots outside the pool
    (-1)."""
    torch = _torch()
    data, blocks, page, heads_k, dim, bits = _quantized(cache)
    here = _here(cache.data)
    if here is None:
        with torch.cuda.device(cache.data.device):
            return read_paged_kv_quantized(cache, slots)
    device, stream = here
    _check(slots, "slots", torch.int32, (None,), device)
    n = slots.shape[0]
    k = torch.empty((n, heads_k, dim), dtype=torch.bfloat16, device=slots.device)
    v = torch.empty_like(k)
    check("zs_paged_read_quant", lib().zs_paged_read_quant(
        stream, data, blocks, page, heads_k, dim, bits, slots.data_ptr(), n, k.data_ptr(), v.data_ptr()))
    return k, v
