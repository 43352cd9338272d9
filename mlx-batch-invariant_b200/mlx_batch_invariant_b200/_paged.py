"""A serving step over a KV cache in pages: layout, rotary write and attention.

The reference keeps one contiguous cache per batch; these three operators are what a server
needs instead, with the property of the rest of the package: a token's bits do not depend on
the other requests of the step, on how many of its request's tokens arrive together, or on
which pages hold its sequence.

A cache is (num_pages, kv_heads, page_size, head_dim): a page holds page_size consecutive
tokens of one request.  A request's row of the block table lists its pages in order; a slot
is page * page_size + place in the page.  One step is

    plan = paged_plan(query_lens, context_lens, block_table, page_size, num_tokens,
                      free_pages=free, free_head=head)
    q = rope_kv_paged(qkv, cos, sin, plan.positions, plan.slots, k_cache, v_cache)  # per layer
    o = paged_attention(q, k_cache, v_cache, block_table, plan.query_start, plan.seq_lens)

All three enqueue work on the current stream of their tensors' device, never wait for the
GPU, and can be captured in a CUDA graph whose replays read new lengths from the same tensors.
"""

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._gemm import _check_cuda

MAX_PAGED_HEAD_DIM = 256
_new_tuple = tuple.__new__


class PagedPlan(NamedTuple):
    """The token layout of one step (see paged_plan)."""
    query_start: torch.Tensor          # (requests + 1,) int32: first row of each request
    seq_lens: torch.Tensor             # (requests,) int32: cached and new tokens
    positions: torch.Tensor            # (num_tokens,) int64, -1 behind the last token
    slots: torch.Tensor                # (num_tokens,) int64, -1 behind the last token
    next_head: Optional[torch.Tensor]  # (1,) int32: free_head of the next step


def _is_vector(name, t, dtype, n=None):
    if t.ndim != 1 or t.dtype != dtype or not t.is_contiguous() or (n is not None
                                                                    and t.shape[0] != n):
        raise ValueError("%s must be a contiguous %s vector%s, got %s %s"
                         % (name, dtype, "" if n is None else " of %d" % n, tuple(t.shape),
                            t.dtype))


def _check_table(block_table, R):
    if (block_table.ndim != 2 or block_table.dtype != torch.int32
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1)
            or (block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1])):
        raise ValueError("block_table must be an int32 matrix with contiguous rows, got %s %s"
                         % (tuple(block_table.shape), block_table.dtype))
    if block_table.shape[0] != R:
        raise ValueError("block_table has %d rows for %d requests" % (block_table.shape[0], R))


def paged_plan(query_lens, context_lens, block_table, page_size, num_tokens, *, free_pages=None,
               free_head=None):
    """The token layout of a step in which request r brings ``query_lens[r]`` new tokens behind
    the ``context_lens[r]`` it has in the cache (both (requests,) int32), as a
    :class:`PagedPlan`: ``query_start``, ``seq_lens``, and for each of ``num_tokens`` rows the
    token's position and cache slot (-1 behind the last token: a padded step).

    With ``free_pages`` ((n,) int32) the pages that the new tokens need are taken from
    ``free_pages[free_head:]`` in request order and entered into ``block_table`` (int32,
    (requests, width), changed in place); ``next_head`` is the head that the next step passes
    as ``free_head`` ((1,) int32).  Without it the table holds every page already.

    The lengths are device data, so what is wrong with them is not raised: a length that is
    negative or exceeds the table's row makes its request bring no tokens, a token without a
    page gets slot -1, and both, like more tokens than ``num_tokens``, are reported by
    ``_lib.device_error()``.

    The outputs may share one allocation: a server that keeps ``next_head`` from step to step
    keeps that step's positions and slots as well until the next one replaces it.
    """
    compiling = torch.compiler.is_compiling()
    if not compiling:
        out = (_lib._short or _lib.short_way()).plan(
            query_lens, context_lens, block_table, page_size, num_tokens, free_pages, free_head)
        if out.__class__ is tuple:
            return _new_tuple(PagedPlan, out)
        if out is not None:
            _lib.check(out, "bi_paged_plan")
    page_size, num_tokens = int(page_size), int(num_tokens)
    if page_size < 1:
        raise ValueError("page_size must be positive, got %d" % page_size)
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative, got %d" % num_tokens)
    _is_vector("query_lens", query_lens, torch.int32)
    R = query_lens.shape[0]
    _is_vector("context_lens", context_lens, torch.int32, R)
    _check_table(block_table, R)
    if (free_pages is None) != (free_head is None):
        raise ValueError("free_pages and free_head go together")
    if free_pages is not None:
        _is_vector("free_pages", free_pages, torch.int32)
        _is_vector("free_head", free_head, torch.int32, 1)
    dev = _check_cuda(query_lens, context_lens, block_table, free_pages, free_head)
    if compiling:
        out = torch.ops.mlx_bi.paged_plan(query_lens, context_lens, block_table, page_size,
                                          num_tokens, free_pages, free_head)
        return PagedPlan(*out[:4], out[4] if free_pages is not None else None)
    return PagedPlan(*_plan_eager(query_lens, context_lens, block_table, page_size, num_tokens,
                                  free_pages, free_head, dev))


def _plan_eager(query_lens, context_lens, block_table, page_size, num_tokens, free_pages,
                free_head, dev):
    R = query_lens.shape[0]
    start = torch.empty(R + 1, dtype=torch.int32, device=dev)
    seq = torch.empty(R, dtype=torch.int32, device=dev)
    pos = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    head = torch.empty(1, dtype=torch.int32, device=dev) if free_pages is not None else None
    with torch.cuda.device(dev):
        st = _lib.lib().bi_paged_plan(
            query_lens.data_ptr(), context_lens.data_ptr(), R, num_tokens,
            block_table.data_ptr(), block_table.stride(0), block_table.shape[1], page_size,
            _list_ptr(free_pages), free_pages.shape[0] if free_pages is not None else 0,
            free_head.data_ptr() if free_head is not None else None, start.data_ptr(),
            seq.data_ptr(), pos.data_ptr(), slots.data_ptr(),
            head.data_ptr() if head is not None else None, _lib.stream_handle(dev))
    _lib.check(st, "bi_paged_plan")
    return start, seq, pos, slots, head


def _list_ptr(free_pages):
    """An empty list of free pages is a list: any pointer but null stands for it."""
    if free_pages is None:
        return None
    return free_pages.data_ptr() or 16


def _check_caches(k_cache, v_cache, dtype):
    if k_cache.ndim != 4 or v_cache.ndim != 4:
        raise ValueError("a cache is (num_pages, kv_heads, page_size, head_dim)")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have one shape, got %s and %s"
                         % (tuple(k_cache.shape), tuple(v_cache.shape)))
    if not (k_cache.dtype == v_cache.dtype == dtype):
        raise ValueError("the caches must have the tokens' dtype %s, got %s and %s"
                         % (dtype, k_cache.dtype, v_cache.dtype))
    if k_cache.shape[2] < 1:
        raise ValueError("page_size must be positive")
    for t in (k_cache, v_cache):
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError("the caches' last dimension must be contiguous")
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise ValueError("the caches must not be expanded tensors")


def _check_aligned(*caches):
    for t in caches:
        vec = 16 // t.element_size()
        if t.data_ptr() % 16 or any(s % vec for s in _cache_strides(t)):
            raise ValueError("the caches must be 16-byte aligned with strides that are multiples "
                             "of 16 bytes")


def _cache_strides(t):
    """Element strides of page, head and token (of a dimension of one: the head dim, so that
    what torch keeps there does not matter)."""
    return [s if n > 1 else t.shape[3] for s, n in zip(t.stride()[:3], t.shape[:3])]


def rope_kv_paged(qkv, cos, sin, positions, slots, k_cache, v_cache, *, out=None):
    """Rotary embedding of a fused projection's q and k heads, and the write of k and v into
    the pages: the paged form of the decoder's bi_rope_kv, with the same arithmetic.

    ``qkv`` (tokens, (q_heads + 2 kv_heads) * head_dim); token t sits at ``positions[t]`` and
    its rotated k and its v go to ``slots[t]`` of the caches (changed in place); the rotated q,
    (tokens, q_heads, head_dim), is returned (in ``out`` where given).  ``cos`` and ``sin`` are
    fp32 (positions, rot / 2); a head's first ``rot`` elements are rotated in halves, the rest
    is copied.  Tokens with a negative position are padding: nothing of theirs is written, in
    ``out`` neither.  A negative slot keeps k and v out of the cache.  Positions past the
    tables and slots past the caches write nothing and are reported by
    ``_lib.device_error()``.  The slots of a call must differ.
    """
    compiling = torch.compiler.is_compiling()
    if not compiling:
        q = (_lib._short or _lib.short_way()).rope(qkv, cos, sin, positions, slots, k_cache,
                                                   v_cache, out)
        if q.__class__ is not int and q is not None:
            return q
        if q is not None:
            _lib.check(q, "bi_rope_kv_paged")
    if qkv.ndim != 2:
        raise ValueError("qkv must be (tokens, (q_heads + 2 kv_heads) * head_dim)")
    _lib.dtype_code(qkv.dtype)
    _check_caches(k_cache, v_cache, qkv.dtype)
    T, width = qkv.shape
    n_pages, hk, page, hd = k_cache.shape
    if hd % 2 or hd == 0:
        raise ValueError("head_dim must be even and positive, got %d" % hd)
    if width % hd or width // hd < 2 * hk:
        raise ValueError("a row of qkv has %d elements: not q heads and 2 x %d kv heads of %d"
                         % (width, hk, hd))
    hq = width // hd - 2 * hk
    if (cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32
            or sin.dtype != torch.float32 or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous float32 (positions, rot / 2)")
    if 2 * cos.shape[1] > hd:
        raise ValueError("rot = %d exceeds the head dim %d" % (2 * cos.shape[1], hd))
    _is_vector("positions", positions, torch.int64, T)
    _is_vector("slots", slots, torch.int64, T)
    if out is not None and (tuple(out.shape) != (T, hq, hd) or out.dtype != qkv.dtype
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous (%d, %d, %d) %s tensor" % (T, hq, hd,
                                                                             qkv.dtype))
    dev = _check_cuda(qkv, cos, sin, positions, slots, k_cache, v_cache, out)
    if compiling:
        if out is not None:
            raise NotImplementedError("rope_kv_paged under torch.compile takes no out=")
        return torch.ops.mlx_bi.rope_kv_paged(qkv, cos, sin, positions, slots, k_cache, v_cache)
    return _rope_eager(qkv, cos, sin, positions, slots, k_cache, v_cache, out, dev)


def _rope_eager(qkv, cos, sin, positions, slots, k_cache, v_cache, out, dev):
    T, width = qkv.shape
    n_pages, hk, page, hd = k_cache.shape
    hq = width // hd - 2 * hk
    if (width > 1 and qkv.stride(1) != 1) or (T > 1 and qkv.stride(0) < width):
        qkv = qkv.contiguous()
    if out is None:
        out = torch.empty((T, hq, hd), dtype=qkv.dtype, device=dev)
    with torch.cuda.device(dev):
        st = _lib.lib().bi_rope_kv_paged(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else width, T, hq, hk, hd, 2 * cos.shape[1],
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
            slots.data_ptr(), out.data_ptr(), k_cache.data_ptr(),
            _lib.i64_3(_cache_strides(k_cache)), v_cache.data_ptr(),
            _lib.i64_3(_cache_strides(v_cache)), n_pages, page, _lib.dtype_code(qkv.dtype),
            _lib.stream_handle(dev))
    _lib.check(st, "bi_rope_kv_paged")
    return out


def paged_attention(q, k_cache, v_cache, block_table, query_start, seq_lens, *, scale=None,
                    window=None, first_tokens=0, sinks=None, out=None):
    """Attention of each request's new tokens over its sequence in the pages.

    ``q`` (tokens, heads, head_dim) holds the requests' tokens one after the other: request
    r's are rows ``query_start[r]`` to ``query_start[r + 1]`` and are the last ones of its
    ``seq_lens[r]`` (whose keys and values are in the caches already).  A token at position p
    sees the keys i <= p; with a ``window`` (None or 0: without) only those with i > p - window,
    and the sequence's ``first_tokens`` first ones.  ``sinks`` is an optional logit per query
    head, as in scaled_dot_product_attention; -inf is none.  Heads are grouped: heads % kv_heads
    == 0.  float16 / bfloat16 with head dim 64 or 128 and pages that divide or are multiples of
    128 run on the tensor cores, with the weights rounded to that type ahead of the product with
    v (scaled_dot_product_attention keeps them in fp32); everything else in fp32 throughout.

    Rows outside every request are not written: pass ``out`` (which may be ``q``, not an expanded
    tensor) where that matters.  A row that sees nothing returns zeros.  Lengths are device data; they are clamped
    to ``q`` and to the table, and pages outside the cache read as zeros.
    """
    compiling = torch.compiler.is_compiling()
    if not compiling:
        o = (_lib._short or _lib.short_way()).attention(
            q, k_cache, v_cache, block_table, query_start, seq_lens, scale, window, first_tokens,
            sinks, out)
        if o.__class__ is not int and o is not None:
            return o
        if o is not None:
            _lib.check(o, "bi_paged_sdpa")
    if q.ndim != 3:
        raise ValueError("q must be (tokens, heads, head_dim)")
    code = _lib.dtype_code(q.dtype)
    _check_caches(k_cache, v_cache, q.dtype)
    T, H, D = q.shape
    n_pages, Hkv, page, Dk = k_cache.shape
    if Dk != D:
        raise ValueError("q has head dim %d, the caches %d" % (D, Dk))
    if Hkv == 0 or H % Hkv:
        raise ValueError("head count %d is not a multiple of kv head count %d" % (H, Hkv))
    if D % 32 or D == 0:
        raise ValueError("the head dimension must be a multiple of 32, got %d" % D)
    if D > MAX_PAGED_HEAD_DIM:
        raise NotImplementedError("paged attention with head dim %d is not built (at most %d)"
                                  % (D, MAX_PAGED_HEAD_DIM))
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 <= scale < 3.0e38:
        raise ValueError("scale must be finite and not negative, got %r" % scale)
    window = 0 if window is None else int(window)
    if window < 0 or int(first_tokens) < 0:
        raise ValueError("window and first_tokens must not be negative")
    if first_tokens and not window:
        raise ValueError("first_tokens needs a window")
    _is_vector("seq_lens", seq_lens, torch.int32)
    R = seq_lens.shape[0]
    _is_vector("query_start", query_start, torch.int32, R + 1)
    _check_table(block_table, R)
    if R and T and (block_table.shape[1] == 0 or n_pages == 0):
        raise ValueError("the block table and the cache must not be empty")
    if sinks is not None:
        if tuple(sinks.shape) != (H,):
            raise ValueError("sinks must have shape (%d,), got %s" % (H, tuple(sinks.shape)))
        sinks = sinks.to(q.dtype).contiguous()
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                            or (D > 1 and out.stride(2) != 1)):
        raise ValueError("out must be %s %s with a contiguous last dimension"
                         % (tuple(q.shape), q.dtype))
    if out is not None and any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError("out must not be an expanded tensor")
    if not compiling:
        _check_aligned(k_cache, v_cache)
    dev = _check_cuda(q, k_cache, v_cache, block_table, query_start, seq_lens, sinks, out)
    if compiling:
        if out is not None:
            raise NotImplementedError("paged_attention under torch.compile takes no out=")
        return torch.ops.mlx_bi.paged_attention(q, k_cache, v_cache, block_table, query_start,
                                                seq_lens, scale, window, int(first_tokens), sinks)
    return _attention_eager(q, k_cache, v_cache, block_table, query_start, seq_lens, scale,
                            window, int(first_tokens), sinks, out, code, dev)


def _attention_eager(q, k_cache, v_cache, block_table, query_start, seq_lens, scale, window,
                     first_tokens, sinks, out, code, dev):
    T, H, D = q.shape
    n_pages, Hkv, page, _ = k_cache.shape
    R, width = block_table.shape
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    if T == 0 or R == 0 or H == 0:
        return out
    vec = 16 // q.element_size()
    if (q.data_ptr() % 16 or q.stride(2) != 1
            or any((s % vec or s == 0) and n > 1 for s, n in zip(q.stride()[:2], q.shape[:2]))):
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    if out.data_ptr() % 16 or any(s % vec for s in out.stride()[:2]):
        # the kernels store 16-byte vectors: go through an aligned copy (rows outside every
        # request come back as they were)
        tmp = _attention_eager(q, k_cache, v_cache, block_table, query_start, seq_lens, scale,
                               window, first_tokens, sinks, out.clone(
                                   memory_format=torch.contiguous_format), code, dev)
        return out.copy_(tmp)
    lib = _lib.lib()
    with torch.cuda.device(dev):
        ws = torch.empty(lib.bi_paged_sdpa_workspace(T, R, H, D, width, page),
                         dtype=torch.uint8, device=dev)
        qs = [s if n > 1 else D for s, n in zip(q.stride()[:2], q.shape[:2])]
        st = lib.bi_paged_sdpa(
            q.data_ptr(), _lib.i64_2(qs), k_cache.data_ptr(),
            _lib.i64_3(_cache_strides(k_cache)), v_cache.data_ptr(),
            _lib.i64_3(_cache_strides(v_cache)), n_pages, page, block_table.data_ptr(),
            block_table.stride(0), width, query_start.data_ptr(), seq_lens.data_ptr(),
            sinks.data_ptr() if sinks is not None else None, float(scale), window, first_tokens,
            T, R, H, Hkv, D, code, out.data_ptr(), _lib.i64_2(out.stride()[:2]), ws.data_ptr(),
            ws.numel(), _lib.stream_handle(dev))
    _lib.check(st, "bi_paged_sdpa")
    return out
