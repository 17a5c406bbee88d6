"""The paged 8-bit KV cache of a serving step: requests of different lengths, one pool of
pages, INT8 codes with one scale per page and KV head (``csrc/paged_cache.cu``,
``csrc/paged_attn.cu``).

The reference decodes one batch of equal lengths over a 16-bit contiguous cache
(src/runtime/graph_decode.py:96-168); this is the same decode attention for requests that
come and go, at about half the bytes per key.  A step is

    plan_step      once: pages, slots and positions of the step's new tokens   (1 launch)
    cache_write    per layer: RoPE of q and k, new K/V into their pages        (1)
    attn_paged     per layer: attention over the pages                         (1)

and every launch may be captured in a CUDA graph: lengths, tables and the free pages live
on the GPU, so a captured step serves every later step of the same shape.

    pool = PagePool(num_pages, max_requests, max_len, page_size=64)
    layers = [KVPages(num_pages, kv_heads, 64, head_dim) for _ in range(n)]
    plan = StepPlan(pool, max_tokens, q_heads=..., kv_heads=..., head_dim=...)
    plan_step(new_lens, pool, plan)                 # int32 [max_requests], 0 for idle slots
    q = cache_write(k, v, layers[i], plan, q=q, cos=cos, sin=sin)
    out = attn_paged(q, layers[i], plan, scale)     # rows as in plan.cu_new
    release_requests(finished, pool)

Token rows are the requests' new tokens in request order (``plan.cu_new``); rows behind the
last one are ignored.  A pool, its plans and its layers belong to one stream at a time: a
step on another stream waits for the one before like any other user of the tensors.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from . import _native as N
from .trace import traced

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


def _device(device) -> torch.device:
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError("the paged cache needs a CUDA device (there is no CPU path)")
    return dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())


def _check_page(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return int(page_size)


def _check_state(t: torch.Tensor, dtype: torch.dtype, numel: int, name: str) -> None:
    if t.dtype != dtype or t.numel() != numel or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {numel} elements")


def _check_rows(t: torch.Tensor, rows: int, width: int, dtype: torch.dtype, what: str) -> None:
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != width or t.dtype != dtype:
        raise ValueError(f"{what} must be a [{rows}, {width}] tensor of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    if t.stride(1) != 1 or (rows > 1 and t.stride(0) < width):
        raise ValueError(f"{what} must have unit column stride and rows that do not overlap")


def _ld(t: torch.Tensor) -> int:
    """Row stride; a single row's is its width (a stride of a size-1 dimension means nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class PagePool:
    """Lengths, block tables and free pages of up to ``max_requests`` requests of up to
    ``max_len`` tokens, on the GPU.

    ``lengths`` int32 [max_requests] (tokens cached), ``block_table`` int32 [max_requests,
    pages per request] (-1: none), ``free_pages`` int32 [num_pages], of which the first
    ``free_count`` [1] are free (the last of them goes first), ``status`` int32 [1]."""

    def __init__(self, num_pages: int, max_requests: int, max_len: int, page_size: int = 64,
                 device: Union[torch.device, str] = "cuda") -> None:
        self.page_size = _check_page(page_size)
        if not 1 <= max_requests <= N.TQ_MAX_REQUESTS:
            raise ValueError(f"max_requests must be in 1..{N.TQ_MAX_REQUESTS}")
        if num_pages < 1 or max_len < 1:
            raise ValueError("num_pages and max_len must be positive")
        self.num_pages, self.max_requests = int(num_pages), int(max_requests)
        self.table_width = (int(max_len) + self.page_size - 1) // self.page_size
        if max(self.num_pages, self.table_width) * self.page_size >= 2**31:
            raise ValueError("more than 2^31 - 1 tokens in the pool or in a request")
        self.device = _device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(self.max_requests, **i32)
        self.block_table = torch.full((self.max_requests, self.table_width), -1, **i32)
        self.free_pages = torch.arange(self.num_pages - 1, -1, -1, **i32)  # page 0 is taken first
        self.free_count = torch.full((1,), self.num_pages, **i32)
        self.status = torch.zeros(1, **i32)

    def reset(self) -> None:
        """Forget every request (stream-ordered)."""
        self.lengths.zero_()
        self.block_table.fill_(-1)
        self.free_pages.copy_(torch.arange(self.num_pages - 1, -1, -1, dtype=torch.int32, device=self.device))
        self.free_count.fill_(self.num_pages)
        self.status.zero_()

    def check_status(self) -> None:
        """Raise ``TileQuantError`` if a step since the last check could not place a request
        or met a bad page id.  Reads the status word, which synchronises, and clears it."""
        st = int(self.status.item())
        if not st:
            return
        self.status.zero_()
        what = [text for bit, text in ((N.TQ_PAGES_POOL_EMPTY, "too few free pages"),
                                       (N.TQ_PAGES_TABLE_FULL, "a request longer than its block table"),
                                       (N.TQ_PAGES_ROWS_FULL, "more new tokens than the plan has rows"),
                                       (N.TQ_PAGES_BAD_PAGE, "a page id outside the pool, or a page given back twice"))
                if st & bit]
        raise N.TileQuantError("page pool: " + "; ".join(what))


class KVPages:
    """One layer's cache: ``k``, ``v`` int8 [pages, kv_heads, page_size, head_dim] and
    ``k_scale``, ``v_scale`` f32 [pages, kv_heads]; a value is code * scale."""

    def __init__(self, num_pages: int, kv_heads: int, page_size: int, head_dim: int,
                 device: Union[torch.device, str] = "cuda") -> None:
        _check_page(page_size)
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if num_pages < 1 or kv_heads < 1:
            raise ValueError("num_pages and kv_heads must be positive")
        if num_pages * kv_heads * page_size * head_dim // 128 >= 2**31:
            raise ValueError("the pool is too large for one layer's TMA coordinates")
        dev = _device(device)
        shape = (int(num_pages), int(kv_heads), int(page_size), int(head_dim))
        self.k = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.v = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.k_scale = torch.zeros(shape[:2], dtype=torch.float32, device=dev)
        self.v_scale = torch.zeros(shape[:2], dtype=torch.float32, device=dev)


def _check_kv(kv: KVPages) -> Tuple[int, int, int, int]:
    if kv.k.dim() != 4 or kv.k.shape != kv.v.shape or kv.k.dtype != torch.int8 or kv.v.dtype != torch.int8 \
            or not (kv.k.is_contiguous() and kv.v.is_contiguous()):
        raise ValueError("KVPages: k and v must be contiguous int8 [pages, kv_heads, page, head_dim] tensors")
    P, H, page, D = (int(n) for n in kv.k.shape)
    for t in (kv.k_scale, kv.v_scale):
        if tuple(t.shape) != (P, H) or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("KVPages: scales must be contiguous float32 [pages, kv_heads] tensors")
    return P, H, page, D


class StepPlan:
    """What ``plan_step`` makes for a step of up to ``max_tokens`` new tokens, and the
    workspace of ``attn_paged`` over it.

    ``cu_new`` int32 [max_requests + 1]: request r's token rows are cu_new[r] .. cu_new[r+1];
    ``slots``, ``positions`` int64 [max_tokens] (-1 for rows without a token); ``kv_len`` int32
    [max_requests]: the keys its tokens see.  ``max_new`` is the usual most new tokens of one
    request: with the query heads per KV head it sets how many query rows share a pass over
    the keys (more tokens per request work too, in several passes)."""

    def __init__(self, pool: PagePool, max_tokens: int, *, q_heads: int, kv_heads: int, head_dim: int,
                 max_new: int = 1) -> None:
        if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
            raise ValueError("q_heads must be a multiple of kv_heads")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if not 1 <= max_tokens < 2**31 or max_new < 1:
            raise ValueError("max_tokens and max_new must be positive")
        self.pool, self.max_tokens = pool, int(max_tokens)
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        group_rows = self.q_heads // self.kv_heads * min(int(max_new), self.max_tokens)
        self.row_tile = 8 if group_rows <= 8 else 16 if group_rows <= 16 else 32
        dev, R = pool.device, pool.max_requests
        lib = N.load()
        with torch.cuda.device(dev):
            self.attn_ctas = int(lib.tq_paged_attn_ctas(self.row_tile))
        i32 = dict(dtype=torch.int32, device=dev)
        self.cu_new = torch.zeros(R + 1, **i32)
        self.slots = torch.full((self.max_tokens,), -1, dtype=torch.int64, device=dev)
        self.positions = torch.full((self.max_tokens,), -1, dtype=torch.int64, device=dev)
        self.kv_len = torch.zeros(R, **i32)
        self.items = torch.zeros((int(lib.tq_plan_items(self.max_tokens, R, pool.page_size)), 4), **i32)
        self.counts = torch.zeros(4, **i32)
        self.cu_work = torch.zeros(R + 1, **i32)
        self.attn_start = torch.zeros(self.attn_ctas, **i32)
        parts = 2 * self.attn_ctas * self.row_tile
        self.ws_o = torch.empty(parts * self.head_dim, dtype=torch.float32, device=dev)
        self.ws_ml = torch.empty(parts * 2, dtype=torch.float32, device=dev)
        self.arrivals = torch.zeros(self.attn_ctas, **i32)
        self.err = torch.zeros(1, **i32)


@traced("tq.plan_step")
def plan_step(new_lens: torch.Tensor, pool: PagePool, plan: StepPlan, lengths_out: Optional[torch.Tensor] = None,
              free_count_out: Optional[torch.Tensor] = None) -> StepPlan:
    """Place ``new_lens`` (int32 [max_requests]) new tokens of every request: fresh pages
    into ``pool.block_table``, and the plan's slots, positions and work lists.

    ``pool.lengths`` and ``pool.free_count`` advance, unless ``lengths_out`` /
    ``free_count_out`` take the new values.  A request for which the pool, its table row or
    the plan's rows are too small keeps its length, its rows get slot and position -1, and
    ``pool.check_status()`` tells; the other requests are served (in request order: after
    the first that finds too few pages none gets any)."""
    lengths_out = pool.lengths if lengths_out is None else lengths_out
    free_count_out = pool.free_count if free_count_out is None else free_count_out
    N.require_cuda(new_lens, pool.lengths, pool.block_table, pool.free_pages, pool.free_count, lengths_out,
                   free_count_out, plan.slots)
    R, P = pool.max_requests, pool.num_pages
    if plan.pool is not pool:
        raise ValueError("plan_step: the plan belongs to another pool")
    for t, n, name in ((new_lens, R, "new_lens"), (pool.lengths, R, "lengths"), (lengths_out, R, "lengths_out"),
                       (pool.block_table, R * pool.table_width, "block_table"), (pool.free_pages, P, "free_pages"),
                       (pool.free_count, 1, "free_count"), (free_count_out, 1, "free_count_out")):
        _check_state(t, torch.int32, n, f"plan_step: {name}")
    a = N.PlanArgs(new_lens=new_lens.data_ptr(), lengths=pool.lengths.data_ptr(), lengths_out=lengths_out.data_ptr(),
                   block_table=pool.block_table.data_ptr(), free_pages=pool.free_pages.data_ptr(),
                   free_count=pool.free_count.data_ptr(), free_count_out=free_count_out.data_ptr(),
                   cu_new=plan.cu_new.data_ptr(), slots=plan.slots.data_ptr(), positions=plan.positions.data_ptr(),
                   kv_len=plan.kv_len.data_ptr(), items=plan.items.data_ptr(), counts=plan.counts.data_ptr(),
                   cu_work=plan.cu_work.data_ptr(), attn_start=plan.attn_start.data_ptr(),
                   status=pool.status.data_ptr(), requests=R, table_width=pool.table_width, page=pool.page_size,
                   pages=P, max_tokens=plan.max_tokens, kv_heads=plan.kv_heads, group=plan.q_heads // plan.kv_heads,
                   row_tile=plan.row_tile, attn_ctas=plan.attn_ctas, reserved=0)
    with torch.cuda.device(pool.device):
        N.check(N.load().tq_plan_step(ctypes.byref(a), N.stream_of(new_lens)), "plan_step")
    return plan


@traced("tq.release_requests")
def release_requests(finished: torch.Tensor, pool: PagePool) -> None:
    """Give back the pages of the requests with ``finished`` (bool or uint8 [max_requests]);
    their lengths become 0."""
    N.require_cuda(finished, pool.lengths, pool.block_table, pool.free_pages, pool.free_count)
    if finished.dtype == torch.bool:
        finished = finished.view(torch.uint8)
    R = pool.max_requests
    _check_state(finished, torch.uint8, R, "release_requests: finished")
    for t, n, name in ((pool.lengths, R, "lengths"), (pool.block_table, R * pool.table_width, "block_table"),
                       (pool.free_pages, pool.num_pages, "free_pages"), (pool.free_count, 1, "free_count")):
        _check_state(t, torch.int32, n, f"release_requests: {name}")
    with torch.cuda.device(pool.device):
        N.check(N.load().tq_release_requests(
            finished.data_ptr(), pool.lengths.data_ptr(), pool.block_table.data_ptr(), pool.free_pages.data_ptr(),
            pool.free_count.data_ptr(), pool.status.data_ptr(), R, pool.table_width, pool.page_size, pool.num_pages,
            N.stream_of(finished)), "release_requests")


def _check_plan(plan: StepPlan, kv: KVPages, what: str) -> Tuple[int, int, int, int]:
    P, H, page, D = _check_kv(kv)
    if (P, page) != (plan.pool.num_pages, plan.pool.page_size):
        raise ValueError(f"{what}: the cache has {P} pages of {page} tokens, the plan's pool "
                         f"{plan.pool.num_pages} of {plan.pool.page_size}")
    if (H, D) != (plan.kv_heads, plan.head_dim):
        raise ValueError(f"{what}: the cache has {H} KV heads of {D}, the plan {plan.kv_heads} of {plan.head_dim}")
    return P, H, page, D


@traced("tq.cache_write")
def cache_write(k: torch.Tensor, v: torch.Tensor, kv: KVPages, plan: StepPlan, q: Optional[torch.Tensor] = None,
                cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The step's new keys and values (``k``, ``v`` [rows, kv_heads * D] views) into the
    pages of ``plan``.  With ``cos``/``sin`` ([rows, D]) and ``q`` ([rows, q_heads * D]), K is
    rotated first and the rotated q is returned (in ``q_out``, which may be ``q``).

    A page and head whose values outgrow its scale gets the larger scale, and the codes it
    holds are rounded again; NaN is stored as 0, an infinity as the page's largest value."""
    N.require_cuda(k, v, kv.k, kv.v, kv.k_scale, kv.v_scale, plan.items, q, cos, sin, q_out)
    P, H, page, D = _check_plan(plan, kv, "cache_write")
    rows, dtype = int(k.shape[0]), k.dtype
    code = N.dtype_code(dtype)
    _check_rows(k, rows, H * D, dtype, "cache_write: k")
    _check_rows(v, rows, H * D, dtype, "cache_write: v")
    if rows > plan.max_tokens:
        raise ValueError(f"cache_write: {rows} rows, the plan has {plan.max_tokens}")
    if not (q is None) == (cos is None) == (sin is None) or (q is None and q_out is not None):
        raise ValueError("cache_write: q, cos and sin come together")
    if q is not None:
        width = plan.q_heads * D
        _check_rows(q, rows, width, dtype, "cache_write: q")
        _check_rows(cos, rows, D, dtype, "cache_write: cos")
        _check_rows(sin, rows, D, dtype, "cache_write: sin")
        if _ld(cos) != _ld(sin):
            raise ValueError("cache_write: cos and sin must share one row stride")
        if q_out is None:
            q_out = torch.empty((rows, width), device=q.device, dtype=dtype)
        _check_rows(q_out, rows, width, dtype, "cache_write: q_out")
    if rows == 0:
        return q_out
    pool = plan.pool
    a = N.CacheWriteArgs(k=k.data_ptr(), v=v.data_ptr(), q=N.ptr(q), cos=N.ptr(cos), sin=N.ptr(sin), q_out=N.ptr(q_out),
                         k_codes=kv.k.data_ptr(), v_codes=kv.v.data_ptr(), k_scale=kv.k_scale.data_ptr(),
                         v_scale=kv.v_scale.data_ptr(), items=plan.items.data_ptr(), counts=plan.counts.data_ptr(),
                         cu_new=plan.cu_new.data_ptr(), status=pool.status.data_ptr(), ld_k=_ld(k), ld_v=_ld(v),
                         ld_q=0 if q is None else _ld(q), ld_qo=0 if q is None else _ld(q_out),
                         ld_cs=0 if q is None else _ld(cos), rows=rows, requests=pool.max_requests, pages=P, page=page,
                         kv_heads=H, q_heads=plan.q_heads, head_dim=D, reserved=0)
    with torch.cuda.device(pool.device):
        N.check(N.load().tq_cache_write(ctypes.byref(a), code, N.stream_of(k)), "cache_write")
    return q_out


@traced("tq.read_pages")
def read_pages(kv: KVPages, page_ids: torch.Tensor, dtype: torch.dtype, k_out: Optional[torch.Tensor] = None,
               v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 16-bit values of the pages ``page_ids`` (int32 [n], e.g. a block-table row): K and
    V [n, kv_heads, page_size, head_dim].  An id outside the pool (-1) gives zeros."""
    N.require_cuda(kv.k, kv.v, kv.k_scale, kv.v_scale, page_ids, k_out, v_out)
    P, H, page, D = _check_kv(kv)
    code = N.dtype_code(dtype)
    if page_ids.dim() != 1 or page_ids.dtype != torch.int32 or not page_ids.is_contiguous():
        raise ValueError("read_pages: page_ids must be a contiguous int32 [n] tensor")
    shape = (int(page_ids.shape[0]), H, page, D)
    outs = []
    for t in (k_out, v_out):
        t = torch.empty(shape, device=kv.k.device, dtype=dtype) if t is None else t
        if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"read_pages: outputs must be contiguous {list(shape)} tensors of {dtype}")
        outs.append(t)
    if shape[0]:
        with torch.cuda.device(kv.k.device):
            N.check(N.load().tq_read_pages(
                kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(), page_ids.data_ptr(),
                shape[0], P, H, page, D, outs[0].data_ptr(), outs[1].data_ptr(), code, N.stream_of(kv.k)), "read_pages")
    return outs[0], outs[1]


@traced("tq.attn_paged")
def attn_paged(q: torch.Tensor, kv: KVPages, plan: StepPlan, scale: float,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's token rows ``q`` ([rows, q_heads * D], rotated) over the pages:
    the i-th new token of a request sees its cached tokens and the new ones up to itself.
    Rows of a request that was not placed give zeros; rows behind the last token are left as
    they are in ``out``."""
    N.require_cuda(q, kv.k, kv.v, kv.k_scale, kv.v_scale, plan.items, out)
    P, H, page, D = _check_plan(plan, kv, "attn_paged")
    rows, width = int(q.shape[0]), plan.q_heads * D
    code = N.dtype_code(q.dtype)
    _check_rows(q, rows, width, q.dtype, "attn_paged: q")
    if rows > plan.max_tokens:
        raise ValueError(f"attn_paged: {rows} rows, the plan has {plan.max_tokens}")
    if not math.isfinite(scale):
        raise ValueError("attn_paged: scale must be finite")
    out = torch.empty((rows, width), device=q.device, dtype=q.dtype) if out is None else out
    _check_rows(out, rows, width, q.dtype, "attn_paged: out")
    if rows == 0:
        return out
    pool = plan.pool
    a = N.PagedAttnArgs(q=q.data_ptr(), out=out.data_ptr(), k_codes=kv.k.data_ptr(), v_codes=kv.v.data_ptr(),
                        k_scale=kv.k_scale.data_ptr(), v_scale=kv.v_scale.data_ptr(),
                        block_table=pool.block_table.data_ptr(), cu_new=plan.cu_new.data_ptr(),
                        kv_len=plan.kv_len.data_ptr(), cu_work=plan.cu_work.data_ptr(),
                        attn_start=plan.attn_start.data_ptr(), counts=plan.counts.data_ptr(), ws_o=plan.ws_o.data_ptr(),
                        ws_ml=plan.ws_ml.data_ptr(), arrivals=plan.arrivals.data_ptr(), err=plan.err.data_ptr(),
                        status=pool.status.data_ptr(), ld_q=_ld(q), ld_out=_ld(out), rows=rows,
                        requests=pool.max_requests, table_width=pool.table_width, pages=P, page=page, kv_heads=H,
                        q_heads=plan.q_heads, head_dim=D, row_tile=plan.row_tile, attn_ctas=plan.attn_ctas,
                        scale_log2=float(scale) * math.log2(math.e), reserved=0)
    with torch.cuda.device(pool.device):
        N.check(N.load().tq_attn_paged(ctypes.byref(a), code, N.stream_of(q)), "attn_paged")
    return out
