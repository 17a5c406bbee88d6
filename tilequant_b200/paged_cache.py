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
last one are ignored.  Outputs that the caller brings keep what they hold there, those that a
call makes have zeros (an activation quantizer's scales are maxima over all rows).  Requests may
share full pages that they only read (a common prompt); a page that is still being written
belongs to one request.  A release gives back every page that the finished request's table row
names, so a page that another request goes on reading is first taken out of that row (its entry
set to -1).  A pool, its plans and its layers belong to one stream at a time: a step on another
stream waits for the one before like any other user of the tensors, and so do two captured
graphs that use one plan.
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
LOG2E = math.log2(math.e)


def _device(device) -> torch.device:
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError("the paged cache needs a CUDA device (there is no CPU path)")
    return dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())


def _check_page(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return int(page_size)


def _check_state(t: torch.Tensor, dtype: torch.dtype, numel: int, index: int, name: str) -> None:
    if not t.is_cuda:
        raise ValueError("tilequant_b200 kernels need CUDA tensors (there is no CPU path)")
    if t.dtype != dtype or t.numel() != numel or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {numel} elements")
    if t.device.index != index:
        raise ValueError(f"{name} is on {t.device}, the pool on cuda:{index}")


def _check_rows(t: torch.Tensor, rows: int, width: int, dtype: torch.dtype, index: int, what: str,
                shared: bool = False) -> int:
    """Checks a [rows, width] operand; its row stride (a single row's is its width: the stride of
    a dimension of size 1 means nothing).  ``shared``: an expanded row (stride 0) will do."""
    if not t.is_cuda:
        raise ValueError("tilequant_b200 kernels need CUDA tensors (there is no CPU path)")
    if t.dtype != dtype or t.shape != (rows, width):
        raise ValueError(f"{what} must be a [{rows}, {width}] tensor of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, the pool on cuda:{index}")
    ld, unit = t.stride()
    if unit != 1 or (rows > 1 and ld < width and not (shared and ld == 0)):
        raise ValueError(f"{what} must have unit column stride and rows that do not overlap")
    return ld if rows > 1 else width


class PagePool(N.FixedTensors):
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
        if self.num_pages * self.page_size >= 2**31 or self.table_width * self.page_size >= 2**31 - 128:
            raise ValueError("more than 2^31 - 1 tokens in the pool or 2^31 - 129 in a request")
        self.device = _device(device)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(self.max_requests, **i32)
        self.block_table = torch.full((self.max_requests, self.table_width), -1, **i32)
        self.free_pages = torch.arange(self.num_pages - 1, -1, -1, **i32)  # page 0 is taken first
        self.free_count = torch.full((1,), self.num_pages, **i32)
        self.status = torch.zeros(1, **i32)

    @torch.inference_mode()  # (the pool may have been made in it, as a decoder's is)
    def reset(self) -> None:
        """Forget every request, and what ``check_status`` would tell (stream-ordered)."""
        self.forget_requests()
        self.status.zero_()

    @torch.inference_mode()
    def forget_requests(self) -> None:
        """Forget every request; the status word stays for ``check_status`` (stream-ordered)."""
        self.lengths.zero_()
        self.block_table.fill_(-1)
        self.free_pages.copy_(torch.arange(self.num_pages - 1, -1, -1, dtype=torch.int32, device=self.device))
        self.free_count.fill_(self.num_pages)

    @torch.inference_mode()
    def check_status(self) -> None:
        """Raise ``TileQuantError`` if a step since the last check could not place a request
        or met a bad page id.  Reads the status word, which synchronises, and clears it."""
        st = int(self.status.item())
        if not st:
            return
        self.status.zero_()
        what = [text for bit, text in ((N.TQ_PAGES_POOL_EMPTY, "too few free pages"),
                                       (N.TQ_PAGES_TABLE_FULL, "a request longer than its block table"),
                                       (N.TQ_PAGES_ROWS_FULL, "more new tokens than the plan, or a cache_write, has rows"),
                                       (N.TQ_PAGES_BAD_PAGE, "a page id outside the pool, or a free page given back"))
                if st & bit]
        raise N.TileQuantError("page pool: " + "; ".join(what))


class KVPages(N.FixedTensors):
    """One layer's cache: ``k``, ``v`` int8 [pages, kv_heads, page_size, head_dim] and
    ``k_scale``, ``v_scale`` f32 [pages, kv_heads]; a value is code * scale.

    One scale serves all channels of a page and head, so a channel keeps steps of 1/127 of the
    largest one's: where a model's keys have channels far above the rest, the rest lose bits."""

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
        self._shape, self._index = shape, dev.index
        self._ptrs = tuple(t.data_ptr() for t in (self.k, self.v, self.k_scale, self.v_scale))


class StepPlan(N.FixedTensors):
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
        self.row_tile = 8 if group_rows <= 8 else 16
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
        self.attn_start = torch.zeros((self.attn_ctas, 8), **i32)
        parts = 2 * self.attn_ctas * self.row_tile
        self.ws_o = torch.empty(parts * self.head_dim, dtype=torch.float32, device=dev)
        self.ws_ml = torch.empty(parts * 2, dtype=torch.float32, device=dev)
        self.arrivals = torch.zeros(self.attn_ctas, **i32)
        self.err = torch.zeros(1, **i32)
        # the arguments that stay the same from call to call
        P, page = pool.num_pages, pool.page_size
        self._index, self._geometry = dev.index, (P, self.kv_heads, page, self.head_dim)
        at = {name: getattr(self, name).data_ptr() for name in ("cu_new", "slots", "positions", "kv_len", "items",
                                                                "counts", "cu_work", "attn_start")}
        status, table = pool.status.data_ptr(), pool.block_table.data_ptr()
        self._plan_args = N.PlanArgs(
            lengths=pool.lengths.data_ptr(), block_table=table, free_pages=pool.free_pages.data_ptr(),
            free_count=pool.free_count.data_ptr(), status=status, requests=R, table_width=pool.table_width, page=page,
            pages=P, max_tokens=self.max_tokens, kv_heads=self.kv_heads, group=self.q_heads // self.kv_heads,
            row_tile=self.row_tile, attn_ctas=self.attn_ctas, **at)
        self._write_args = N.CacheWriteArgs(
            items=at["items"], counts=at["counts"], cu_new=at["cu_new"], status=status, requests=R, pages=P, page=page,
            kv_heads=self.kv_heads, q_heads=self.q_heads, head_dim=self.head_dim)
        self._attn_args = N.PagedAttnArgs(
            block_table=table, cu_new=at["cu_new"], kv_len=at["kv_len"], cu_work=at["cu_work"],
            attn_start=at["attn_start"], counts=at["counts"], ws_o=self.ws_o.data_ptr(), ws_ml=self.ws_ml.data_ptr(),
            arrivals=self.arrivals.data_ptr(), err=self.err.data_ptr(), status=status, requests=R,
            table_width=pool.table_width, pages=P, page=page, kv_heads=self.kv_heads, q_heads=self.q_heads,
            head_dim=self.head_dim, row_tile=self.row_tile, attn_ctas=self.attn_ctas)

    @torch.inference_mode()
    def check_status(self) -> None:
        """Raise ``TileQuantError`` if a wait of ``attn_paged`` for a load gave up (that call's
        output is then undefined).  Reads the error word, which synchronises, and clears it."""
        st = int(self.err.item())
        if st:
            self.err.zero_()
            raise N.TileQuantError(f"attn_paged: a wait for a load of the cache ran out (status {st})")


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
    if plan.pool is not pool:
        raise ValueError("plan_step: the plan belongs to another pool")
    lengths_out = pool.lengths if lengths_out is None else lengths_out
    free_count_out = pool.free_count if free_count_out is None else free_count_out
    index = plan._index
    _check_state(new_lens, torch.int32, pool.max_requests, index, "plan_step: new_lens")
    _check_state(lengths_out, torch.int32, pool.max_requests, index, "plan_step: lengths_out")
    _check_state(free_count_out, torch.int32, 1, index, "plan_step: free_count_out")
    a = N.PlanArgs.from_buffer_copy(plan._plan_args)
    a.new_lens, a.lengths_out = new_lens.data_ptr(), lengths_out.data_ptr()
    a.free_count_out = free_count_out.data_ptr()
    N.check(N.on_device(index, N.load().tq_plan_step, ctypes.byref(a), N.raw_stream(index)), "plan_step")
    return plan


@traced("tq.release_requests")
def release_requests(finished: torch.Tensor, pool: PagePool) -> None:
    """Give back the pages of the requests with ``finished`` (bool or uint8 [max_requests]);
    their lengths become 0.  Table entries of -1 give nothing back.  A page that is free already
    is not freed again, and ``pool.check_status()`` tells; one that another request still holds
    is the caller's to take out of the row first."""
    if finished.dtype == torch.bool:
        finished = finished.view(torch.uint8)
    index = pool.device.index
    _check_state(finished, torch.uint8, pool.max_requests, index, "release_requests: finished")
    N.check(N.on_device(index, N.load().tq_release_requests, finished.data_ptr(), pool.lengths.data_ptr(),
                        pool.block_table.data_ptr(), pool.free_pages.data_ptr(), pool.free_count.data_ptr(),
                        pool.status.data_ptr(), pool.max_requests, pool.table_width, pool.page_size, pool.num_pages,
                        N.raw_stream(index)), "release_requests")


def _check_plan(plan: StepPlan, kv: KVPages, what: str) -> None:
    if kv._shape != plan._geometry:
        raise ValueError(f"{what}: the cache is {kv._shape} (pages, KV heads, page, head_dim), the plan's "
                         f"{plan._geometry}")
    if kv._index != plan._index:
        raise ValueError(f"{what}: the cache is on cuda:{kv._index}, the plan on cuda:{plan._index}")


@traced("tq.cache_write")
def cache_write(k: torch.Tensor, v: torch.Tensor, kv: KVPages, plan: StepPlan, q: Optional[torch.Tensor] = None,
                cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """The step's new keys and values (``k``, ``v`` [rows, kv_heads * D] views) into the
    pages of ``plan``.  With ``cos``/``sin`` ([rows, D], or one expanded row) and ``q`` ([rows,
    q_heads * D]), K is rotated first and the rotated q is returned (in ``q_out``, which may be
    ``q``; rows behind the last token as for ``attn_paged``'s output).

    Pages with new tokens behind the last of ``rows`` are left as they are, and
    ``pool.check_status()`` tells.  A page and head whose values outgrow its scale gets the larger scale, and the codes it
    holds are rounded again; NaN is stored as 0, an infinity as the page's largest value."""
    _check_plan(plan, kv, "cache_write")
    index, rows, dtype = plan._index, int(k.shape[0]), k.dtype
    code, width = N.dtype_code(dtype), plan.kv_heads * plan.head_dim
    a = N.CacheWriteArgs.from_buffer_copy(plan._write_args)
    a.ld_k = _check_rows(k, rows, width, dtype, index, "cache_write: k")
    a.ld_v = _check_rows(v, rows, width, dtype, index, "cache_write: v")
    if rows > plan.max_tokens:
        raise ValueError(f"cache_write: {rows} rows, the plan has {plan.max_tokens}")
    if not (q is None) == (cos is None) == (sin is None) or (q is None and q_out is not None):
        raise ValueError("cache_write: q, cos and sin come together")
    if q is not None:
        width = plan.q_heads * plan.head_dim
        a.ld_q = _check_rows(q, rows, width, dtype, index, "cache_write: q")
        a.ld_cs = _check_rows(cos, rows, plan.head_dim, dtype, index, "cache_write: cos", shared=True)
        if _check_rows(sin, rows, plan.head_dim, dtype, index, "cache_write: sin", shared=True) != a.ld_cs:
            raise ValueError("cache_write: cos and sin must share one row stride")
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            a.ld_qo, a.flags = width, N.TQ_CLEAR_REST
        else:
            a.ld_qo = _check_rows(q_out, rows, width, dtype, index, "cache_write: q_out")
        a.q, a.cos, a.sin, a.q_out = q.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_out.data_ptr()
    if rows == 0:
        return q_out
    a.k, a.v, a.rows = k.data_ptr(), v.data_ptr(), rows
    a.k_codes, a.v_codes, a.k_scale, a.v_scale = kv._ptrs
    N.check(N.on_device(index, N.load().tq_cache_write, ctypes.byref(a), code, N.raw_stream(index)), "cache_write")
    return q_out


@traced("tq.read_pages")
def read_pages(kv: KVPages, page_ids: torch.Tensor, dtype: torch.dtype, k_out: Optional[torch.Tensor] = None,
               v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 16-bit values of the pages ``page_ids`` (int32 [n], e.g. a block-table row): K and
    V [n, kv_heads, page_size, head_dim].  An id outside the pool (-1) gives zeros."""
    P, H, page, D = kv._shape
    index, code = kv._index, N.dtype_code(dtype)
    n = int(page_ids.shape[0]) if page_ids.dim() == 1 else -1
    _check_state(page_ids, torch.int32, n, index, "read_pages: page_ids")
    shape = (n, H, page, D)
    for t in (k_out, v_out):
        if t is not None and (t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != index):
            raise ValueError(f"read_pages: outputs must be contiguous {list(shape)} tensors of {dtype} on cuda:{index}")
    k_out = kv.k.new_empty(shape, dtype=dtype) if k_out is None else k_out
    v_out = torch.empty_like(k_out) if v_out is None else v_out
    if n:
        N.check(N.on_device(index, N.load().tq_read_pages, *kv._ptrs, page_ids.data_ptr(), n, P, H, page, D,
                            k_out.data_ptr(), v_out.data_ptr(), code, N.raw_stream(index)), "read_pages")
    return k_out, v_out


@traced("tq.attn_paged")
def attn_paged(q: torch.Tensor, kv: KVPages, plan: StepPlan, scale: float,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's token rows ``q`` ([rows, q_heads * D], rotated) over the pages:
    the i-th new token of a request sees its cached tokens and the new ones up to itself.
    Rows of a request that was not placed give zeros; rows behind the last token are left as
    they are in ``out``, which may be ``q``, and are zero in a tensor made here."""
    _check_plan(plan, kv, "attn_paged")
    index, rows, width, dtype = plan._index, int(q.shape[0]), plan.q_heads * plan.head_dim, q.dtype
    code = N.dtype_code(dtype)
    a = N.PagedAttnArgs.from_buffer_copy(plan._attn_args)
    a.ld_q = _check_rows(q, rows, width, dtype, index, "attn_paged: q")
    if rows > plan.max_tokens:
        raise ValueError(f"attn_paged: {rows} rows, the plan has {plan.max_tokens}")
    if not math.isfinite(scale):
        raise ValueError("attn_paged: scale must be finite")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a.ld_out, a.flags = width, N.TQ_CLEAR_REST
    else:
        a.ld_out = _check_rows(out, rows, width, dtype, index, "attn_paged: out")
    if rows == 0:
        return out
    a.q, a.out, a.rows, a.scale_log2 = q.data_ptr(), out.data_ptr(), rows, scale * LOG2E
    a.k_codes, a.v_codes, a.k_scale, a.v_scale = kv._ptrs
    N.check(N.on_device(index, N.load().tq_attn_paged, ctypes.byref(a), code, N.raw_stream(index)), "attn_paged")
    return out
