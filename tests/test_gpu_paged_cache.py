"""The paged 8-bit KV cache on the GPU against plain restatements: page planning and release
(whole numbers, equal), the write (codes and scales, equal), the read-back (equal), attention
(64-bit softmax over the cache's values, within the rounding errors counted in
``paged_reference.attend``), and whole steps captured and replayed."""

from __future__ import annotations

import math

import pytest
import torch

import tilequant_b200 as tq
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
BITS = {torch.bfloat16: torch.int16, torch.float16: torch.int16}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _check_plan(pool, plan, rp, want):
    assert plan.slots.tolist() == want["slots"]
    assert plan.positions.tolist() == want["positions"]
    assert plan.cu_new.tolist() == want["cu_new"]
    assert plan.kv_len.tolist() == want["kv_len"]
    assert pool.lengths.tolist() == rp.lengths
    assert pool.block_table.tolist() == rp.table
    assert int(pool.free_count) == len(rp.stack)
    assert pool.free_pages.tolist()[:len(rp.stack)] == rp.stack
    assert int(pool.status) == want["status"]


# ------------------------------------------------------------------ planning
@pytest.mark.parametrize("R,page,pages,max_len,max_tokens,steps", [
    (1, 16, 9, 100, 40, [[0], [1], [15], [16], [0], [17], [40]]),
    (3, 32, 20, 200, 300, [[1, 31, 64], [31, 1, 1], [0, 0, 0], [1, 1, 1], [-5, 2, 0], [100, 0, 0]]),
    (5, 64, 7, 256, 400, [[64, 65, 1, 0, 63], [1, 63, 1, 200, 1], [1, 1, 200, 1, 1], [1, 0, 0, 3, 200]]),  # pool empty
    (4, 16, 100, 48, 64, [[40, 49, 1, 8], [8, 48, 47, 0], [1, 1, 1, 1]]),  # a table row too short
    (4, 16, 100, 480, 10, [[4, 4, 4, 4], [1, 8, 1, 1], [11, 1, 1, 1]]),  # more tokens than rows
    (130, 128, 300, 1000, 9000, [[(i * 7) % 131 for i in range(130)], [1] * 130]),  # several CTAs
])
def test_plan_and_release_match_a_list_of_pages(cuda_device, R, page, pages, max_len, max_tokens, steps):
    pool = tq.PagePool(pages, R, max_len, page_size=page, device=cuda_device)
    plan = tq.StepPlan(pool, max_tokens, q_heads=4, kv_heads=2, head_dim=64)
    rp = ref.RefPool(pages, R, pool.table_width, page)
    for i, new in enumerate(steps):
        pool.status.zero_()
        tq.plan_step(_i32(new, cuda_device), pool, plan)
        _check_plan(pool, plan, rp, rp.step(new, max_tokens))
        if i % 2:
            done = [(r + i) % 3 == 0 for r in range(R)]
            tq.release_requests(torch.tensor(done, device=cuda_device), pool)
            rp.release(done)
            assert pool.lengths.tolist() == rp.lengths and pool.block_table.tolist() == rp.table
            assert pool.free_pages.tolist()[:len(rp.stack)] == rp.stack and int(pool.free_count) == len(rp.stack)


def test_plan_of_many_requests_and_rows(cuda_device):
    """4096 requests, more than one per thread, tokens over several CTAs."""
    R, page = 4096, 16
    g = torch.Generator().manual_seed(3)
    new = torch.randint(-1, 14, (R,), generator=g).tolist()
    pool = tq.PagePool(6000, R, 64, page_size=page, device=cuda_device)
    plan = tq.StepPlan(pool, 40000, q_heads=8, kv_heads=8, head_dim=64)
    rp = ref.RefPool(6000, R, pool.table_width, page)
    for _ in range(2):
        tq.plan_step(_i32(new, cuda_device), pool, plan)
        _check_plan(pool, plan, rp, rp.step(new, 40000))


def test_plan_leaves_the_pool_when_given_other_outputs(cuda_device):
    pool = tq.PagePool(10, 2, 64, page_size=16, device=cuda_device)
    plan = tq.StepPlan(pool, 40, q_heads=2, kv_heads=1, head_dim=64)
    lengths, count = torch.empty_like(pool.lengths), torch.empty_like(pool.free_count)
    for _ in range(2):  # the same step twice: the same result
        tq.plan_step(_i32([17, 0], cuda_device), pool, plan, lengths_out=lengths, free_count_out=count)
        assert lengths.tolist() == [17, 0] and int(count) == 8
        assert pool.lengths.tolist() == [0, 0] and int(pool.free_count) == 10
        assert pool.block_table[0].tolist() == [0, 1, -1, -1]


def test_status_is_reported_and_cleared(cuda_device):
    pool = tq.PagePool(1, 2, 64, page_size=16, device=cuda_device)
    plan = tq.StepPlan(pool, 40, q_heads=2, kv_heads=1, head_dim=64)
    tq.plan_step(_i32([16, 1], cuda_device), pool, plan)
    with pytest.raises(tq._native.TileQuantError, match="too few free pages"):
        pool.check_status()
    pool.check_status()
    pool.reset()
    assert int(pool.free_count) == 1 and pool.lengths.tolist() == [0, 0]


def test_a_page_given_back_twice_is_reported(cuda_device):
    pool = tq.PagePool(4, 2, 64, page_size=16, device=cuda_device)
    pool.lengths.copy_(_i32([64, 16], cuda_device))
    pool.block_table.copy_(_i32([[0, 1, 2, 3], [0, -1, -1, -1]], cuda_device))
    pool.free_count.zero_()
    tq.release_requests(torch.tensor([True, True], device=cuda_device), pool)
    assert int(pool.free_count) == 4 and int(pool.status) == ref.BAD_PAGE


def test_a_shared_page_taken_out_of_a_row_is_not_given_back(cuda_device):
    """Requests 1 and 2 read request 0's prompt; each but the last takes the shared pages out of its
    row before it goes, and every page is on the stack once in the end."""
    P, page, W = 1500, 16, 1300
    pool = tq.PagePool(P, 3, W * page, page_size=page, device=cuda_device)
    plan = tq.StepPlan(pool, W * page, q_heads=2, kv_heads=1, head_dim=64)
    tq.plan_step(_i32([1200 * page + 5, 0, 0], cuda_device), pool, plan)
    pool.block_table[1:, :1200] = pool.block_table[0, :1200]
    pool.lengths[1:] = 1200 * page
    tq.plan_step(_i32([0, 17, 33], cuda_device), pool, plan)
    own = [pool.block_table[r, 1200:1203].tolist() for r in range(3)]
    shared = pool.block_table[0, :1200].tolist()
    stack = pool.free_pages[:int(pool.free_count)].tolist()
    for r in (1, 0):
        pool.block_table[r, 0:1200:1 + r] = -1  # request 0 keeps none, 1 gives every other page back itself
        if r:
            pool.block_table[2, 1:1200:2] = -1
            pool.block_table[0, 1:1200:2] = -1
    tq.release_requests(torch.tensor([False, True, False], device=cuda_device), pool)
    stack += shared[1::2] + [i for i in own[1] if i >= 0]
    assert pool.free_pages[:int(pool.free_count)].tolist() == stack
    tq.release_requests(torch.tensor([True, False, False], device=cuda_device), pool)
    stack += [i for i in own[0] if i >= 0]
    assert pool.free_pages[:int(pool.free_count)].tolist() == stack
    tq.release_requests(torch.tensor([False, False, True], device=cuda_device), pool)
    stack += shared[0::2] + [i for i in own[2] if i >= 0]
    assert pool.free_pages[:int(pool.free_count)].tolist() == stack
    assert sorted(stack) == list(range(P)) and pool.lengths.tolist() == [0, 0, 0]
    pool.check_status()
    assert int(pool.block_table.max()) == -1


# ------------------------------------------------------------------ write and read
class Case:
    """A pool with ``before`` tokens per request, random codes everywhere, and one planned step."""

    def __init__(self, dev, dtype, hq, hk, d, page, before, new, seed, max_tokens=None, max_new=None, spare=3):
        g = _gen(dev, seed)
        self.dev, self.dtype, self.hq, self.hk, self.d, self.page = dev, dtype, hq, hk, d, page
        need = sum(-(-(b + max(n, 0)) // page) for b, n in zip(before, new))
        P = need + spare
        R = len(before)
        max_len = max(b + max(n, 0) for b, n in zip(before, new))
        self.pool = tq.PagePool(P, R, max(1, max_len), page_size=page, device=dev)
        self.rp = ref.RefPool(P, R, self.pool.table_width, page)
        ids = torch.randperm(P, generator=g, device=dev).tolist()
        self.rp.stack = ids
        self.rp.step(before, sum(before) + 1)
        self.pool.lengths.copy_(_i32(self.rp.lengths, dev))
        self.pool.block_table.copy_(_i32(self.rp.table, dev))
        self.pool.free_pages[:len(self.rp.stack)] = _i32(self.rp.stack, dev)
        self.pool.free_count.fill_(len(self.rp.stack))
        self.rows = sum(max(n, 0) for n in new)
        self.max_tokens = max_tokens or max(self.rows, 1)
        self.plan = tq.StepPlan(self.pool, self.max_tokens, q_heads=hq, kv_heads=hk, head_dim=d,
                                max_new=max_new or max(1, max(new)))
        self.kv = tq.KVPages(P, hk, page, d, device=dev)
        for t in (self.kv.k, self.kv.v):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device=dev).to(torch.int8))
        for t in (self.kv.k_scale, self.kv.v_scale):
            t.copy_(torch.rand(t.shape, generator=g, device=dev) * 0.03 + 0.002)
        tq.plan_step(_i32(new, dev), self.pool, self.plan)
        self.want = self.rp.step(new, self.max_tokens)
        _check_plan(self.pool, self.plan, self.rp, self.want)
        qkv = torch.randn(self.rows, (hq + 2 * hk) * d, generator=g, device=dev)
        qkv *= torch.exp(0.5 * torch.randn(self.rows, 1, generator=g, device=dev))
        qkv = qkv.to(dtype)
        self.q, self.k, self.v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        ang = torch.rand(self.rows, d // 2, generator=g, device=dev) * 6.3
        ang = torch.cat([ang, ang], 1)
        self.cos, self.sin = ang.cos().to(dtype), ang.sin().to(dtype)
        self.scale = d ** -0.5

    def reference_cache(self):
        return [t.clone() for t in (self.kv.k, self.kv.v, self.kv.k_scale, self.kv.v_scale)]

    def check_cache(self, want):
        for got, w, name in zip((self.kv.k, self.kv.v, self.kv.k_scale, self.kv.v_scale), want, "k v ks vs".split()):
            assert torch.equal(got, w), (name, int((got != w).sum()))

    def attend(self, **kw):
        return tq.attn_paged(self.q, self.kv, self.plan, self.scale, **kw)

    def check_attention(self, got, q=None):
        want, tol = ref.attend(self.q if q is None else q, self.kv.k, self.kv.v, self.kv.k_scale, self.kv.v_scale,
                               self.rp.table, self.want["cu_new"], self.want["kv_len"], self.scale,
                               torch.finfo(self.dtype).eps)
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))


WRITES = [
    # hq, hk, d, page, tokens before, new tokens
    (4, 2, 64, 16, [0, 1, 15, 16, 17, 31], [1, 1, 1, 1, 1, 1]),
    (4, 2, 64, 16, [0, 5, 16, 33, 7], [37, 16, 1, 0, 90]),
    (3, 1, 128, 32, [31, 32, 0, 64], [1, 33, 64, 31]),
    (8, 8, 128, 64, [63, 1, 0], [2, 62, 200]),
    (7, 1, 64, 64, [100], [1]),
    (5, 5, 128, 128, [127, 0, 5], [130, 128, 0]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("hq,hk,d,page,before,new", WRITES)
def test_write_stores_the_codes_and_scales_of_the_definition(cuda_device, dtype, turn, hq, hk, d, page, before, new):
    c = Case(cuda_device, dtype, hq, hk, d, page, before, new, seed=hq + page)
    want = c.reference_cache()
    k, v = c.k.reshape(-1, hk, d), c.v.reshape(-1, hk, d).double()
    k = ref.rotate(k, c.cos, c.sin) if turn else k.double()
    ref.write_side(k, want[0], want[2], c.want["slots"], c.want["positions"])
    ref.write_side(v, want[1], want[3], c.want["slots"], c.want["positions"])
    if turn:
        q = tq.cache_write(c.k, c.v, c.kv, c.plan, q=c.q, cos=c.cos, sin=c.sin)
        assert torch.equal(q.double().view(-1, hq, d), ref.rotate(c.q.reshape(-1, hq, d), c.cos, c.sin))
    else:
        assert tq.cache_write(c.k, c.v, c.kv, c.plan) is None
    c.check_cache(want)
    c.pool.check_status()
    # a second write of the same step finds its own scales and stores the same codes
    tq.cache_write(c.k, c.v, c.kv, c.plan, **(dict(q=c.q, cos=c.cos, sin=c.sin) if turn else {}))
    c.check_cache(want)


def test_rotated_queries_may_replace_the_queries(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 6, 2, 128, 16, [3, 20], [5, 1], seed=4)
    q = c.q.contiguous()
    want = tq.cache_write(c.k, c.v, c.kv, c.plan, q=q.clone(), cos=c.cos, sin=c.sin)
    assert tq.cache_write(c.k, c.v, c.kv, c.plan, q=q, cos=c.cos, sin=c.sin, q_out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_zeros_infinities_nan_and_the_smallest_values(cuda_device, dtype):
    c = Case(cuda_device, dtype, 2, 2, 64, 16, [0, 0, 8, 8, 0, 0], [4, 4, 4, 4, 4, 4], seed=9)
    k = c.k.clone()
    k[0:4] = 0  # a page of zeros: scale 0
    k[4:8, 3], k[4:8, 5], k[4:8, 7] = math.inf, -math.inf, math.nan
    k[8:12] = math.nan  # nothing finite: the held codes stay
    k[12:16] = 0
    k[16:20] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # the smallest subnormal
    k[20:24] = torch.finfo(dtype).max * torch.sign(k[20:24].float()).to(dtype)
    want = c.reference_cache()
    ref.write_side(k.view(-1, 2, 64).double(), want[0], want[2], c.want["slots"], c.want["positions"])
    ref.write_side(c.v.reshape(-1, 2, 64).double(), want[1], want[3], c.want["slots"], c.want["positions"])
    tq.cache_write(k, c.v, c.kv, c.plan)
    c.check_cache(want)
    pg = c.want["slots"][0] // 16
    assert float(c.kv.k_scale[pg].abs().max()) == 0.0


def test_a_page_filled_token_by_token_keeps_its_values_within_its_steps(cuda_device):
    """31 single tokens of growing size into two pages: every re-rounding is off by half a step
    of the scale at that time, and the scales grow, so at most the sum of the half steps."""
    dev, d = cuda_device, 64
    pool = tq.PagePool(4, 1, 64, page_size=16, device=dev)
    plan = tq.StepPlan(pool, 1, q_heads=1, kv_heads=1, head_dim=d)
    kv = tq.KVPages(4, 1, 16, d, device=dev)
    g = _gen(dev, 2)
    x = (torch.randn(31, d, generator=g, device=dev) * torch.linspace(0.1, 3, 31, device=dev)[:, None]).half()
    room = torch.zeros(31, device=dev)
    for t in range(31):
        tq.plan_step(_i32([1], dev), pool, plan)
        before = kv.k_scale.clone()
        tq.cache_write(x[t:t + 1], x[t:t + 1], kv, plan)
        pg = int(pool.block_table[0, t // 16])
        if t % 16 == 0 or float(kv.k_scale[pg, 0]) > float(before[pg, 0]):
            room[t // 16 * 16:t] += float(kv.k_scale[pg, 0]) / 2 * 1.001
        room[t] += float(kv.k_scale[pg, 0]) / 2 * 1.001
    k, v = tq.read_pages(kv, pool.block_table[0, :2].contiguous(), torch.float16)
    got = k[:, 0].reshape(32, d)[:31].float()
    slack = room[:, None] + got.abs() * 2.0**-11  # the read-back's own rounding
    assert bool(((got - x.float()).abs() <= slack).all())
    assert torch.equal(k, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,page,hk", [(64, 16, 3), (128, 128, 1), (128, 32, 8)])
def test_read_pages_gives_code_times_scale(cuda_device, dtype, d, page, hk):
    c = Case(cuda_device, dtype, hk, hk, d, page, [page + 1], [1], seed=d + page, spare=5)
    ids = _i32([2, -1, 0, c.kv.k.shape[0], 2, 1], cuda_device)
    k, v = tq.read_pages(c.kv, ids, dtype)
    for got, codes, scale in ((k, c.kv.k, c.kv.k_scale), (v, c.kv.v, c.kv.v_scale)):
        want = (codes.double() * scale.double()[..., None, None]).float().to(dtype)
        for i, p in enumerate(ids.tolist()):
            if 0 <= p < codes.shape[0]:
                assert torch.equal(got[i], want[p])
            else:
                assert not bool(got[i].any())
    e = tq.read_pages(c.kv, ids[:0], dtype)
    assert e[0].shape == (0, hk, page, d)


def test_write_skips_bad_pages_and_reports_them(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 2, 2, 64, 16, [3, 3, 3], [1, 1, 1], seed=5)
    c.plan.items[1, 3] = c.kv.k.shape[0]  # the plan's own list, damaged
    want = c.reference_cache()
    slots = list(c.want["slots"])
    slots[1] = -1
    ref.write_side(c.k.reshape(-1, 2, 64).double(), want[0], want[2], slots, c.want["positions"])
    ref.write_side(c.v.reshape(-1, 2, 64).double(), want[1], want[3], slots, c.want["positions"])
    tq.cache_write(c.k, c.v, c.kv, c.plan)
    c.check_cache(want)
    with pytest.raises(tq._native.TileQuantError, match="page id"):
        c.pool.check_status()


@pytest.mark.parametrize("rows", [1, 3, 22, 43])
def test_a_write_with_too_few_rows_is_reported(cuda_device, rows):
    """Pages whose rows are all there are written, the others stay."""
    c = Case(cuda_device, torch.bfloat16, 2, 2, 64, 16, [3, 14, 0], [3, 21, 20], seed=6)
    want = c.reference_cache()
    slots, pages = list(c.want["slots"]), [s // 16 for s in c.want["slots"]]
    for i, p in enumerate(pages):
        if p in pages[rows:]:
            slots[i] = -1
    ref.write_side(c.k.reshape(-1, 2, 64).double(), want[0], want[2], slots, c.want["positions"])
    ref.write_side(c.v.reshape(-1, 2, 64).double(), want[1], want[3], slots, c.want["positions"])
    tq.cache_write(c.k[:rows], c.v[:rows], c.kv, c.plan)
    c.check_cache(want)
    with pytest.raises(tq._native.TileQuantError, match="cache_write"):
        c.pool.check_status()


# ------------------------------------------------------------------ attention
ATTENDS = [
    # hq, hk, d, page, tokens before, new tokens
    (1, 1, 64, 16, [0], [1]),
    (4, 2, 64, 16, [0, 1, 15, 16, 31, 32, 127, 128], [1] * 8),
    (7, 1, 128, 32, [31, 126, 127, 128, 129, 255, 700], [1] * 7),
    (28, 4, 128, 64, [0, 63, 64, 1000, 5, 200], [1, 1, 1, 1, 0, 1]),
    (24, 8, 128, 128, [2047, 1], [1, 1]),
    (8, 8, 64, 64, [4095], [1]),
    (16, 1, 128, 16, [77, 300], [1, 1]),  # 16 query heads per KV head
    (40, 8, 128, 32, [500, 0, 31, 129], [3, 4, 1, 2]),
    (12, 2, 64, 16, [0, 40, 3], [37, 16, 5]),  # several row tiles
    (48, 2, 128, 64, [100], [1]),  # 24 query heads per KV head
    (20, 4, 128, 128, [0, 511], [130, 9]),  # a prompt and a draft in one step
    (6, 6, 64, 32, [300] * 70, [1] * 70),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d,page,before,new", ATTENDS)
def test_attention_matches_a_64_bit_softmax(cuda_device, dtype, hq, hk, d, page, before, new):
    c = Case(cuda_device, dtype, hq, hk, d, page, before, new, seed=hq * 3 + page)
    out = c.attend()
    c.check_attention(out)
    assert int(c.plan.err) == 0 and not bool(c.plan.arrivals.any())
    assert torch.equal(c.attend().view(torch.int16), out.view(torch.int16))  # the same bits again
    c.pool.check_status()


@pytest.mark.parametrize("max_new", [1, 2, 8])
def test_every_row_tile_gives_the_result(cuda_device, max_new):
    """The row tile follows from max_new; requests with more tokens than it take several."""
    c = Case(cuda_device, torch.bfloat16, 15, 3, 128, 32, [90, 260, 0], [5, 1, 9], seed=1, max_new=max_new)
    assert c.plan.row_tile == {1: 8, 2: 16, 8: 16}[max_new]
    c.check_attention(c.attend())


def test_rows_without_a_place_are_zero_and_rows_behind_stay(cuda_device):
    dev = cuda_device
    c = Case(dev, torch.bfloat16, 4, 2, 64, 16, [20, 16, 33], [1, 1, 1], seed=8, max_tokens=7, spare=0)
    c.pool.lengths.copy_(_i32([20, 16, 33], dev))
    c.rp.lengths = [20, 16, 33]
    c.pool.free_count.zero_()  # request 1 needs a page and finds none
    c.rp.stack = []
    c.pool.status.zero_()
    tq.plan_step(_i32([1, 1, 1], dev), c.pool, c.plan)
    c.want = c.rp.step([1, 1, 1], 7)
    assert c.want["kv_len"] == [21, 0, 34] and c.plan.kv_len.tolist() == c.want["kv_len"]
    q = torch.randn(7, 4 * 64, device=dev).bfloat16()
    out = torch.full_like(q, 7.0)
    tq.attn_paged(q, c.kv, c.plan, c.scale, out=out)
    assert not bool(out[1].any()) and bool((out[3:] == 7.0).all())
    c.check_attention(out[:3], q=q[:3])
    kv = c.reference_cache()
    tq.cache_write(q[:, :128], q[:, 128:], c.kv, c.plan)  # rows behind the last token are not written
    changed = (c.kv.k != kv[0]).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {c.rp.table[0][1], c.rp.table[2][2]}


def test_only_the_keys_in_use_are_read(cuda_device):
    """NaN scales on pages nobody holds and wild codes behind the last key change nothing."""
    c = Case(cuda_device, torch.float16, 8, 2, 128, 32, [40, 31, 95], [1, 1, 2], seed=3, spare=6)
    out = c.attend()
    held = {p for r, n in enumerate(c.want["kv_len"]) for p in c.rp.table[r][:-(-n // 32)]}
    for p in range(c.kv.k.shape[0]):
        if p not in held:
            for t in (c.kv.k_scale, c.kv.v_scale):
                t[p] = math.nan
            c.kv.k[p] = c.kv.v[p] = -128
    for r, n in enumerate(c.want["kv_len"]):
        if n % 32:
            for t in (c.kv.k, c.kv.v):
                t[c.rp.table[r][n // 32], :, n % 32:] = -128
    assert torch.equal(c.attend().view(torch.int16), out.view(torch.int16))


def test_a_query_of_infinities_or_nan_spoils_its_own_row_only(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 4, 2, 64, 16, [50, 70], [2, 1], seed=6)
    clean = c.attend()
    q = c.q.clone()
    q[1, 64 + 5] = math.nan  # token 1, head 1
    q[2, 130] = math.inf  # token 2, head 2
    c.q = q
    got = c.attend().view(3, 4, 64)
    clean = clean.view(3, 4, 64)
    for t in range(3):
        for h in range(4):
            if (t, h) in ((1, 1), (2, 2)):
                assert bool(torch.isnan(got[t, h]).all())
            else:
                assert torch.equal(got[t, h], clean[t, h])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-4, 300.0])
def test_small_and_large_queries_keep_their_precision(cuda_device, dtype, size):
    """Query rows are scaled to f16's range each, so their size does not matter.  (f16 itself
    holds nothing at 1e-30.)"""
    c = Case(cuda_device, dtype, 6, 2, 64, 32, [100, 300], [1, 1], seed=7)
    c.q = (c.q.float() * size).to(dtype)
    c.scale = 0.125 / size if size < 1 else 0.125 / size / 4
    c.check_attention(c.attend())


def test_strided_queries_and_outputs(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 4, 4, 64, 16, [30, 60, 90], [1, 1, 1], seed=2)
    want = c.attend()
    wide = torch.zeros(3, 1000, device=cuda_device, dtype=torch.bfloat16)
    got = c.attend(out=wide[:, 8:8 + 256])
    assert torch.equal(got, want) and not bool(wide[:, :8].any()) and not bool(wide[:, 264:].any())
    one = Case(cuda_device, torch.bfloat16, 4, 4, 64, 16, [30], [1], seed=2)
    assert one.attend().shape == (1, 256)


@pytest.mark.parametrize("hq,hk,d,before,new", [
    (28, 4, 128, [4000, 61, 129, 1], [1, 1, 1, 1]),  # groups split over many blocks
    (8, 2, 64, [300, 0, 5], [90, 200, 1]),  # several passes of query rows
    (16, 1, 128, [9000], [4]),
])
def test_outputs_may_replace_the_queries(cuda_device, hq, hk, d, before, new):
    c = Case(cuda_device, torch.bfloat16, hq, hk, d, 64, before, new, seed=21)
    want = c.attend()
    c.check_attention(want)
    for _ in range(5):
        q = c.q.contiguous()
        assert tq.attn_paged(q, c.kv, c.plan, c.scale, out=q) is q
        assert torch.equal(q, want)


def test_requests_may_share_pages_they_only_read(cuda_device):
    """Two requests with the same prompt: the full prompt pages are one copy."""
    c = Case(cuda_device, torch.bfloat16, 8, 2, 64, 16, [64, 64], [1, 1], seed=12)
    c.pool.block_table[1, :4] = c.pool.block_table[0, :4]
    c.rp.table[1][:4] = c.rp.table[0][:4]
    c.check_attention(c.attend())


def test_bad_page_ids_are_masked_and_reported(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 8, 2, 128, 32, [200, 40], [1, 1], seed=13)
    out = c.attend()
    c.pool.block_table[0, 2] = c.kv.k.shape[0] + 5
    c.pool.block_table[0, 3] = -1
    got = c.attend()
    assert torch.equal(got[1], out[1]) and bool(torch.isfinite(got[0].float()).all())
    with pytest.raises(tq._native.TileQuantError, match="page id"):
        c.pool.check_status()


def test_long_caches_pass_32_bit_offsets(cuda_device):
    """A pool of 4.6e9 code bytes a side, its pages used from the far end."""
    dev, hk, d, page, P = cuda_device, 4, 128, 64, 140000
    if torch.cuda.mem_get_info(dev)[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    pool = tq.PagePool(P, 2, 40000, page_size=page, device=dev)
    pool.free_pages.copy_(torch.arange(P, dtype=torch.int32, device=dev))  # the last page goes first
    plan = tq.StepPlan(pool, 33000, q_heads=hk, kv_heads=hk, head_dim=d)
    kv = tq.KVPages(P, hk, page, d, device=dev)
    new = [32770, 130]
    rp = ref.RefPool(P, 2, pool.table_width, page)
    rp.stack = list(range(P))
    tq.plan_step(_i32(new, dev), pool, plan)
    rp.step(new, 33000)
    g = _gen(dev, 1)
    x = torch.randn(32900, 2 * hk * d, generator=g, device=dev).bfloat16()
    tq.cache_write(x[:, :hk * d], x[:, hk * d:], kv, plan)
    one = tq.StepPlan(pool, 2, q_heads=hk, kv_heads=hk, head_dim=d)
    tq.plan_step(_i32([1, 1], dev), pool, one)
    want = rp.step([1, 1], 2)
    y = torch.randn(2, 3 * hk * d, generator=g, device=dev).bfloat16()
    tq.cache_write(y[:, hk * d:2 * hk * d], y[:, 2 * hk * d:], kv, one)
    out = tq.attn_paged(y[:, :hk * d], kv, one, d ** -0.5)
    ref_out, tol = ref.attend(y[:, :hk * d], kv.k, kv.v, kv.k_scale, kv.v_scale, rp.table, want["cu_new"],
                              want["kv_len"], d ** -0.5, 2.0**-7)
    assert bool(((out.double() - ref_out).abs() <= tol).all())
    k, _ = tq.read_pages(kv, pool.block_table[0, :3].contiguous(), torch.bfloat16)
    top = x[:192, :hk * d].view(3, page, hk, d).transpose(1, 2)
    step = kv.k_scale[pool.block_table[0, :3].long()][..., None, None]
    assert bool(((k.float() - top.float()).abs() <= step * 0.51 + top.float().abs() * 2.0**-8).all())


# ------------------------------------------------------------------ whole steps
def _steps(dev, pool, plan, kv, x, cos, sin, new, hq, hk, d, out):
    tq.plan_step(new, pool, plan)
    q = tq.cache_write(x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:], kv, plan, q=x[:, :hq * d], cos=cos, sin=sin)
    return tq.attn_paged(q, kv, plan, d ** -0.5, out=out)


def test_a_captured_step_replays_as_eager_steps(cuda_device):
    """Forty decode steps of five requests, two of them starting late and one ending early,
    through one captured step; the pool, cache and outputs equal the eager run's."""
    dev, hq, hk, d, page, R = cuda_device, 8, 2, 64, 16, 5
    results = []
    for captured in (False, True):
        g = _gen(dev, 5)
        pool = tq.PagePool(30, R, 80, page_size=page, device=dev)
        plan = tq.StepPlan(pool, R, q_heads=hq, kv_heads=hk, head_dim=d)
        kv = tq.KVPages(30, hk, page, d, device=dev)
        new = torch.ones(R, dtype=torch.int32, device=dev)
        x = torch.zeros(R, (hq + 2 * hk) * d, device=dev, dtype=torch.bfloat16)
        cos, sin = torch.ones(R, d, device=dev).bfloat16(), torch.zeros(R, d, device=dev).bfloat16()
        out = torch.zeros(R, hq * d, device=dev, dtype=torch.bfloat16)
        run = lambda: _steps(dev, pool, plan, kv, x, cos, sin, new, hq, hk, d, out)  # noqa: E731
        if captured:
            run()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                run()
            pool.reset()
            for t in (kv.k, kv.v, kv.k_scale, kv.v_scale):
                t.zero_()
        outs = []
        for i in range(40):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
            live = [i < 25, True, i >= 7, i >= 19, True]
            new.copy_(_i32([int(v) for v in live], dev))
            out.zero_()
            graph.replay() if captured else run()
            outs.append(out.clone())
            if i == 25:
                tq.release_requests(torch.tensor([True, False, False, False, False], device=dev), pool)
        pool.check_status()
        results.append((torch.stack(outs), kv.k.clone(), kv.v_scale.clone(), pool.block_table.clone(),
                        pool.lengths.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][4].tolist() == [0, 40, 33, 21, 40]


def test_a_side_stream_gives_the_same(cuda_device):
    c = Case(cuda_device, torch.bfloat16, 8, 2, 128, 64, [300, 5000], [1, 1], seed=21)
    want = c.attend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_many_requests_most_of_them_idle(cuda_device):
    """1500 slots, runs of idle ones longer than a warp between the live, several blocks each."""
    before, new = [0] * 1500, [0] * 1500
    for r, b in ((0, 5), (1, 0), (40, 130), (41, 17), (700, 1000), (701, 3), (1499, 250)):
        before[r], new[r] = b, 1
    c = Case(cuda_device, torch.bfloat16, 8, 2, 64, 16, before, new, seed=17)
    c.check_attention(c.attend())
    want = c.reference_cache()
    ref.write_side(c.k.reshape(-1, 2, 64).double(), want[0], want[2], c.want["slots"], c.want["positions"])
    ref.write_side(c.v.reshape(-1, 2, 64).double(), want[1], want[3], c.want["slots"], c.want["positions"])
    tq.cache_write(c.k, c.v, c.kv, c.plan)
    c.check_cache(want)


def test_one_angle_for_all_rows(cuda_device):
    c = Case(cuda_device, torch.float16, 4, 2, 64, 16, [5, 9, 30], [1, 1, 1], seed=18)
    cos, sin = (t[:1].expand(3, -1) for t in (c.cos, c.sin))
    want = c.reference_cache()
    ref.write_side(ref.rotate(c.k.reshape(-1, 2, 64), cos, sin), want[0], want[2], c.want["slots"], c.want["positions"])
    ref.write_side(c.v.reshape(-1, 2, 64).double(), want[1], want[3], c.want["slots"], c.want["positions"])
    q = tq.cache_write(c.k, c.v, c.kv, c.plan, q=c.q, cos=cos, sin=sin)
    c.check_cache(want)
    assert torch.equal(q.double().view(-1, 4, 64), ref.rotate(c.q.reshape(-1, 4, 64), cos, sin))


def test_calls_that_are_refused(cuda_device):
    dev = cuda_device
    c = Case(dev, torch.bfloat16, 4, 2, 64, 16, [5, 9], [1, 1], seed=1)
    other = Case(dev, torch.bfloat16, 4, 2, 64, 32, [5, 9], [1, 1], seed=1)
    bad = [
        (lambda: tq.plan_step(_i32([1, 1], dev), c.pool, other.plan), "another pool"),
        (lambda: tq.plan_step(_i32([1], dev), c.pool, c.plan), "new_lens"),
        (lambda: tq.plan_step(_i32([1, 1], dev).long(), c.pool, c.plan), "new_lens"),
        (lambda: tq.plan_step(_i32([1, 1], "cpu"), c.pool, c.plan), "no CPU path"),
        (lambda: tq.release_requests(torch.zeros(3, device=dev, dtype=torch.bool), c.pool), "finished"),
        (lambda: tq.cache_write(c.k, c.v, other.kv, c.plan), "the cache is"),
        (lambda: tq.cache_write(c.k, c.v.half(), c.kv, c.plan), "cache_write: v"),
        (lambda: tq.cache_write(c.k.float(), c.v.float(), c.kv, c.plan), "float32"),
        (lambda: tq.cache_write(c.k.cpu(), c.v, c.kv, c.plan), "no CPU path"),
        (lambda: tq.cache_write(c.k, c.v, c.kv, c.plan, cos=c.cos, sin=c.sin), "come together"),
        (lambda: tq.cache_write(c.k, c.v, c.kv, c.plan, q=c.q[:, :128], cos=c.cos, sin=c.sin), "cache_write: q"),
        (lambda: tq.cache_write(c.k[:, ::2], c.v, c.kv, c.plan), "cache_write: k"),
        (lambda: tq.cache_write(c.k.repeat(3, 1), c.v.repeat(3, 1), c.kv, c.plan), "rows"),
        (lambda: tq.cache_write(c.k[:1].expand(2, -1), c.v, c.kv, c.plan), "overlap"),
        (lambda: tq.attn_paged(c.q.repeat(2, 1), c.kv, c.plan, 0.1), "rows"),
        (lambda: tq.attn_paged(c.q, c.kv, c.plan, math.inf), "finite"),
        (lambda: tq.attn_paged(c.q, c.kv, c.plan, 0.1, out=c.q.half()), "attn_paged: out"),
        (lambda: tq.attn_paged(torch.zeros(2, 257, device=dev, dtype=torch.bfloat16)[:, 1:], c.kv, c.plan, 0.1), "16-byte"),
        (lambda: tq.read_pages(c.kv, _i32([[0]], dev), torch.bfloat16), "page_ids"),
        (lambda: tq.read_pages(c.kv, _i32([0], dev), torch.float32), "float32"),
        (lambda: tq.read_pages(c.kv, _i32([0], dev), torch.float16, k_out=torch.zeros(1, device=dev).half()), "outputs"),
    ]
    before = c.reference_cache() + [c.pool.lengths.clone(), c.pool.block_table.clone()]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(AttributeError, match="copy into it"):
        c.pool.lengths = _i32([0, 0], dev)
    after = c.reference_cache() + [c.pool.lengths, c.pool.block_table]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
