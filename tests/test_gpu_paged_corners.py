"""The paged 8-bit cache on the GPU where its use can go wrong: pages given back more than once, rows
behind the step's last token."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

import tilequant_b200 as tq
from tests import paged_reference as ref
from tests.golden import inputs as I
from tests.test_gpu_paged_cache import Case

pytestmark = pytest.mark.gpu


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _mask(values, dev):
    return torch.tensor(values, dtype=torch.bool, device=dev)


def _stack(pool):
    return pool.free_pages[:int(pool.free_count)].tolist()


# ------------------------------------------------------------------ release
def test_a_page_given_back_by_both_of_its_readers_is_free_once(cuda_device):
    dev = cuda_device
    pool = tq.PagePool(20, 4, 64, page_size=16, device=dev)
    plan = tq.StepPlan(pool, 200, q_heads=2, kv_heads=1, head_dim=64)
    tq.plan_step(_i32([32, 0, 40, 32], dev), pool, plan)  # pages 0 1, 2 3 4, 5 6 stay in use
    pool.block_table[1, :2] = pool.block_table[0, :2]
    pool.lengths[1] = 32
    tq.release_requests(_mask([1, 0, 0, 0], dev), pool)
    assert int(pool.status) == 0
    stack = list(range(19, 6, -1)) + [0, 1]
    assert _stack(pool) == stack
    tq.release_requests(_mask([0, 1, 0, 0], dev), pool)
    assert _stack(pool) == stack and pool.lengths.tolist() == [0, 0, 40, 32]
    assert pool.block_table[:2].tolist() == [[-1] * 4] * 2
    with pytest.raises(tq._native.TileQuantError, match="free page given back"):
        pool.check_status()
    tq.plan_step(_i32([32, 32, 0, 0], dev), pool, plan)
    assert pool.block_table[:2, :2].tolist() == [[1, 0], [7, 8]]
    pool.check_status()


@pytest.mark.parametrize("R,W,P", [(2, 4, 9), (70, 40, 1500), (3, 1500, 6000), (5, 7, (1 << 20) + 77), (4, 900, 3 << 20)])
def test_release_of_shared_and_free_pages_matches_a_list(cuda_device, R, W, P):
    """Rows with ids from a small range (so that many meet, in one turn of 1024 entries and across
    turns), some already on the stack, some outside the pool; the first of equal entries counts."""
    dev, page = cuda_device, 16
    g = torch.Generator().manual_seed(R + W)
    pool = tq.PagePool(P, R, W * page, page_size=page, device=dev)
    some = torch.randperm(P, generator=g)[:min(P, R * W)]
    for turn in range(3):
        stack = torch.randperm(P, generator=g)[:P * turn // 3].tolist()
        pool.free_pages[:len(stack)] = _i32(stack, dev)
        pool.free_count.fill_(len(stack))
        pool.status.zero_()
        table = some[torch.randint(0, len(some), (R, W), generator=g)].int()
        table[torch.rand(R, W, generator=g) < 0.1] = -1
        if turn == 1:
            table[0, 0], table[-1, 1] = P, -7
        lengths = torch.randint(0, W * page + 1, (R,), generator=g).int()
        lengths[0] = lengths[-1] = W * page
        finished = torch.rand(R, generator=g) < 0.8
        finished[0] = finished[-1] = True
        pool.lengths.copy_(lengths)
        pool.block_table.copy_(table)
        tq.release_requests(finished.to(dev), pool)
        free, bad = set(stack), False
        for r in range(R):
            if not bool(finished[r]):
                continue
            for i in range(-(-int(lengths[r]) // page)):
                e = int(table[r, i])
                table[r, i] = -1
                if e == -1:
                    continue
                if e < 0 or e >= P or e in free:
                    bad = True
                    continue
                free.add(e)
                stack.append(e)
            lengths[r] = 0
        assert _stack(pool) == stack
        assert pool.block_table.tolist() == table.tolist() and pool.lengths.tolist() == lengths.tolist()
        assert int(pool.status) == (ref.BAD_PAGE if bad else 0)


def test_release_in_a_captured_step(cuda_device):
    """Captured as the first call of its kind, with a pool that needs the larger shared memory."""
    dev = cuda_device
    pool = tq.PagePool(900000, 2, 64, page_size=16, device=dev)
    plan = tq.StepPlan(pool, 64, q_heads=2, kv_heads=1, head_dim=64)
    new, done = _i32([20, 20], dev), _mask([0, 0], dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tq.release_requests(done, pool)
        tq.plan_step(new, pool, plan)
    graph.replay()
    assert pool.lengths.tolist() == [20, 20] and pool.block_table[:, :2].tolist() == [[0, 1], [2, 3]]
    done.copy_(_mask([1, 0], dev))
    graph.replay()
    assert pool.lengths.tolist() == [20, 40] and pool.block_table[:, :3].tolist() == [[1, 0, -1], [2, 3, 4]]
    pool.check_status()


# ------------------------------------------------------------------ rows behind the last token
def _linear(m, k):
    """A MixedLinear of m x k weights, a tenth of its tiles 16-bit."""
    cfg = SimpleNamespace(tile_m=64, tile_n=64, pad_to_tile=True, quant_style="gi", dtype_out="bf16")
    w = I.weight(m, k, 3).to("cuda")
    n = (m // 64) * (k // 64)
    keep = I.keep_ids(m // 64, k // 64, 0.1, 4)
    return tq.MixedLinear(tq.pack_weight_from_tile_ids(w, n_tr=m // 64, n_tc=k // 64, cfg=cfg, fp16_tile_ids=keep,
                                                       int8_tile_ids=I.complement_ids(keep, n)), None, cfg)


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("rows", [5, 40, 700])
def test_spare_rows_of_a_captured_step_do_not_reach_the_real_ones(cuda_device, hq, hk, d, rows):
    """A step captured with spare rows, replayed with fewer and fewer requests: the rows behind the last
    token are zero whatever they held, so the output projection's activation scales, maxima over all
    rows, and the real rows' codes are those of the real rows alone.  Outputs the caller brings keep theirs."""
    dev, page, R = cuda_device, 16, 5
    pool = tq.PagePool(60, R, 160, page_size=page, device=dev)
    plan = tq.StepPlan(pool, rows, q_heads=hq, kv_heads=hk, head_dim=d)
    kv = tq.KVPages(60, hk, page, d, device=dev)
    proj = _linear(128, hq * d)
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(rows, (hq + 2 * hk) * d, generator=g, device=dev).bfloat16()
    cos, sin = torch.ones(rows, d, device=dev).bfloat16(), torch.zeros(rows, d, device=dev).bfloat16()
    new = torch.ones(R, dtype=torch.int32, device=dev)

    def step():
        tq.plan_step(new, pool, plan)
        q = tq.cache_write(x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:], kv, plan, q=x[:, :hq * d], cos=cos, sin=sin)
        out = tq.attn_paged(q, kv, plan, d ** -0.5)
        return q, out, proj(out)

    with torch.inference_mode():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, out, y = step()
        for counts in ([1] * 5, [1, 0, 1, 1, 0], [0, 0, 0, 1, 0], [0] * 5, [0, 2, 0, 0, 1]):
            new.copy_(_i32(counts, dev))
            for t in (q, out, y):
                t.fill_(float("nan"))
            graph.replay()
            n = sum(counts)
            assert bool(torch.isfinite(out).all()) and not bool(out[n:].any()) and not bool(q[n:].any())
            if n:
                assert bool(out[:n].any()) and torch.equal(q[:n], x[:n, :hq * d])
                codes, scales = tq.quantize_activation_tile_absmax(out)
                alone, alone_scales = tq.quantize_activation_tile_absmax(out[:n].contiguous())
                assert torch.equal(codes[:n], alone) and torch.equal(scales, alone_scales)
                assert torch.equal(y, proj(out)) and bool(torch.isfinite(y).all())
            held = [torch.full_like(t, 7.0) for t in (q, out)]
            tq.cache_write(x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:], kv, plan, q=x[:, :hq * d], cos=cos, sin=sin,
                           q_out=held[0])
            tq.attn_paged(held[0], kv, plan, d ** -0.5, out=held[1])
            assert all(bool((t[n:] == 7.0).all()) for t in held)
            if n:
                assert torch.equal(held[1][:n], out[:n])
    pool.check_status()
    plan.check_status()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("size", [0.5, 2.0, 6.0])
@pytest.mark.parametrize("hq,hk,d,page,before,new", [
    (16, 2, 64, 16, [0, 1, 15, 16, 40, 512], [1] * 6),
    (28, 4, 128, 64, [3, 63, 64, 1000, 5], [1] * 5),
    (40, 8, 128, 32, [500, 0, 31], [3, 4, 1]),
    (20, 4, 64, 128, [0, 511], [130, 9]),
])
def test_f16_attention_is_off_by_little_more_than_its_outputs_rounding(cuda_device, hq, hk, d, page, before, new, size):
    """f16 outputs have steps of 2^-11, so neither q nor the weights may be rounded as coarsely.  Per
    output, with A = sum p |v|: the output's rounding 2^-11 |o|; the weights held to 2^-21; a
    score's error, D / 16 sums of 16 exact products each off by 2^-22 of the sum of magnitudes and
    four f32 roundings of s, 2^-21 |s|, which enters numerator and sum; ex2 and the f32 sums of P and P V,
    (n / 32 + 64) 2^-23 each."""
    c = Case(cuda_device, torch.float16, hq, hk, d, page, before, new, seed=hq + d)
    c.q = (c.q.float() * size).half()
    got, G = c.attend(), hq // hk
    for r, n in enumerate(c.want["kv_len"]):
        t0, t1 = c.want["cu_new"][r:r + 2]
        at = c.rp.table[r][:-(-n // page)]
        late = torch.arange(n, device=got.device) > (n - (t1 - t0) + torch.arange(t1 - t0, device=got.device))[:, None]
        for h in range(hk):
            k, v = ((x[at, h].double() * s[at, h].double()[:, None, None]).reshape(-1, d)[:n]
                    for x, s in ((c.kv.k, c.kv.k_scale), (c.kv.v, c.kv.v_scale)))
            q = c.q[t0:t1].view(t1 - t0, hk, G, d)[:, h].double()
            s = torch.einsum("wgd,nd->wgn", q, k) * c.scale
            sums = torch.einsum("wgd,nd->wgn", q.abs(), k.abs()) * c.scale
            p = s.masked_fill(late[:, None], -math.inf).softmax(-1)
            o = torch.einsum("wgn,nd->wgd", p, v)
            ds = ((d / 16 * 2.0**-22 * sums + 2.0**-21 * s.abs()) * ~late[:, None]).amax(-1, keepdim=True)
            rel = 2.0**-21 + 2 * ds + 2 * (n / 32 + 64) * 2.0**-23
            tol = 2.0**-11 * o.abs() + rel * torch.einsum("wgn,nd->wgd", p, v.abs()) + 2.0**-25
            err = (got[t0:t1].view(t1 - t0, hk, G, d)[:, h].double() - o).abs()
            assert bool((err <= tol).all()), (r, h, float((err / tol).max()))


# ------------------------------------------------------------------ status words
def test_the_status_of_a_pool_made_in_inference_mode_is_told_and_cleared(cuda_device):
    """A decoder makes its pool in inference mode and is asked for errors outside."""
    with torch.inference_mode():
        pool = tq.PagePool(1, 2, 64, page_size=16, device=cuda_device)
        plan = tq.StepPlan(pool, 40, q_heads=2, kv_heads=1, head_dim=64)
        tq.plan_step(_i32([16, 1], cuda_device), pool, plan)
        plan.err.fill_(tq._native.TQ_ERR_TIMEOUT)
    with pytest.raises(tq._native.TileQuantError, match="too few free pages"):
        pool.check_status()
    pool.check_status()
    with pytest.raises(tq._native.TileQuantError, match="ran out"):
        plan.check_status()
    plan.check_status()
    pool.reset()
    assert int(pool.free_count) == 1 and pool.lengths.tolist() == [0, 0]


def test_the_status_of_a_decode_step_made_in_inference_mode_is_cleared(cuda_device):
    from tests.test_gpu_paged_decode import _model, _prepare, _prompt

    model, vocab = _model("llama", cuda_device)
    for kv_cache in ("16bit", "int8"):
        dec = _prepare(model, _prompt(vocab, 2, 20), 3, cuda_device, eager=True, kv_cache=kv_cache)
        with torch.inference_mode():
            (dec._step.ws if kv_cache == "16bit" else dec._step.pages.plan).err.fill_(tq._native.TQ_ERR_TIMEOUT)
        with pytest.raises(tq._native.TileQuantError, match="ran out"):
            dec.check_step_status()
        dec.check_step_status()
        dec.close()


def test_the_state_of_the_operators_keeps_its_memory(cuda_device):
    pool = tq.PagePool(5, 2, 64, page_size=16, device=cuda_device)
    plan = tq.StepPlan(pool, 40, q_heads=2, kv_heads=1, head_dim=64)
    kv = tq.KVPages(5, 1, 16, 64, device=cuda_device)
    for t in (pool.lengths, pool.block_table, plan.slots, plan.ws_o, kv.k, kv.v_scale):
        shape = t.shape
        with pytest.raises(AttributeError, match="keeps its memory"):
            t.resize_(1 << 20)
        assert t.shape == shape
    pool.lengths += 3
    pool.free_count -= 1
    assert pool.lengths.tolist() == [3, 3] and int(pool.free_count) == 4
    kv.k.data = torch.ones_like(kv.k)  # the kernels go on with the memory of the construction
    other = torch.empty(1 << 20, dtype=torch.int8, device=cuda_device).fill_(-1)
    k, _ = tq.read_pages(kv, _i32([0, 1], cuda_device), torch.float16)
    assert not bool(k.any()) and bool((other == -1).all())


# ------------------------------------------------------------------ the cache's steps
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_channels_far_above_the_rest_set_the_steps_of_all(cuda_device, dtype):
    """Keys with two channels of 64 a hundred times the others: every value is within half a step, the
    page's and head's largest / 127, and the 16-bit rounding of the value read back."""
    dev, hk, d, page, n = cuda_device, 2, 64, 16, 70
    pool = tq.PagePool(6, 1, 96, page_size=page, device=dev)
    plan = tq.StepPlan(pool, n, q_heads=hk, kv_heads=hk, head_dim=d)
    kv = tq.KVPages(6, hk, page, d, device=dev)
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(n, hk, d, generator=g, device=dev)
    x[:, :, [5, 40]] *= 100
    x = x.to(dtype)
    tq.plan_step(_i32([n], dev), pool, plan)
    tq.cache_write(x.flatten(1), x.flatten(1), kv, plan)
    k, v = tq.read_pages(kv, pool.block_table[0, :5].contiguous(), dtype)
    assert torch.equal(k, v)
    got = k.transpose(1, 2).reshape(5 * page, hk, d)[:n].double()
    want = x.double()
    largest = torch.stack([want[i:i + page].abs().amax((0, 2)) for i in range(0, n, page)]).repeat_interleave(page, 0)[:n]
    half = torch.finfo(dtype).eps / 2
    tol = largest[..., None] / 127 * (0.5 + 2.0**-16) + half * got.abs()  # (a quotient's and a scale's f32 rounding)
    assert bool(((got - want).abs() <= tol).all())
    assert float((got - want)[..., :5].abs().max()) > 0.1  # the others' steps are near their own size
    pool.check_status()
