"""Sampling on the GPU against the definition in 64 bits (``paged_reference.sample_row``): the
same token for the same random number, over sizes, filters, ties and masks."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tilequant_b200 as tq
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _logits(dev, rows, vocab, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=dev) * 2 - 1
    x[:, ::97] += 4
    return x.to(dtype), torch.rand(rows, generator=g, device=dev)


def _vec(dev, rows, value, dtype=torch.float32):
    return None if value is None else torch.full((rows,), value, dtype=dtype, device=dev)


def _check(logits, u, T=None, k=None, p=None, m=None):
    dev, rows = logits.device, logits.shape[0]
    as_vec = lambda v, t=torch.float32: v if v is None or torch.is_tensor(v) else _vec(dev, rows, v, t)  # noqa: E731
    T, k, p, m = as_vec(T), as_vec(k, torch.int32), as_vec(p), as_vec(m)
    ids, lp = tq.sample_tokens(logits, u, temperature=T, top_k=k, top_p=p, min_p=m)
    x = logits.double().cpu().numpy()
    for r in range(rows):
        at = lambda v, d: d if v is None else float(v[r].double())  # noqa: E731
        want, wlp = ref.sample_row(x[r], float(u[r].double()), at(T, 1.0), int(at(k, 0)), at(p, 1.0), at(m, 0.0))
        assert int(ids[r]) == want, (r, int(ids[r]), want, x[r][int(ids[r])], x[r][want])
        # the log of a quotient of f64 sums, rounded to f32 once; 1e-12 for the sums
        if math.isinf(wlp):
            assert float(lp[r]) == wlp
        else:
            assert abs(float(lp[r]) - wlp) <= 2.0**-24 * abs(wlp) + 1e-12, (r, float(lp[r]), wlp)
    return ids


FILTERS = [dict(), dict(T=0.7), dict(T=1.5, k=50), dict(p=0.9), dict(m=0.05), dict(T=0.8, k=40, p=0.95, m=0.02),
           dict(k=1), dict(T=0.0, p=0.5), dict(p=0.0), dict(p=1e-9, k=7), dict(m=1.0), dict(m=2.0), dict(k=10**9, p=1.0),
           dict(T=math.inf, k=9), dict(T=1e-3), dict(T=30.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 1000), (17, 32003), (3, 128256)])
@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_the_token_of_the_definition(cuda_device, dtype, rows, vocab, f):
    logits, u = _logits(cuda_device, rows, vocab, dtype, rows + vocab + f)
    _check(logits, u, **FILTERS[f])


@pytest.mark.parametrize("vocab", [65528, 65529, 65536, 131071, 152064, 524224, 1 << 20])
def test_large_vocabularies_and_rows_of_one_value(cuda_device, vocab):
    """A slice's counter must hold a whole slice of equal logits."""
    x = torch.zeros(3, vocab, device=cuda_device).bfloat16()
    x[1] = torch.finfo(torch.bfloat16).min
    x[2, 5:] = -2.0
    u = torch.tensor([0.99999, 0.5, 0.75], device=cuda_device)
    _check(x, u)
    _check(x, u, k=vocab - 1, p=0.999)
    _check(x, u, p=0.5)


@pytest.mark.parametrize("rows,vocab", [(160, 70001), (150, 152064), (150, 32760), (150, 65529)])
def test_many_rows_of_few_values(cuda_device, rows, vocab):
    """Many rows have one CTA each, whose counters give counts away between rounds: rows of one
    value, of two, of a value and its negative, of a mask of the lowest value, and ordinary ones."""
    x, u = _logits(cuda_device, rows, vocab, torch.bfloat16, vocab)
    x[0] = 1.5
    x[1] = -1.5
    x[2, ::2], x[2, 1::2] = 2.0, -2.0
    x[3, ::3], x[3, 1::3], x[3, 2::3] = 0.25, -0.25, 0.5
    x[4, 100:] = torch.finfo(torch.bfloat16).min
    x[5] = torch.finfo(torch.bfloat16).min
    x[6, 9:] = 0.0
    x[6, 10::2] = -0.0
    x[7] = torch.finfo(torch.bfloat16).max
    x[8, ::2] = -math.inf
    x[9, ::2] = math.nan
    x[9, 1::2] = 3.0
    keep = list(range(12)) + [rows - 1]
    for f in (dict(T=0.8), dict(k=40000, p=0.7), dict(m=0.3)):
        as_vec = {n: _vec(cuda_device, rows, f[s], t) for n, s, t in (("temperature", "T", torch.float32), ("top_p", "p", torch.float32),
                                                                   ("min_p", "m", torch.float32), ("top_k", "k", torch.int32)) if s in f}
        ids, _ = tq.sample_tokens(x, u, **as_vec)
        want = _check(x[keep], u[keep], **f)  # few rows: other cluster sizes
        assert torch.equal(ids[keep], want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_counts_that_pass_half_of_a_counter(cuda_device, dtype):
    """One CTA counts a row of 152064 in five rounds of 32704: values whose counts pass half of a
    16-bit counter in the first round's end, in a middle one or in the last only, both signs of one
    magnitude, and counts around the 2048 from which a value gives counts away."""
    rows, vocab, turn = 150, 152064, 32704
    x, u = _logits(cuda_device, rows, vocab, dtype, 77)
    x[0, :2 * turn] = 1.5
    x[1, turn:3 * turn], x[1, 3 * turn:] = 0.5, -0.5
    x[2, 4 * turn - 32000:] = -1.25  # past half in the last round
    x[3, :33000], x[3, 33000:66000], x[3, 66000:99000] = 2.0, -2.0, 2.0
    x[4, :40000] = 3.0  # passes; then counts around the border when it does
    for i, n in enumerate((2046, 2047, 2048, 2049)):
        x[4, 40000 + 2100 * i:40000 + 2100 * i + n] = 4.0 + i
        x[4, 50000 + 2100 * i:50000 + 2100 * i + n] = -4.0 - i
    x[5] = -0.0
    x[5, ::2] = 0.0
    x[6, ::5], x[6, 1::5], x[6, 2::5] = torch.finfo(dtype).max, -math.inf, torch.finfo(dtype).min
    x[7] = torch.finfo(dtype).max
    x[7, -9:] = torch.finfo(dtype).min
    keep = list(range(9)) + [rows - 1]
    for f in (dict(T=2.0), dict(T=1.3, k=70000), dict(T=5.0, p=0.8), dict(k=vocab - 1, m=0.01)):
        as_vec = {n: _vec(cuda_device, rows, f[s], t) for n, s, t in (("temperature", "T", torch.float32), ("top_p", "p", torch.float32),
                                                                   ("min_p", "m", torch.float32), ("top_k", "k", torch.int32)) if s in f}
        for v in (u, torch.zeros_like(u), torch.full_like(u, 0.999999)):
            ids, _ = tq.sample_tokens(x, v, **as_vec)
            assert torch.equal(ids[keep], _check(x[keep], v[keep], **f))


@pytest.mark.parametrize("rows", [2, 64, 150, 300])
def test_row_counts_around_a_wave(cuda_device, rows):
    logits, u = _logits(cuda_device, rows, 5003, torch.bfloat16, rows)
    _check(logits, u, T=0.9, k=100, p=0.9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_by_index(cuda_device, dtype):
    x = torch.full((8, 4099), -3.0, device=cuda_device)
    x[:, 1000:3000:7] = 1.5
    x[:, 1003] = 1.75
    x[:, 17], x[:, 19] = 0.0, -0.0  # equal
    u = torch.linspace(0, 0.9999, 8, device=cuda_device)
    for f in (dict(), dict(k=100), dict(k=2), dict(p=0.3), dict(m=0.9), dict(k=290, p=0.999), dict(T=0.1, k=288)):
        _check(x.to(dtype), u, **f)
    z = torch.full((4, 50), -9.0, device=cuda_device)
    z[:, 30], z[:, 10], z[:, 20] = 0.0, -0.0, 0.0
    assert _check(z.to(dtype), torch.zeros(4, device=cuda_device), T=0.0).tolist() == [10] * 4
    ids = _check(z.to(dtype), torch.tensor([0.0, 0.4, 0.7, 0.999], device=cuda_device), k=3)
    assert ids.tolist() == [10, 20, 30, 30]


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(cuda_device, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.randn(9, 20011, generator=g, device=cuda_device).to(dtype)
    u = torch.rand(9, generator=g, device=cuda_device)
    x[0] = -math.inf  # nothing left
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 777] = -5.0  # one token left
    x[3, 5:] = -math.inf
    x[4, 5:] = torch.finfo(dtype).min
    x[5] = torch.finfo(dtype).min  # a mask of the lowest value over everything: uniform
    x[6, 100] = math.inf
    x[7, [3, 900, 20010]] = math.inf
    x[8, ::2] = math.nan
    for f in (dict(), dict(k=3), dict(p=0.7), dict(m=0.1), dict(T=0.0), dict(T=2.0, k=500, p=0.9, m=0.001)):
        ids = _check(x, u, **f)
        assert ids[0] == 0 and ids[1] == 0 and ids[2] == 777


def test_numbers_at_the_ends(cuda_device):
    logits, _ = _logits(cuda_device, 6, 3001, torch.bfloat16, 1)
    logits[1:] = logits[0]
    below_one = 1 - 2.0**-24
    u = torch.tensor([0.0, below_one, 1.0, -1.0, 7.0, math.nan], device=cuda_device)
    ids, _ = tq.sample_tokens(logits, u)
    want = [ref.sample_row(logits[0].double().cpu().numpy(), v)[0] for v in (0.0, below_one, 1.0, 0.0, 1.0, 0.0)]
    assert ids.tolist() == want


def test_every_number_of_a_fine_sweep(cuda_device):
    """Random numbers on and beside the borders of five tokens of equal weight, and a sweep:
    the inverse of the running sum."""
    x = torch.full((1, 40), -math.inf, device=cuda_device)
    x[0, [3, 8, 9, 21, 39]] = 2.5
    u = torch.cat([torch.arange(1024) / 1024, torch.tensor([0.2, 0.4, 0.6, 0.8]),
                   torch.nextafter(torch.tensor([0.2, 0.4, 0.6, 0.8]), torch.tensor(0.0))]).to(cuda_device)
    ids, lp = tq.sample_tokens(x.expand(len(u), 40).contiguous().half(), u)
    order = np.array([3, 8, 9, 21, 39])
    want = order[np.floor(u.double().cpu().numpy() * 5.0).astype(int)]
    assert ids.cpu().numpy().tolist() == want.tolist()
    assert bool((lp == float(np.float32(math.log(0.2)))).all())


def test_strided_and_unaligned_rows(cuda_device):
    wide, u = _logits(cuda_device, 4, 10007, torch.float16, 9)
    for lo, hi in ((0, 10007), (1, 10000), (3, 12), (7, 9007), (5, 6)):
        view = wide[:, lo:hi]
        ids = _check(view, u, T=0.9)
        assert torch.equal(ids, tq.sample_tokens(view.contiguous(), u, temperature=_vec(cuda_device, 4, 0.9))[0])


def test_rows_take_their_own_parameters(cuda_device):
    rows = 11
    logits, u = _logits(cuda_device, rows, 9001, torch.bfloat16, 3)
    g = torch.Generator(device=cuda_device).manual_seed(8)
    T = torch.rand(rows, generator=g, device=cuda_device) * 2
    T[3], T[4], T[5] = 0.0, -1.0, math.nan
    k = torch.randint(-2, 300, (rows,), generator=g, device=cuda_device, dtype=torch.int32)
    p = torch.rand(rows, generator=g, device=cuda_device) * 1.3
    m = torch.rand(rows, generator=g, device=cuda_device) * 0.2 - 0.05
    _check(logits, u, T=T, k=k, p=p, m=m)


def test_all_16_bit_patterns_in_one_row(cuda_device):
    bits = torch.arange(65536, device=cuda_device).to(torch.int32).to(torch.int16)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    for dtype in DTYPES:
        x = bits.view(dtype)[torch.randperm(65536, generator=g, device=cuda_device)][None]
        _check(x.contiguous(), torch.tensor([0.3], device=cuda_device), T=1e30)
        y = x.clone()
        y[torch.isinf(y)] = 0.0
        for T, p in ((1.0, None), (1e4, None), (1e4, 0.9), (3e38, None), (3e38, 0.99)):
            _check(y.contiguous(), torch.tensor([0.77], device=cuda_device), T=T, p=p)


def test_no_rows(cuda_device):
    ids, lp = tq.sample_tokens(torch.zeros(0, 5, device=cuda_device).half(), torch.zeros(0, device=cuda_device))
    assert ids.shape == (0,) and lp.shape == (0,)


@pytest.mark.parametrize("captured", [False, True])
def test_sampled_pick_and_bookkeeping(cuda_device, captured):
    dev, B, V, prompt, steps = cuda_device, 3, 501, 10, 6
    g = torch.Generator(device=dev).manual_seed(2)
    logits = torch.zeros(B, V, device=dev, dtype=torch.bfloat16)
    uniform = torch.rand(B, steps + 1, generator=g, device=dev)
    keys = torch.zeros(B, dtype=torch.int64, device=dev)
    position = torch.full((1,), prompt, dtype=torch.int64, device=dev)
    nxt, token = (torch.full((B, 1), -1, dtype=torch.int64, device=dev) for _ in range(2))
    generated = torch.full((B, steps + 1), -1, dtype=torch.int64, device=dev)
    T, k = _vec(dev, B, 0.8), _vec(dev, B, 30, torch.int32)
    run = lambda: tq.sample_pick(logits, uniform, keys, position, prompt, temperature=T, top_k=k, next_ids=nxt,  # noqa: E731
                                 token=token, generated=generated)
    if captured:
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        position.fill_(prompt)
        generated.fill_(-1)
    for i in range(steps):
        logits.copy_(torch.randn(B, V, generator=g, device=dev) * 2)
        graph.replay() if captured else run()
        x = logits.double().cpu().numpy()
        want = [ref.sample_row(x[b], float(uniform[b, i + 1].double()), float(T[0].double()), 30)[0] for b in range(B)]
        assert generated[:, i + 1].tolist() == want and token.flatten().tolist() == want
        assert nxt.flatten().tolist() == want and int(position) == prompt + i + 1 and not bool(keys.any())
    assert generated[:, 0].tolist() == [-1] * B
    run()  # beyond the last column: the last number again, nothing stored
    assert generated[:, 0].tolist() == [-1] * B and int(position) == prompt + steps + 1


def test_a_temperature_of_zero_is_the_greedy_pick(cuda_device):
    from tilequant_b200.decode_step import greedy_pick

    logits, u = _logits(cuda_device, 7, 4001, torch.bfloat16, 6)
    logits[2, 50] = logits[2, 3999] = 60.0
    keys = torch.zeros(7, dtype=torch.int64, device=cuda_device)
    pos = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    nxt = torch.zeros(7, dtype=torch.int64, device=cuda_device)
    greedy_pick(logits, keys, pos, 0, next_ids=nxt)
    ids, lp = tq.sample_tokens(logits, u, temperature=_vec(cuda_device, 7, 0.0))
    assert torch.equal(ids, nxt) and not bool(lp.any())


def test_calls_that_are_refused(cuda_device):
    x, u = _logits(cuda_device, 3, 50, torch.float16, 1)
    two = u[:, None].repeat(1, 4)
    keys, pos = torch.zeros(3, dtype=torch.int64, device=cuda_device), torch.zeros(1, dtype=torch.int64, device=cuda_device)
    bad = [
        (lambda: tq.sample_tokens(x.float(), u), "float32"),
        (lambda: tq.sample_tokens(x[0], u), "rows, vocab"),
        (lambda: tq.sample_tokens(x[:, ::2], u), "unit column stride"),
        (lambda: tq.sample_tokens(x[:1].expand(3, -1), u), "overlap"),
        (lambda: tq.sample_tokens(x, u[:2]), "uniform"),
        (lambda: tq.sample_tokens(x, u.double()), "uniform"),
        (lambda: tq.sample_tokens(x, two), "uniform"),
        (lambda: tq.sample_tokens(x, u.cpu()), "no CPU path"),
        (lambda: tq.sample_tokens(x, u, top_k=u), "top_k"),
        (lambda: tq.sample_tokens(x, u, temperature=u[:1]), "temperature"),
        (lambda: tq.sample_tokens(x, u, top_p=u.cpu()), "cuda"),
        (lambda: tq.sample_tokens(x, u, out=keys.int()), "out"),
        (lambda: tq.sample_tokens(torch.zeros(1, (1 << 20) + 1, device=cuda_device).half(), u[:1]), "at most"),
        (lambda: tq.sample_pick(x, u, keys, pos, 0), "uniform"),
        (lambda: tq.sample_pick(x, two, keys[:2], pos, 0), "keys"),
        (lambda: tq.sample_pick(x, two, keys, pos.int(), 0), "position"),
        (lambda: tq.sample_pick(x, two, keys, pos, 0, token=keys[:2]), "token"),
        (lambda: tq.sample_pick(x, two, keys, pos, 0, generated=keys), "generated"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()


def test_the_first_call_of_a_process_may_be_captured(cuda_device):
    """Launch settings are asked of the device on first use, also while a stream is captured."""
    import subprocess
    import sys

    code = ("import torch, tilequant_b200 as tq\n"
            "x = torch.randn(20, 5000, device='cuda').half(); u = torch.rand(20, device='cuda')\n"
            "ids, lp = torch.empty(20, dtype=torch.int64, device='cuda'), torch.empty(20, device='cuda')\n"
            "torch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    tq.sample_tokens(x, u, out=ids, logprobs=lp)\n"
            "g.replay()\n"
            "assert torch.equal(ids, tq.sample_tokens(x, u)[0])\n"
            "pool = tq.PagePool(9, 2, 64, page_size=16); plan = tq.StepPlan(pool, 4, q_heads=4, kv_heads=2, head_dim=64)\n"
            "kv = tq.KVPages(9, 2, 16, 64); n = torch.ones(2, dtype=torch.int32, device='cuda')\n"
            "k = torch.randn(2, 128, device='cuda').half(); q = torch.randn(2, 256, device='cuda').half()\n"
            "out = torch.empty_like(q)\n"
            "torch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    tq.plan_step(n, pool, plan); tq.cache_write(k, k, kv, plan); tq.attn_paged(q, kv, plan, 0.1, out=out)\n"
            "g.replay(); g.replay()\n"
            "torch.cuda.synchronize()\n"
            "assert pool.lengths.tolist() == [2, 2] and bool(torch.isfinite(out).all())\n"
            "print('captured')\n")
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "captured" in res.stdout, res.stderr[-2000:]
