"""Sampling on the GPU where its counting and its sums can go wrong: masses of NaN logits, random
numbers that fall between two roundings of one sum."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tilequant_b200 as tq
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _vec(dev, rows, value, dtype=torch.float32):
    return torch.full((rows,), value, dtype=dtype, device=dev)


@pytest.mark.parametrize("dtype,first_nan", [(torch.bfloat16, 0x7F81), (torch.float16, 0x7C01)])
def test_thousands_of_equal_nan_logits_are_never_sampled(cuda_device, dtype, first_nan):
    """150 rows of 152064 have one block each, which looks its counters through between rounds once a
    count passed half of their range.  The NaNs beside +inf share its block of 64 values."""
    rows, vocab = 150, 152064
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.randn(rows, vocab, generator=g, device=cuda_device).to(dtype)
    bits = x.view(torch.int16)
    infinite = {0: [140000], 1: [140000], 2: [7, 100001, 152063], 3: [], 4: []}
    for r, at in infinite.items():
        n = (5000, 2100, 66000, 5000, 70000)[r]
        nan = (first_nan, first_nan + 3, first_nan, first_nan + 0x3E, first_nan + 0x20)[r]
        bits[r, 10:10 + n] = torch.tensor(nan, dtype=torch.int32).to(torch.int16)
        x[r, 70100:140000] = -1.0  # passes half of a counter's range
        x[r, at] = math.inf
    bits[4, 70100:100000] = torch.tensor(first_nan | 0x8000, dtype=torch.int32).to(torch.int16)
    u = torch.rand(rows, generator=g, device=cuda_device)
    keep = [0, 1, 2, 3, 4, rows - 1]
    values = x[keep].double().cpu().numpy()
    for k, p, m in ((50, 1.0, 0.0), (2, 0.9, 0.0), (0, 0.95, 0.01), (4000, 1.0, 0.0)):
        ids, logprobs = tq.sample_tokens(x, u, top_k=_vec(cuda_device, rows, k, torch.int32),
                                         top_p=_vec(cuda_device, rows, p), min_p=_vec(cuda_device, rows, m))
        for r, v in zip(keep, values):
            want, logprob = ref.sample_row(v, float(u[r].double()), 1.0, k, float(np.float32(p)), float(np.float32(m)))
            assert int(ids[r]) == want and not math.isnan(float(logprobs[r]))
            assert abs(float(logprobs[r]) - logprob) <= 2.0**-24 * abs(logprob) + 1e-12  # rounded to f32 once


def _nearly_equal_weights(dev, rows, seed):
    """Rows of 20 to 600 different logits whose weights, at the row's temperature, differ from one by at
    most 2^-48: sums of them in different orders differ by their last bits, and half of the kept sum
    lies on the border between two tokens.  Returns logits, temperatures and each row's token count."""
    g = torch.Generator(device=dev).manual_seed(seed)
    values = torch.cat([torch.arange(128, 256), torch.arange(64, 128, 0.5), torch.arange(32, 64, 0.25),
                        torch.arange(16, 32, 0.125), torch.arange(8, 16, 0.0625)]).to(dev)
    there = torch.rand(rows, len(values), generator=g, device=dev) < torch.rand(rows, 1, generator=g, device=dev) * 0.8 + 0.1
    order = torch.randperm(len(values), generator=g, device=dev)
    x = torch.where(there, values[order], -math.inf).bfloat16()
    T = 2.0**58 * torch.exp2(3 * torch.rand(rows, generator=g, device=dev))
    return x, T, there.sum(1)


@pytest.mark.parametrize("what", ["uniform", "top_p"])
def test_a_border_between_two_roundings_of_a_sum_is_off_by_one_token_at_most(cuda_device, what):
    """Half of the kept sum falls at half of the tokens.  Sums of at most 640 weights of at most one in
    64 bits are off by less than 640 * 640 * 2^-53, far less than one weight, so the token is the
    definition's or its neighbour."""
    rows = 16384
    x, T, n = _nearly_equal_weights(cuda_device, rows, 11)
    if what == "uniform":
        ids, _ = tq.sample_tokens(x, _vec(cuda_device, rows, 0.5), temperature=T)
    else:  # the last of the kept half
        ids, _ = tq.sample_tokens(x, _vec(cuda_device, rows, 1 - 2.0**-24), temperature=T,
                                  top_p=_vec(cuda_device, rows, 0.5))
    rank = (x > x.gather(1, ids[:, None])).sum(1)
    off = (rank - (n - 1) / 2).abs()
    assert bool((off <= 1.5).all()), (int((off > 1.5).sum()), float(off.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [7, 3001, 70001])
@pytest.mark.parametrize("T", [math.inf, 3e38, 1e30, 1e20, 1e13, 1e8])
def test_min_p_of_weights_that_are_one_or_almost(cuda_device, dtype, vocab, T):
    """At high temperatures many logits, or all, weigh one in 64 bits and min_p = 1 keeps them all.  (At
    1e13 the next logit is 2^-10 away at least, so no weight is near the tie at 1 - 2^-54.)"""
    rows = 6
    g = torch.Generator(device=cuda_device).manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g, device=cuda_device) * 40).to(dtype)
    x[1] = x[1].abs() + 1
    x[2] = -x[2].abs() - 1
    x[3, ::2] = -math.inf
    x[4, 5] = math.inf
    u = torch.rand(rows, generator=g, device=cuda_device)
    t = float(np.float32(T))
    for m in (1.0, 1 - 2.0**-24, 0.5, 1.5, math.inf):
        ids, _ = tq.sample_tokens(x, u, temperature=_vec(cuda_device, rows, T), min_p=_vec(cuda_device, rows, m))
        want = [ref.sample_row(v, float(u[r].double()), t, 0, 1.0, m)[0] for r, v in enumerate(x.double().cpu().numpy())]
        assert ids.tolist() == want, (m, ids.tolist(), want)


def test_a_single_column_may_have_any_stride(cuda_device):
    rows = 3
    g = torch.Generator(device=cuda_device).manual_seed(1)
    wide = torch.randn(rows, 400, generator=g, device=cuda_device).half()
    u = torch.rand(5, rows, generator=g, device=cuda_device)
    ids, logprobs = tq.sample_tokens(wide[:, ::2][:, :1], u[0])
    assert ids.tolist() == [0] * rows and logprobs.tolist() == [0.0] * rows
    keys = torch.zeros(rows, dtype=torch.int64, device=cuda_device)
    for step in range(2):
        position = torch.full((1,), 9, dtype=torch.int64, device=cuda_device)
        generated = torch.full((5, rows), -1, dtype=torch.int64, device=cuda_device)
        tq.sample_pick(wide, u.t()[:, step:step + 1], keys, position, 10, generated=generated.t()[:, 2:3])
        assert generated[2].tolist() == tq.sample_tokens(wide, u[step].contiguous())[0].tolist()
        assert int((generated != -1).sum()) == rows and int(position) == 10
