"""The graph decoder over the paged 8-bit cache where it can go wrong: errors of a request that are
asked for later, prompts that one plan cannot place."""

from __future__ import annotations

import pytest
import torch

import tilequant_b200 as tq
from tests.test_gpu_paged_decode import _check_prompt, _Heads, _model, _prepare, _prompt, _prompt_cache
from tilequant_b200 import _native as N
from tilequant_b200 import decode_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eager", [True, False])
def test_an_error_of_a_request_is_told_after_the_next_requests_prompt(cuda_device, eager):
    """A step that finds no free page; the prompts that follow, captured or not, leave that for the
    check."""
    model, vocab = _model("llama", cuda_device)
    dec = _prepare(model, _prompt(vocab, 2, 60), 5, cuda_device, eager=eager, kv_cache="int8")
    dec.generate(_prompt(vocab, 2, 60))
    dec.check_step_status()
    pool = dec._step.pages.pool
    dec.prefill(_prompt(vocab, 2, 60, 6))
    with torch.inference_mode():
        pool.lengths.fill_(64)  # (the next token takes a page)
        pool.free_count.zero_()
    dec.decode(1)
    dec.generate(_prompt(vocab, 2, 60, 7))
    dec.generate(_prompt(vocab, 2, 60, 8))
    with pytest.raises(N.TileQuantError, match="too few free pages"):
        dec.check_step_status()
    dec.check_step_status()
    dec.generate(_prompt(vocab, 2, 60, 9))
    dec.check_step_status()
    assert pool.lengths.tolist() == [64, 64]
    pool.forget_requests()  # (outside the inference mode it was made in)
    assert pool.lengths.tolist() == [0, 0] and int(pool.free_count) == pool.num_pages
    dec.close()


def test_two_errors_of_a_request_are_told_together_and_once(cuda_device):
    model, vocab = _model("llama", cuda_device)
    dec = _prepare(model, _prompt(vocab, 2, 20), 3, cuda_device, eager=True, kv_cache="int8")
    pages = dec._step.pages
    with torch.inference_mode():
        pages.pool.status.fill_(N.TQ_PAGES_POOL_EMPTY)
        pages.plan.err.fill_(N.TQ_ERR_TIMEOUT)
    with pytest.raises(N.TileQuantError, match="ran out.*too few free pages"):
        dec.check_step_status()
    dec.generate(_prompt(vocab, 2, 20))
    dec.check_step_status()
    dec.close()


def _pages_of(cache, r, heads, d, prompt):
    """Request r's codes and scales, in the order of its tokens."""
    at = cache.pool.block_table[r, :-(-prompt // 64)].long()
    kv = cache.layers[0]
    n = at.numel() * 64
    keep = torch.arange(n, device=at.device) < prompt
    return [t[at].transpose(0, 1).reshape(heads, n, d)[:, keep] for t in (kv.k, kv.v)] + \
        [t[at] for t in (kv.k_scale, kv.v_scale)]


@pytest.mark.parametrize("batch,prompt,piece", [(1, 200, 64), (3, 333, 128), (2, 64, 64), (2, 65, 64)])
def test_a_prompt_placed_in_pieces_is_the_prompt_placed_at_once(cuda_device, monkeypatch, batch, prompt, piece):
    want = decode_step.PagedDecodeCache([_Heads], batch, prompt, prompt + 9, cuda_device)
    monkeypatch.setattr(decode_step, "_prompt_requests", lambda *a: 1)
    monkeypatch.setattr(decode_step, "_prompt_piece", lambda *a: piece)
    got = decode_step.PagedDecodeCache([_Heads], batch, prompt, prompt + 9, cuda_device)
    assert got.prompt_plan.max_tokens == piece
    cache = _prompt_cache(cuda_device, batch, prompt, _Heads)
    for c in (want, got):
        for _ in range(2):
            c.load_prompt(cache)
        assert c.pool.lengths.tolist() == [prompt] * batch
        c.next_step()
        c.check_status()
    for r in range(batch):
        for a, b in zip(_pages_of(want, r, 4, 128, prompt), _pages_of(got, r, 4, 128, prompt)):
            assert torch.equal(a, b)


def test_one_prompt_longer_than_a_plan_counts_is_placed(cuda_device):
    """400000 tokens with 32 KV heads: 2.5e9 chunks of attention that a prompt does not run."""

    class Heads:
        Hq, Hkv, D = 32, 32, 64

    prompt = 400000
    pages = decode_step.PagedDecodeCache([Heads], 1, prompt, prompt + 64, cuda_device)
    assert pages.prompt_plan.max_tokens < prompt
    cache = _prompt_cache(cuda_device, 1, prompt, Heads)
    pages.load_prompt(cache)
    pages.next_step()
    pages.check_status()
    assert pages.plan.kv_len.tolist() == [prompt + 1]
    border = pages.prompt_plan.max_tokens // 64
    for first in (0, border - 2, prompt // 64 - 3):
        _check_prompt(pages, cache, 0, first)


@pytest.mark.parametrize("kw", [dict(), dict(kv_cache="int8"), dict(fused_decode=False),
                                dict(fused_decode=False, sampling=tq.Sampling(seed=1))])
@pytest.mark.parametrize("eager", [True, False])
def test_steps_beyond_the_cache_are_refused(cuda_device, kw, eager):
    """Calls of decode after one prefill add up; the step after the last would write behind the cache."""
    model, vocab = _model("llama", cuda_device)
    prompt = _prompt(vocab, 2, 12)
    dec = _prepare(model, prompt, 6, cuda_device, eager=eager, **kw)
    with pytest.raises(ValueError, match="0 of 5 are left"):
        dec.decode(1)
    runs = []
    for calls in ([5], [2, 3], [1, 1, 1, 1, 1], [4, None]):
        if "sampling" in kw:
            dec._generator.manual_seed(3)
        dec.prefill(prompt)
        for n in calls:
            dec.decode(n)
        for n in (1, 5):
            with pytest.raises(ValueError, match="0 of 5 are left"):
                dec.decode(n)
        dec.decode(0)
        assert int(dec._position) == 12 + 5
        runs.append(dec._generated.tolist())
    assert all(r == runs[0] for r in runs)
    dec.check_step_status()
    dec.close()
