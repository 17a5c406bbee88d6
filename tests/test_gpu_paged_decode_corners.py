"""The graph decoder over the paged 8-bit cache where it can go wrong: errors of a request that are
asked for later."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_decode import _model, _prepare, _prompt
from tilequant_b200 import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eager", [True, False])
def test_an_error_of_a_request_is_told_after_the_next_requests_prompt(cuda_device, eager):
    """Decoding past the prepared length finds the table row full; the prompts that follow, captured or
    not, leave that for the check."""
    model, vocab = _model("llama", cuda_device)
    dec = _prepare(model, _prompt(vocab, 2, 60), 5, cuda_device, eager=eager, kv_cache="int8")
    dec.generate(_prompt(vocab, 2, 60))
    dec.check_step_status()
    for _ in range(17):  # two pages of 64 are full at 128 tokens
        dec.decode(4)
    dec.generate(_prompt(vocab, 2, 60, 7))
    dec.generate(_prompt(vocab, 2, 60, 8))
    with pytest.raises(N.TileQuantError, match="longer than its block table"):
        dec.check_step_status()
    dec.check_step_status()
    dec.generate(_prompt(vocab, 2, 60, 9))
    dec.check_step_status()
    pool = dec._step.pages.pool
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
