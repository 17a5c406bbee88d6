"""Host-side checks of the serving operators' corners (no GPU)."""

from __future__ import annotations

import copy
import ctypes
import pickle
from types import SimpleNamespace

import pytest
import torch

from tilequant_b200 import _native as N

A = 4096  # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from tilequant_b200 import build

        build.build()
    return N.load()


def _args(cls, **kw):
    return cls(**{**{name: A for name, t in cls._fields_ if t is ctypes.c_void_p}, **kw})


def test_unknown_flags_are_refused(lib):
    write = _args(N.CacheWriteArgs, ld_k=128, ld_v=128, ld_q=512, ld_qo=512, ld_cs=64, rows=0, requests=4, pages=40,
                  page=16, kv_heads=2, q_heads=8, head_dim=64)
    attn = _args(N.PagedAttnArgs, ld_q=512, ld_out=512, rows=0, requests=4, table_width=10, pages=40, page=16, kv_heads=2,
                 q_heads=8, head_dim=64, row_tile=8, attn_ctas=296, scale_log2=0.1)
    for call, a in ((lib.tq_cache_write, write), (lib.tq_attn_paged, attn)):
        for flags, rc in ((0, N.TQ_OK), (N.TQ_CLEAR_REST, N.TQ_OK), (2, N.TQ_ERR_INVALID), (-1, N.TQ_ERR_INVALID)):
            a.flags = flags
            assert call(ctypes.byref(a), 0, None) == rc
            assert rc == N.TQ_OK or b"flags" in lib.tq_last_error()


class _Words:
    """Stands in for a fused step over the INT8 cache with an attention error and a pool error."""

    def __init__(self, err, status):
        self.err, self.told = err, status
        self.pages = SimpleNamespace(pool=SimpleNamespace(check_status=self._pool))

    def status(self):
        return self.err

    def reset_status(self):
        self.err = N.TQ_OK

    def _pool(self):
        if self.told:
            self.told = 0
            raise N.TileQuantError("page pool: too few free pages")


@pytest.mark.parametrize("err", [N.TQ_OK, N.TQ_ERR_TIMEOUT])
@pytest.mark.parametrize("status", [0, N.TQ_PAGES_POOL_EMPTY])
def test_a_step_check_tells_and_clears_every_error_word(err, status):
    from tilequant_b200.graph_decode import CudaGraphGreedyDecoder

    dec = CudaGraphGreedyDecoder.__new__(CudaGraphGreedyDecoder)
    dec._step = _Words(err, status)
    if err or status:
        with pytest.raises(N.TileQuantError) as e:
            dec.check_step_status()
        assert ("ran out" in str(e.value)) == bool(err) and ("too few" in str(e.value)) == bool(status)
    dec.check_step_status()


def test_a_benchmark_request_that_went_wrong_is_an_error(monkeypatch):
    from tilequant_b200 import benchmark_generation as B

    monkeypatch.setattr(B.torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(B.torch.cuda, "reset_peak_memory_stats", lambda device=None: None)
    calls = []

    class Decoder:
        wrong = None

        def __getattr__(self, name):
            def call(*args):
                calls.append(name)
                if name == self.wrong:
                    raise N.TileQuantError(name)
            return call

    dec = Decoder()
    start, first, end, e0, e1 = B.graph_request(dec, [1, 2], 3, 5, None, None)
    assert start <= first <= end and e0 is None and e1 is None
    assert calls == ["prefill", "decode", "check_peer_status", "check_step_status"]
    for dec.wrong in ("check_peer_status", "check_step_status"):
        with pytest.raises(N.TileQuantError, match=dec.wrong):
            B.graph_request(dec, [1, 2], 3, 5, None, None)


@pytest.mark.parametrize("argv,text", [
    (["--method", "bf16", "--kv_cache", "int8"], "--kv_cache"),
    (["--method", "bf16", "--temperature", "0.8"], "--temperature"),
    (["--method", "bf16", "--temperature", "0", "--top_k", "5"], "--temperature, --top_k"),
    (["--method", "bf16", "--seed", "3"], "--seed"),
    (["--top_k", "5"], "--top_k without --temperature"),
    (["--kv_cache", "int8", "--top_p", "0.9", "--min_p", "0.1"], "--top_p, --min_p without"),
    (["--seed", "1"], "--seed without"),
    (["--temperature", "-1"], "temperature must be"),
    (["--temperature", "1", "--top_p", "1.5"], "top_p and min_p"),
])
def test_benchmark_options_that_would_not_be_followed_are_refused(monkeypatch, capsys, argv, text):
    from tilequant_b200 import benchmark_generation as B

    monkeypatch.setattr(B, "run", lambda args: pytest.fail("the run began"))
    with pytest.raises(SystemExit):
        B.main(["--model_dir", "m", *argv])
    assert text in capsys.readouterr().err


@pytest.mark.parametrize("argv", [[], ["--method", "bf16"], ["--temperature", "0"], ["--kv_cache", "int8"],
                                  ["--kv_cache", "int8", "--temperature", "0.8", "--top_k", "20", "--seed", "4"]])
def test_benchmark_options_that_go_together_reach_the_run(monkeypatch, argv):
    from tilequant_b200 import benchmark_generation as B

    monkeypatch.setattr(B, "run", vars)
    assert B.main(["--model_dir", "m", *argv])["model_dir"] == "m"


@pytest.mark.parametrize("batch", [1, 8, 64])
@pytest.mark.parametrize("prompt", [1, 77, 8192, 131072, 400000, 500000, 3000000])
@pytest.mark.parametrize("kv_heads", [1, 4, 8, 32])
def test_every_prompt_is_placed_in_plans_that_count_their_work(batch, prompt, kv_heads):
    from tilequant_b200.decode_step import _prompt_piece, _prompt_requests

    room = (prompt + 64 + 63) // 64 * 64
    n = _prompt_requests(batch, prompt, kv_heads, room)
    piece = _prompt_piece(batch, prompt, kv_heads, room, 64) if n == 1 else prompt
    work = lambda tokens: (tokens / 16 + batch) * kv_heads * (room / 128 + 4)  # noqa: E731  (as tq_plan_step bounds it)
    assert work(n * piece) < 2**31
    assert piece == prompt or (piece % 64 == 0 and work(1.1 * piece + 64) > 0.95 * 2**31)  # no more plans than needed


def _holder():
    class Holder(N.FixedTensors):
        def __init__(self):
            self.a, self.n = torch.zeros(4), 1

    return Holder()


def test_fixed_tensors_take_in_place_operators():
    h = _holder()
    h.a += 2
    h.a *= 3
    h.a[1:] -= 1
    assert h.a.tolist() == [6, 5, 5, 5]
    with pytest.raises(AttributeError, match="copy into it"):
        h.a = h.a.clone()
    with pytest.raises(AttributeError, match="copy into it"):
        h.a = None
    h.n += 1
    assert h.n == 2


def test_the_memory_of_fixed_tensors_stays():
    """Addresses that were taken once stay valid whatever is done to the tensors."""
    h = _holder()
    at = h.a.data_ptr()
    for change in (lambda: h.a.resize_(1000), lambda: h.a.resize_as_(torch.zeros(9)), lambda: h.a.set_(torch.zeros(4))):
        with pytest.raises(AttributeError, match="Holder.a keeps its memory"):
            change()
    assert h.a.shape == (4,) and h.a.data_ptr() == at
    h.a.fill_(7)
    h.a.data = torch.zeros(4)
    assert ctypes.cast(at, ctypes.POINTER(ctypes.c_float))[3] == 7.0
    assert h._memory[0].data_ptr() == at


@pytest.mark.parametrize("kw,text", [
    # a request's keys, rounded up to a chunk of 128, would pass 2^31
    (dict(table_width=2**27 - 1, page=16, pages=1, max_tokens=1, kv_heads=1, group=1, row_tile=16), b"2^31"),
    # fewer than 2^31 chunks, but 2^32 query rows
    (dict(table_width=4, page=16, pages=40, max_tokens=2**30, kv_heads=1, group=4, row_tile=16), b"query rows"),
    (dict(table_width=4, page=16, pages=40, max_tokens=2**29 - 3, kv_heads=1, group=4, row_tile=16), b"query rows"),
])
def test_plan_step_refuses_what_passes_32_bits(lib, kw, text):
    a = _args(N.PlanArgs, requests=4, attn_ctas=296, **kw)
    assert lib.tq_plan_step(ctypes.byref(a), None) == N.TQ_ERR_INVALID and text in lib.tq_last_error()


def test_a_pool_of_too_long_requests_is_refused():
    import tilequant_b200 as tq

    with pytest.raises(ValueError, match="2\\^31"):
        tq.PagePool(4, 1, 2**31 - 20, page_size=16)
    with pytest.raises(ValueError, match="2\\^31"):
        tq.PagePool(4, 1, 2**31 - 200, page_size=128)


def test_decode_calls_after_one_prefill_add_up_to_the_prepared_bound():
    from tilequant_b200.graph_decode import CudaGraphGreedyDecoder

    dec = CudaGraphGreedyDecoder.__new__(CudaGraphGreedyDecoder)
    dec._prepared, dec._prefill_only, dec.max_new_tokens, dec._steps_left = True, False, 5, 0
    dec._decode_graph = dec._prefill_graph = dec._sampling = dec._decode_logits = None
    dec._prefill_logits, dec._token, dec._prompt = torch.zeros(1), torch.zeros(1), torch.zeros(1, 2, dtype=torch.long)
    dec.batch_size, dec.prompt_tokens, dec._generated, steps = 1, 2, torch.zeros(1, 5), []
    dec._decode_body, dec._prefill_body = lambda: steps.append(1), steps.clear
    with pytest.raises(ValueError, match="0 of 4 are left"):
        dec.decode(1)
    for calls, done in (([4], 4), ([1, 2], 3), ([3, None], 4), ([None], 4), ([0, 2], 2)):
        dec.prefill([[1, 2]])
        for n in calls:
            dec.decode(n)
        assert len(steps) == done
        if done < 4:
            with pytest.raises(ValueError, match=f"{4 - done} of 4 are left"):
                dec.decode(4 - done + 1)
        with pytest.raises(ValueError, match="steps must be"):
            dec.decode(5)
        assert len(steps) == done


def test_fixed_tensors_are_not_copied_or_pickled():
    """A copy would have new tensors and the old ones' addresses."""
    h = _holder()
    for way in (copy.copy, copy.deepcopy, pickle.dumps, lambda x: copy.deepcopy([x])):
        with pytest.raises(TypeError, match="cannot be copied or pickled"):
            way(h)
