"""Host-side checks of the paged cache and of sampling (no GPU): what the entry points refuse
before any CUDA call, that the operators refuse CPU tensors and bad arguments, and that the
argument structs have the header's layout."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

import tilequant_b200 as tq
from tilequant_b200 import _native as N

ROOT = Path(__file__).resolve().parents[1]
A = 4096  # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from tilequant_b200 import build

        build.build()
    return N.load()


def _plan(**kw):
    base = {name: A for name, t in N.PlanArgs._fields_ if t is ctypes.c_void_p}
    base.update(requests=4, table_width=10, page=16, pages=40, max_tokens=64, kv_heads=2, group=4, row_tile=8,
                attn_ctas=296, reserved=0)
    base.update(kw)
    return N.PlanArgs(**base)


def _write(**kw):
    base = {name: A for name, t in N.CacheWriteArgs._fields_ if t is ctypes.c_void_p}
    base.update(ld_k=128, ld_v=128, ld_q=512, ld_qo=512, ld_cs=64, rows=4, requests=4, pages=40, page=16, kv_heads=2,
                q_heads=8, head_dim=64, reserved=0)
    base.update(kw)
    return N.CacheWriteArgs(**base)


def _attn(**kw):
    base = {name: A for name, t in N.PagedAttnArgs._fields_ if t is ctypes.c_void_p}
    base.update(ld_q=512, ld_out=512, rows=4, requests=4, table_width=10, pages=40, page=16, kv_heads=2, q_heads=8,
                head_dim=64, row_tile=8, attn_ctas=296, scale_log2=0.1, reserved=0)
    base.update(kw)
    return N.PagedAttnArgs(**base)


def _sample(**kw):
    base = {name: A for name, t in N.SampleArgs._fields_ if t is ctypes.c_void_p}
    base.update(ld=1000, u_ld=1, u_cols=1, gen_ld=8, gen_cols=8, prompt_tokens=0, n_rows=4, vocab=1000)
    base.update(kw)
    return N.SampleArgs(**base)


@pytest.mark.parametrize("cls,name", [(N.PlanArgs, "tq_plan_args"), (N.CacheWriteArgs, "tq_cache_write_args"),
                                      (N.PagedAttnArgs, "tq_paged_attn_args"), (N.SampleArgs, "tq_sample_args")])
def test_structs_have_the_header_layout(tmp_path, cls, name):
    fields = [f for f, _ in cls._fields_]
    text = (ROOT / "include" / "tilequant_b200.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    declared = [re.sub(r".*[\s*]", "", part.strip()) for line in body.split(";") for part in line.split(",") if part.strip()]
    assert declared == fields
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tilequant_b200.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu ", offsetof({name}, {f}));\n' for f in fields)
                   + f'  printf("%zu", sizeof({name}));\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(n) for n in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(cls, f).offset for f in fields] + [ctypes.sizeof(cls)]


@pytest.mark.parametrize("kw,rc,text", [
    (dict(requests=0), N.TQ_ERR_INVALID, b"requests"), (dict(requests=4097), N.TQ_ERR_INVALID, b"requests"),
    (dict(page=24), N.TQ_ERR_INVALID, b"page size"), (dict(max_tokens=0), N.TQ_ERR_INVALID, b"positive"),
    (dict(row_tile=24), N.TQ_ERR_INVALID, b"row_tile"), (dict(status=None), N.TQ_ERR_INVALID, b"null"),
    (dict(items=A + 8), N.TQ_ERR_INVALID, b"aligned"), (dict(table_width=2**28), N.TQ_ERR_INVALID, b"2^31"),
    (dict(pages=2**28), N.TQ_ERR_INVALID, b"2^31"),
    (dict(table_width=2**20, max_tokens=2**20, kv_heads=8), N.TQ_ERR_INVALID, b"attention work"),
])
def test_plan_step_refusals(lib, kw, rc, text):
    assert lib.tq_plan_step(_plan(**kw), None) == rc and text in lib.tq_last_error()


def test_plan_items_bounds_the_touched_pages(lib):
    assert [lib.tq_plan_items(*a) for a in ((0, 4, 16), (5, 0, 16), (5, 4, 17), (5, 5000, 16))] == [0, 0, 0, 0]
    for page in (16, 32, 64, 128):
        for requests in (1, 3, 50):
            for tokens in (1, 2, page, page + 1, page + 2, 5 * page + 7, 333):
                # the worst split: every request's first token takes the last place of a page
                worst, active = 0, min(tokens, requests)
                for lead in range(1, active + 1):  # one long request beside lead - 1 single tokens
                    n = tokens - (lead - 1)
                    worst = max(worst, lead - 1 + 1 + -(-(n - 1) // page))
                    each = tokens // lead  # or equal ones
                    worst = max(worst, lead * (1 + -(-(each - 1) // page)))
                assert lib.tq_plan_items(tokens, requests, page) >= worst


@pytest.mark.parametrize("kw,dtype,rc,text", [
    (dict(), 7, N.TQ_ERR_INVALID, b"dtype"), (dict(head_dim=96), 0, N.TQ_ERR_UNSUPPORTED, b"head_dim"),
    (dict(page=8), 0, N.TQ_ERR_INVALID, b"page size"), (dict(rows=-1), 0, N.TQ_ERR_INVALID, b"sizes"),
    (dict(k=None), 0, N.TQ_ERR_INVALID, b"null"), (dict(cos=None), 0, N.TQ_ERR_INVALID, b"together"),
    (dict(q_out=None), 0, N.TQ_ERR_INVALID, b"together"), (dict(ld_k=64), 0, N.TQ_ERR_INVALID, b"row stride"),
    (dict(ld_cs=56), 0, N.TQ_ERR_INVALID, b"row stride"), (dict(ld_v=132), 0, N.TQ_ERR_INVALID, b"16-byte"),
    (dict(k=A + 2), 0, N.TQ_ERR_INVALID, b"16-byte"), (dict(sin=A + 8), 0, N.TQ_ERR_INVALID, b"16-byte"),
    (dict(rows=0), 0, N.TQ_OK, b""),
])
def test_cache_write_refusals(lib, kw, dtype, rc, text):
    assert lib.tq_cache_write(_write(**kw), dtype, None) == rc
    assert not text or text in lib.tq_last_error()


@pytest.mark.parametrize("kw,dtype,rc,text", [
    (dict(), 7, N.TQ_ERR_INVALID, b"dtype"), (dict(head_dim=256), 0, N.TQ_ERR_UNSUPPORTED, b"head_dim"),
    (dict(q_heads=7), 0, N.TQ_ERR_INVALID, b"sizes"), (dict(row_tile=4), 0, N.TQ_ERR_INVALID, b"row_tile"),
    (dict(ws_o=None), 0, N.TQ_ERR_INVALID, b"null"), (dict(ld_out=256), 0, N.TQ_ERR_INVALID, b"row stride"),
    (dict(q=A + 8), 0, N.TQ_ERR_INVALID, b"16-byte"), (dict(ld_q=516), 0, N.TQ_ERR_INVALID, b"16-byte"),
    (dict(pages=2**26, kv_heads=4, page=128), 0, N.TQ_ERR_UNSUPPORTED, b"too large"), (dict(rows=0), 0, N.TQ_OK, b""),
])
def test_attn_paged_refusals(lib, kw, dtype, rc, text):
    assert lib.tq_attn_paged(_attn(**kw), dtype, None) == rc
    assert not text or text in lib.tq_last_error()


@pytest.mark.parametrize("kw,dtype,rc,text", [
    (dict(), 3, N.TQ_ERR_INVALID, b"dtype"), (dict(vocab=1048577, ld=1048577), 0, N.TQ_ERR_UNSUPPORTED, b"vocab"),
    (dict(vocab=0), 0, N.TQ_ERR_INVALID, b"rows"), (dict(ld=999), 0, N.TQ_ERR_INVALID, b"rows"),
    (dict(logits=None), 0, N.TQ_ERR_INVALID, b"null"), (dict(ids=None, keys=None), 0, N.TQ_ERR_INVALID, b"null"),
    (dict(u_cols=0), 0, N.TQ_ERR_INVALID, b"random"), (dict(u_cols=3, position=None), 0, N.TQ_ERR_INVALID, b"random"),
    (dict(position=None), 0, N.TQ_ERR_INVALID, b"null"), (dict(n_rows=0), 0, N.TQ_OK, b""),
])
def test_sample_refusals(lib, kw, dtype, rc, text):
    assert lib.tq_sample(_sample(**kw), dtype, None) == rc
    assert not text or text in lib.tq_last_error()


def test_read_and_release_refusals(lib):
    read = lambda **kw: lib.tq_read_pages(*{**dict(k=A, v=A, ks=A, vs=A, ids=A, n=2, pages=4, kv=2, page=16, d=64,  # noqa: E731
                                                   ko=A, vo=A, dtype=0, stream=None), **kw}.values())
    assert read(dtype=9) == N.TQ_ERR_INVALID and read(d=32) == N.TQ_ERR_UNSUPPORTED
    assert read(page=20) == N.TQ_ERR_INVALID and read(n=-1) == N.TQ_ERR_INVALID and read(n=0) == N.TQ_OK
    assert read(ko=A + 8) == N.TQ_ERR_INVALID and b"16-byte" in lib.tq_last_error()
    release = lambda **kw: lib.tq_release_requests(*{**dict(f=A, l=A, t=A, p=A, c=A, s=A, R=4, W=10, page=16, P=40,  # noqa: E731
                                                            stream=None), **kw}.values())
    assert release(R=0) == N.TQ_ERR_INVALID and release(page=1) == N.TQ_ERR_INVALID and release(f=None) == N.TQ_ERR_INVALID


# ------------------------------------------------------------------ the Python operators
def test_construction_errors_come_before_any_device_work():
    with pytest.raises(ValueError, match="page_size"):
        tq.PagePool(4, 1, 64, page_size=20)
    with pytest.raises(ValueError, match="max_requests"):
        tq.PagePool(4, 5000, 64)
    with pytest.raises(ValueError, match="positive"):
        tq.PagePool(0, 1, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        tq.PagePool(2**26, 1, 64)
    with pytest.raises(ValueError, match="CUDA device"):
        tq.PagePool(4, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        tq.KVPages(4, 1, 16, 96)
    with pytest.raises(ValueError, match="too large"):
        tq.KVPages(2**24, 8, 16, 128)
    pool = SimpleNamespace(device=torch.device("cpu"), max_requests=2, page_size=16)
    with pytest.raises(ValueError, match="multiple"):
        tq.StepPlan(pool, 4, q_heads=5, kv_heads=2, head_dim=64)
    with pytest.raises(ValueError, match="max_tokens"):
        tq.StepPlan(pool, 0, q_heads=4, kv_heads=2, head_dim=64)


def test_sampling_refuses_cpu_tensors_and_bad_shapes():
    x, u = torch.zeros(2, 10).half(), torch.zeros(2)
    with pytest.raises(ValueError, match="no CPU path"):
        tq.sample_tokens(x, u)
    with pytest.raises(ValueError, match="no CPU path"):
        tq.sample_pick(x, u[:, None], torch.zeros(2).long(), torch.zeros(1).long(), 0)


def test_sampling_settings_are_checked():
    for kw in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(top_p=1.1), dict(min_p=-0.5),
               dict(top_k=2**31)):
        with pytest.raises(ValueError):
            tq.Sampling(**kw)
    rows = tq.Sampling(temperature=0.5, top_k=3).rows(2, torch.device("cpu"))
    assert rows["temperature"].tolist() == [0.5, 0.5] and rows["top_k"].tolist() == [3, 3]
    assert rows["top_k"].dtype == torch.int32


def test_decoder_refuses_what_the_int8_cache_cannot_do():
    from transformers import LlamaConfig, LlamaForCausalLM

    from tilequant_b200.graph_decode import CudaGraphGreedyDecoder

    cfg = dict(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2,
               head_dim=32, vocab_size=32)
    model = LlamaForCausalLM(LlamaConfig(**cfg)).eval()
    with pytest.raises(ValueError, match="kv_cache"):
        CudaGraphGreedyDecoder(model, prompt_tokens=4, max_new_tokens=4, kv_cache="fp8")
    with pytest.raises(ValueError, match="head_dim 32"):
        CudaGraphGreedyDecoder(model, prompt_tokens=4, max_new_tokens=4, kv_cache="int8")
    with pytest.raises(ValueError, match="fused_decode is off"):
        CudaGraphGreedyDecoder(model, prompt_tokens=4, max_new_tokens=4, kv_cache="int8", fused_decode=False)


def test_fixed_tensors_are_copied_into_not_replaced():
    class Holder(N.FixedTensors):
        def __init__(self):
            self.a, self.n = torch.zeros(2), 1

    h = Holder()
    h.n = 2
    h.a.fill_(1)
    with pytest.raises(AttributeError, match="copy into it"):
        h.a = torch.ones(2)


def test_benchmark_sampling_arguments():
    from tilequant_b200.benchmark_generation import sampling_of

    args = SimpleNamespace(temperature=None, top_k=0, top_p=1.0, min_p=0.0, seed=0)
    assert sampling_of(args) is None
    args.temperature, args.top_k = 0.7, 5
    assert sampling_of(args) == tq.Sampling(temperature=0.7, top_k=5)


@pytest.mark.parametrize("batch", [1, 8, 64])
@pytest.mark.parametrize("prompt", [1, 77, 8192, 131072, 500000])
@pytest.mark.parametrize("kv_heads", [1, 4, 8, 32])
def test_prompts_of_one_plan_stay_in_its_count(batch, prompt, kv_heads):
    from tilequant_b200.decode_step import _prompt_requests

    room = (prompt + 64 + 63) // 64 * 64
    n = _prompt_requests(batch, prompt, kv_heads, room)
    work = lambda n: (n * prompt / 16 + batch) * kv_heads * (room / 128 + 4)  # noqa: E731  (as tq_plan_step bounds it)
    assert 1 <= n <= batch
    assert work(n) < 2**31 or n == 1
    assert n == batch or work(n + 1) > 0.95 * 2**31  # no more plans than needed
