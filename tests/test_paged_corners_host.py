"""Host-side checks of the serving operators' corners (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

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
