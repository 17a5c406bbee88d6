"""Token sampling from given random numbers (``csrc/sample.cu``), the sampled counterpart of
``decode_step.greedy_pick``.

Tokens are taken in falling order of their logit, equal ones by index, with weights
exp((logit - max) / temperature) in 64 bits.  Each filter keeps a head of that order, and they
apply one after the other: ``top_k`` the first k, ``top_p`` the shortest head that holds at
least that share of what top_k kept, ``min_p`` the tokens of at least that weight relative to
the first.  The first token always stays.  The sampled token is the first whose running sum of
weights exceeds ``uniform`` times the kept sum, so a call is a function of its inputs alone.
(A share that falls on the border between two tokens, to within the 64-bit rounding of their
sums, may take either.)
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _native as N
from .trace import traced

MAX_VOCAB = 1 << 20


@dataclass(frozen=True)
class Sampling:
    """Sampling settings of a whole batch, with the seed of its random numbers."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self) -> None:
        if not self.temperature >= 0.0:
            raise ValueError("temperature must be 0 or above")
        if not 0.0 <= self.top_p <= 1.0 or not 0.0 <= self.min_p <= 1.0:
            raise ValueError("top_p and min_p must be in [0, 1]")
        if not -(2**31) <= self.top_k < 2**31:
            raise ValueError("top_k must be a 32-bit number")

    def rows(self, n: int, device: torch.device) -> dict:
        """The settings as the operators' arguments for ``n`` rows."""
        full = lambda v, dtype: torch.full((n,), v, dtype=dtype, device=device)  # noqa: E731
        return dict(temperature=full(self.temperature, torch.float32), top_k=full(self.top_k, torch.int32),
                    top_p=full(self.top_p, torch.float32), min_p=full(self.min_p, torch.float32))


def _unit_columns(t: torch.Tensor) -> bool:
    return t.stride(1) == 1 or t.shape[1] == 1  # (the stride of a dimension of size 1 means nothing)


def _param(t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, index: int, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [{rows}] tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}, not {t.device}")
    return t.data_ptr()


def _args(logits: torch.Tensor, uniform: torch.Tensor, temperature, top_k, top_p, min_p, what: str) -> N.SampleArgs:
    if not (logits.is_cuda and uniform.is_cuda):
        raise ValueError("tilequant_b200 kernels need CUDA tensors (there is no CPU path)")
    if logits.dim() != 2 or logits.shape[1] < 1 or not _unit_columns(logits):
        raise ValueError(f"{what}: logits must be a [rows, vocab] tensor with unit column stride")
    rows, vocab = logits.shape
    index = logits.get_device()
    if rows > 1 and logits.stride(0) < vocab:
        raise ValueError(f"{what}: rows of logits must not overlap")
    if vocab > MAX_VOCAB:
        raise ValueError(f"{what}: at most {MAX_VOCAB} logits per row")
    if uniform.dtype != torch.float32 or uniform.dim() not in (1, 2) or uniform.shape[0] != rows \
            or uniform.get_device() != index:
        raise ValueError(f"{what}: uniform must be a float32 tensor of one number (or row) per row of logits")
    a = N.SampleArgs()
    a.logits, a.uniform = logits.data_ptr(), uniform.data_ptr()
    a.temperature = _param(temperature, torch.float32, rows, index, f"{what}: temperature")
    a.top_k = _param(top_k, torch.int32, rows, index, f"{what}: top_k")
    a.top_p = _param(top_p, torch.float32, rows, index, f"{what}: top_p")
    a.min_p = _param(min_p, torch.float32, rows, index, f"{what}: min_p")
    a.ld, a.u_ld, a.u_cols = logits.stride(0) if rows > 1 else vocab, uniform.stride(0), 1
    a.n_rows, a.vocab = rows, vocab
    return a


@traced("tq.sample_tokens")
def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Optional[torch.Tensor] = None,
                  top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                  min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  logprobs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token id per row of ``logits`` [rows, vocab] (bf16 or f16) and its
    log-probability among the kept tokens (int64 and float32 [rows]).

    ``uniform`` float32 [rows] in [0, 1).  ``temperature``, ``top_p``, ``min_p`` float32 and
    ``top_k`` int32 [rows], each optional: a temperature of 0 (or below, or NaN) takes the largest
    logit; top_k <= 0, top_p >= 1 and min_p <= 0 keep everything.  -inf and NaN logits are never sampled; a
    row of nothing else gives token 0 and log-probability -inf."""
    a = _args(logits, uniform, temperature, top_k, top_p, min_p, "sample_tokens")
    code = N.dtype_code(logits.dtype)
    if uniform.dim() != 1:
        raise ValueError("sample_tokens: uniform must be a float32 [rows] tensor")
    rows, index = a.n_rows, logits.get_device()
    out = torch.empty(rows, dtype=torch.int64, device=logits.device) if out is None else out
    logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device) if logprobs is None else logprobs
    a.ids = _param(out, torch.int64, rows, index, "sample_tokens: out")
    a.logprobs = _param(logprobs, torch.float32, rows, index, "sample_tokens: logprobs")
    if rows:
        N.check(N.on_device(index, N.load().tq_sample, ctypes.byref(a), code, N.raw_stream(index)), "sample_tokens")
    return out, logprobs


@traced("tq.sample_pick")
def sample_pick(logits: torch.Tensor, uniform: torch.Tensor, keys: torch.Tensor, position: torch.Tensor,
                prompt_tokens: int, *, temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
                top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None,
                next_ids: Optional[torch.Tensor] = None, token: Optional[torch.Tensor] = None,
                generated: Optional[torch.Tensor] = None) -> None:
    """A decode step's sampled pick and bookkeeping: ``greedy_pick`` with the token of
    ``sample_tokens``.  ``uniform`` [B, n] holds the numbers of n steps: the step uses column
    position - prompt_tokens + 1 (the column of ``generated`` it fills)."""
    N.require_cuda(logits, uniform, keys, position, next_ids, token, generated)
    a = _args(logits, uniform, temperature, top_k, top_p, min_p, "sample_pick")
    code = N.dtype_code(logits.dtype)
    B = int(a.n_rows)
    if uniform.dim() != 2 or uniform.shape[1] < 1 or not _unit_columns(uniform):
        raise ValueError("sample_pick: uniform must be a float32 [B, n] tensor with unit column stride")
    if not 1 <= B <= 1024:
        raise ValueError("sample_pick: 1..1024 rows of logits")
    if keys.dtype != torch.int64 or keys.numel() < B or not keys.is_contiguous() or position.dtype != torch.int64 \
            or position.numel() != 1:
        raise ValueError("sample_pick: int64 keys [B] and position [1]")
    for t in (next_ids, token):
        if t is not None and (t.dtype != torch.int64 or t.numel() != B or not t.is_contiguous()):
            raise ValueError("sample_pick: next/token must be contiguous int64 [B] tensors")
    if generated is not None and (generated.dtype != torch.int64 or generated.dim() != 2 or generated.shape[0] != B
                                  or not _unit_columns(generated)):
        raise ValueError("sample_pick: generated must be int64 [B, T] with unit column stride")
    a.u_cols, a.keys, a.position, a.prompt_tokens = uniform.shape[1], keys.data_ptr(), position.data_ptr(), int(prompt_tokens)
    a.next, a.token, a.generated = N.ptr(next_ids), N.ptr(token), N.ptr(generated)
    a.gen_ld = 0 if generated is None else generated.stride(0)
    a.gen_cols = 0 if generated is None else generated.shape[1]
    index = logits.get_device()
    N.check(N.on_device(index, N.load().tq_sample, ctypes.byref(a), code, N.raw_stream(index)), "sample_pick")
