"""Plain restatements of the paged-cache operators and of sampling, for their tests: whole
numbers request by request, values in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import torch

POOL_EMPTY, TABLE_FULL, ROWS_FULL, BAD_PAGE = 1, 2, 4, 8


class RefPool:
    """A page pool as Python lists."""

    def __init__(self, num_pages, requests, width, page):
        self.P, self.R, self.W, self.page = num_pages, requests, width, page
        self.lengths = [0] * requests
        self.table = [[-1] * width for _ in range(requests)]
        self.stack = list(range(num_pages - 1, -1, -1))

    def step(self, new, max_tokens):
        page, status = self.page, 0
        slots, positions = [-1] * max_tokens, [-1] * max_tokens
        cu, kv, tok, wanted = [0], [], 0, 0
        avail = len(self.stack)
        for r, n in enumerate(new):
            n, L = max(n, 0), self.lengths[r]
            first, tok = tok, tok + n
            ok = n > 0
            if n and L + n > self.W * page:
                status, ok = status | TABLE_FULL, False
            if n and tok > max_tokens:
                status, ok = status | ROWS_FULL, False
            if ok:
                need = -(-(L + n) // page) - -(-L // page)
                wanted += need
                if need and wanted > avail:
                    status, ok = status | POOL_EMPTY, False
            cu.append(min(tok, max_tokens))
            kv.append(L + n if ok else 0)
            if not ok:
                continue
            for i in range(n):
                p = L + i
                if p % page == 0:
                    self.table[r][p // page] = self.stack.pop()
                positions[first + i] = p
                slots[first + i] = self.table[r][p // page] * page + p % page
            self.lengths[r] = L + n
        return dict(slots=slots, positions=positions, cu_new=cu, kv_len=kv, status=status)

    def release(self, finished):
        for r, f in enumerate(finished):
            if f:
                for i in range(-(-self.lengths[r] // self.page)):
                    self.stack.append(self.table[r][i])
                    self.table[r][i] = -1
                self.lengths[r] = 0


def f32(x):
    """Rounded to 32 bits, held in 64 (for quotients and products of 32-bit values this is
    the 32-bit operation)."""
    return x.float().double()


def rotate(x, cos, sin):
    """[tokens, heads, D] 16-bit; each product and the sum rounded, as the decoder does."""
    t = x.dtype

    def r(v):
        return v.float().to(t).double()

    h = x.shape[-1] // 2
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([r(r(a * cos[..., :h]) + r(-b * sin[..., :h])), r(r(b * cos[..., h:]) + r(a * sin[..., h:]))], -1)


def write_side(x, codes, scale, slots, positions):
    """x [tokens, heads, D] (64 bits, of 16-bit values) into codes int8 [P, H, page, D] and scale f32
    [P, H], both changed in place.  Tokens of one page are consecutive rows."""
    page = codes.shape[2]
    t, n = 0, x.shape[0]
    while t < n:
        if slots[t] < 0:
            t += 1
            continue
        pg, off = divmod(slots[t], page)
        e = t + 1
        while e < n and slots[e] == slots[t] + e - t and slots[e] // page == pg and positions[e] == positions[t] + e - t:
            e += 1
        rows = x[t:e].transpose(0, 1)  # heads, tokens, D
        finite = torch.isfinite(rows)
        most = torch.where(finite, rows.abs(), 0.0).amax((1, 2))
        old = scale[pg].double() if off else torch.zeros_like(most)
        s = torch.maximum(old, f32(most / 127))
        grown = s > old
        if off and bool(grown.any()):
            ratio = f32(old / s)[:, None, None]
            held = codes[pg, :, :off].double()
            codes[pg, :, :off] = torch.where(grown[:, None, None], torch.round(f32(held * ratio)), held).to(torch.int8)
        q = torch.round(f32(rows / s[:, None, None])).clamp(-127, 127)
        q = torch.where((s[:, None, None] > 0) & ~torch.isnan(rows), q, 0.0)
        codes[pg, :, off:off + e - t] = q.to(torch.int8)
        scale[pg] = s.float()
        t = e


def attend(q, k_codes, v_codes, k_scale, v_scale, table, cu_new, kv_len, scale, eps):
    """(out, tolerance) [rows, Hq * D] in 64 bits, on the tensors' device.

    The tolerance counts, for the kernel's arithmetic, per output: the output's rounding eps/2
    |o|; with A = sum p |v| / sum p: P's rounding to f16, 2^-11 A; the scores' error d, from q's
    rounding to integers of a row scaled to [2^14, 2^15) (|rounding| |k| scale, summed) and four
    f32 roundings of s and of the exponent's argument (2^-21 |s|), entering numerator and sum:
    2 d A; ex2 and the f32 sums of P and P V, (n / 32 + 64) 2^-23 A each, twice."""
    rows, hk, d, page = q.shape[0], k_codes.shape[1], k_codes.shape[3], k_codes.shape[2]
    G = q.shape[1] // d // hk
    out = torch.zeros(rows, q.shape[1], dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for r in range(len(kv_len)):
        n, t0, t1 = kv_len[r], cu_new[r], min(cu_new[r + 1], rows)
        if n == 0 or t1 <= t0:
            continue
        w = cu_new[r + 1] - t0
        at = table[r][:-(-n // page)]
        for h in range(hk):
            k = (k_codes[at, h].double() * k_scale[at, h].double()[:, None, None]).reshape(-1, d)[:n]
            v = (v_codes[at, h].double() * v_scale[at, h].double()[:, None, None]).reshape(-1, d)[:n]
            qq = q[t0:t1].view(t1 - t0, hk, G, d)[:, h].double()
            s = torch.einsum("wgd,nd->wgn", qq, k) * scale
            top = torch.floor(torch.log2(qq.abs().amax(-1, keepdim=True).clamp(min=2.0**-120)))
            unit = torch.exp2(top - 14)
            qe = (qq - torch.round(qq / unit) * unit).abs()
            sa = torch.einsum("wgd,nd->wgn", qe, k.abs()) * abs(scale)
            late = torch.arange(n, device=q.device) > (n - w + torch.arange(t1 - t0, device=q.device))[:, None]
            s = s.masked_fill(late[:, None], -math.inf)
            p = torch.softmax(s, -1)
            o = torch.einsum("wgn,nd->wgd", p, v)
            A = torch.einsum("wgn,nd->wgd", p, v.abs())
            seen = torch.where(late[:, None], 0.0, 1.0)
            ds = (sa * seen).amax(-1) + 2.0**-21 * torch.where(late[:, None], 0.0, s).abs().amax(-1)
            rel = 2.0**-11 + 2 * ds + 2 * (n / 32 + 64) * 2.0**-23
            out.view(rows, hk, G, d)[t0:t1, h] = o
            tol.view(rows, hk, G, d)[t0:t1, h] = eps / 2 * o.abs() + rel[..., None] * A + 2.0**-25
    return out, tol


def sample_row(x, u, T=1.0, k=0, p=1.0, min_p=0.0):
    """(id, log-probability) of one row of logits (64-bit numpy values)."""
    order = np.lexsort((np.arange(len(x)), -np.where(np.isnan(x), -np.inf, x)))
    order = order[(x[order] > -np.inf)]
    if not len(order):
        return 0, -np.inf
    top = x[order[0]]
    if not T > 0:
        return int(order[0]), 0.0
    if np.isinf(top):
        w = (x[order] == top).astype(np.longdouble)
    else:
        with np.errstate(under="ignore", over="ignore"):
            w = np.exp((x[order] - top) / T).astype(np.longdouble)
    if k > 0:
        w = w[:k]
    if p < 1.0:
        w = w[:int(np.searchsorted(np.cumsum(w), np.longdouble(p) * w.sum(), side="left")) + 1]
    if min_p > 0:
        w = w[:max(1, int((w >= min_p).sum()))]
    total = w.sum()
    u = u if u > 0 else 0.0
    at = min(int(np.searchsorted(np.cumsum(w), np.longdouble(u) * total, side="right")), len(w) - 1)
    while at > 0 and w[at] == 0:  # nothing of no weight is sampled
        at -= 1
    return int(order[at]), float(np.log(w[at] / total))
