"""64-bit restatement of the paged key/value cache: rows, 8-bit rows, write, read and attention, from the definitions and
without the library.  Runs on whatever device its inputs are on.

Test infrastructure only.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

E_MIN, E_MAX = -100, 120


def exponent(most: torch.Tensor) -> torch.Tensor:
    """The least integer e in [E_MIN, E_MAX] with most * 2^-e <= 448 (fp64, most >= 0 and finite)."""
    m, x = torch.frexp(most.double())               # most = m 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, x - 8, x - 9)
    return torch.where(most > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def nearest_e4m3(y: torch.Tensor) -> torch.Tensor:
    """y (fp64, |y| <= 448) rounded to the nearest e4m3 value, ties to even."""
    _, x = torch.frexp(y.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(y), x - 4)   # 3 bits behind the leading one; 2^-9 below 2^-6
    return torch.round(y / step) * step


def quantise(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of x (any float type) as 8-bit rows: (the e4m3 numbers in fp64, NaN where x is not finite; e int [..., 1])."""
    x = x.double()
    fine = torch.isfinite(x)
    e = exponent(torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True))
    y = nearest_e4m3(torch.where(fine, x, torch.zeros_like(x)) * torch.exp2(-e.double()))
    return torch.where(fine, y, torch.full_like(y, math.nan)), e


def rows(pages: torch.Tensor, scales: Optional[torch.Tensor], which: int, table: torch.Tensor, b: int, n: int) -> torch.Tensor:
    """The first n rows of sequence b, fp64 [H, n, D]."""
    size = pages.shape[2]
    out = []
    for p in range(-(-n // size)):
        page = int(table[b, p])
        x = pages[page].double()
        if scales is not None:
            x = x * torch.exp2(scales[page, :, :, which].double() - 127.0).unsqueeze(-1)
        out.append(x)
    return torch.cat(out, 1)[:, :n] if out else pages.new_zeros(pages.shape[1], 0, pages.shape[3], dtype=torch.float64)


def attention(q, k_pages, v_pages, table, lens, scale, scales=None, causal=False):
    """(o, M, L, A, S) in fp64 [B, Hq, T, (D)]: output, base-2 row statistics, the weighted sum of |V| and the largest
    scale * sum |q||k| of a row's keys (what the bounds of rounding errors are relative to)."""
    B, Hq, T, D = q.shape
    H = k_pages.shape[1]
    G = Hq // H
    dev = q.device
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=dev)
    A = torch.zeros_like(o)
    M = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=dev)
    L = torch.zeros(B, Hq, T, dtype=torch.float64, device=dev)
    S = torch.zeros(B, Hq, T, dtype=torch.float64, device=dev)
    for b in range(B):
        n = int(lens[b])
        k, v = rows(k_pages, scales, 0, table, b, n), rows(v_pages, scales, 1, table, b, n)
        for t in range(T):
            see = max(0, n - T + t + 1) if causal else n
            if see == 0:
                continue
            qt = q[b, :, t].double().view(H, G, D)
            x = torch.matmul(qt, k[:, :see].transpose(1, 2)) * scale * math.log2(math.e)
            m = x.amax(-1, keepdim=True)
            p = torch.exp2(x - m)
            l = p.sum(-1, keepdim=True)
            o[b, :, t] = (torch.matmul(p, v[:, :see]) / l).reshape(Hq, D)
            A[b, :, t] = (torch.matmul(p, v[:, :see].abs()) / l).reshape(Hq, D)
            M[b, :, t], L[b, :, t] = m.reshape(Hq), l.reshape(Hq)
            S[b, :, t] = (torch.matmul(qt.abs(), k[:, :see].abs().transpose(1, 2)).amax(-1) * scale).reshape(Hq)
    return o, M, L, A, S


def prologue(q, k, scale_mul=None, q_weight=None, k_weight=None, eps=None, cos=None, sin=None, halves=False, start=None):
    """Norm and rotation of q [B, L, Hq, D] and k [B, L, H, D] in fp64, and for every element the sum of the magnitudes
    that its rotation adds (what rounding errors are relative to): (q, k, |q|, |k|)."""
    B, L = q.shape[:2]
    D = q.shape[-1]
    out = []
    for x, mul, w in ((q.double(), scale_mul, q_weight), (k.double(), None, k_weight)):
        if scale_mul is not None:
            x = x / x.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-12)
            if mul is not None:
                x = x * mul.double()[:, None]
        elif eps is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
            if w is not None:
                x = x * w.double()
        size = x.abs()
        if cos is not None:
            pos = torch.as_tensor([[int(s) + i for i in range(L)] for s in start], device=q.device)
            c, s = cos.double()[pos].unsqueeze(2), sin.double()[pos].unsqueeze(2)
            i = torch.arange(D // 2, device=q.device)
            ia, ib = (i, i + D // 2) if halves else (2 * i, 2 * i + 1)
            a, b = x[..., ia], x[..., ib]
            y, size = torch.empty_like(x), torch.empty_like(x)
            y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
            size[..., ia] = size[..., ib] = a.abs() + b.abs()
            x = y
        out += [x, size]
    return out[0], out[2], out[1], out[3]
