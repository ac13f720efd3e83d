"""The 8-bit cache in 64 bits: its format, and attention over rows held in it, from the definitions."""

from __future__ import annotations

import torch

F64 = torch.float64


def e4m3_numbers() -> torch.Tensor:
    """All e4m3 numbers >= 0, in the order of their codes: 2^(max(E, 1) - 7) * (M / 8 + [E > 0])."""
    code = torch.arange(127, dtype=torch.int64)               # 127 is no number
    e, m = code >> 3, (code & 7).to(F64)
    return torch.exp2((e.clamp(min=1) - 7).to(F64)) * (m / 8 + (e > 0).to(F64))


def nearest_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number, ties to the even code."""
    table = e4m3_numbers()
    a = x.abs().to(F64)
    hi = torch.searchsorted(table, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = a - table[lo], table[hi] - a
    take_lo = (below < above) | ((below == above) & (lo % 2 == 0))
    return torch.where(take_lo, table[lo], table[hi]) * torch.where(torch.signbit(x), -1.0, 1.0)


def row_exponents(x: torch.Tensor) -> torch.Tensor:
    """Per row (last dimension) of finite numbers: the smallest e in -120..120 with 448 * 2^e >= max |x|."""
    steps = 448 * torch.exp2(torch.arange(-120, 121, dtype=F64))
    return torch.searchsorted(steps, x.abs().to(F64).amax(dim=-1).contiguous()).clamp(max=240) - 120


def quantise(x: torch.Tensor):
    """(codes as numbers, exponents; exponent 128 for rows that are not finite) of rows."""
    x = x.to(F64)
    fine = torch.isfinite(x).all(dim=-1)
    safe = torch.where(fine[..., None], x, torch.zeros_like(x))
    e = row_exponents(safe)
    codes = nearest_e4m3(safe * torch.exp2(-e.to(F64))[..., None])
    limit = torch.where(e == 120, 240.0, 448.0)[..., None]
    codes = torch.minimum(torch.maximum(codes, -limit), limit)
    return torch.where(fine[..., None], codes, torch.zeros_like(codes)), torch.where(fine, e, torch.full_like(e, 128))


def to_tensors(codes: torch.Tensor, e: torch.Tensor):
    """(float8_e4m3fn codes, uint8 exponent bytes): exact."""
    held = codes.to(torch.float32).to(torch.float8_e4m3fn)
    assert torch.equal(held.to(F64), codes.to(F64))
    return held, (e + 127).to(torch.uint8)


def dequantise(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    power = torch.where(byte == 255, torch.full((), float("nan"), dtype=F64), torch.exp2(byte.to(F64) - 127))
    return codes.to(F64) * power[..., None]


def sees(pos: int, length: int, window=None, chunk=None, keep_first: int = 0) -> torch.Tensor:
    """Which of ``length`` keys the query at ``pos`` reads."""
    j = torch.arange(length)
    ok = torch.ones(length, dtype=torch.bool)
    if window:
        ok &= j > pos - window
    if chunk:
        ok &= j // chunk == pos // chunk
    return (ok | (j < keep_first)) & (j <= pos)


def attention(q, k, v, scale: float, before: int, window=None, chunk=None, keep_first=0, sink=None):
    """q [n, nq, d] at positions ``before``..; k, v [L, nkv, d] (a key or value that is NaN spoils the queries that read it,
    all entries).  Returns (out [n, nq, d], its error's yardsticks: sum of weights times |v|, largest sum |q k| scale)."""
    n, nq, d = q.shape
    rep = nq // k.shape[1]
    q, k, v = q.to(F64), k.to(F64).repeat_interleave(rep, 1), v.to(F64).repeat_interleave(rep, 1)
    out, spread, size = torch.empty_like(q), torch.empty_like(q), torch.zeros(n, nq, dtype=F64)
    for i in range(n):
        at = sees(before + i, k.shape[0], window, chunk, keep_first)
        kk, vv = k[at], v[at]
        spoilt = (torch.isnan(kk).any(-1) | torch.isnan(vv).any(-1)).any(0)                 # per head
        s = torch.einsum("hd,lhd->hl", q[i], torch.nan_to_num(kk)) * scale
        size[i] = (q[i].abs()[None] * torch.nan_to_num(kk).abs()).sum(-1).amax(0) * scale
        s = torch.cat([s, sink.to(F64)[:, None]], 1) if sink is not None else s
        p = torch.softmax(s, dim=1)[:, :kk.shape[0]]
        out[i] = torch.einsum("hl,lhd->hd", p, torch.nan_to_num(vv))
        spread[i] = torch.einsum("hl,lhd->hd", p, torch.nan_to_num(vv).abs())
        out[i][spoilt] = float("nan")
    return out, spread, size
