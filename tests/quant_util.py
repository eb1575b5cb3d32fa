"""Plain 64-bit forms of the 8-bit cache operators, shared by their tests."""

from __future__ import annotations

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def quantise(x: torch.Tensor, code: torch.dtype):
    """Codes and scales of rows x [..., D], every step rounded to fp32 (tensor by tensor
    division: torch divides by a Python scalar with its reciprocal)."""
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.maximum(amax / torch.full_like(amax, QMAX[code]), torch.full_like(amax, 2.0**-126))
    y = x * (torch.ones_like(scale) / scale).unsqueeze(-1)
    if code == torch.int8:
        return torch.round(y).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def dequantise(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return codes.float().double() * scale.double().unsqueeze(-1)


def rotate(key: torch.Tensor, positions: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """Split-half RoPE in fp32 (positions [T], key [T, H, D], table [P, D])."""
    half = key.shape[-1] // 2
    cs = table.float()[positions].unsqueeze(1)
    c, s = cs[..., :half], cs[..., half:]
    lo, hi = key.float()[..., :half], key.float()[..., half:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def sequence(pool: torch.Tensor, table_row: torch.Tensor, n: int) -> torch.Tensor:
    """The first n tokens of a sequence, [Hkv, n, ...], from [blocks, Hkv, bs, ...]."""
    bs = pool.shape[2]
    ids = table_row[: (n + bs - 1) // bs].long()
    raw = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    x = raw[ids].transpose(0, 1).flatten(1, 2)[:, :n]
    return x.view(pool.dtype) if pool.element_size() == 1 else x


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """(out, sum of p |v|) in float64: q [Hq, D], k/v [Hkv, n, D]."""
    hkv = k.shape[0]
    x = torch.einsum("hgd,hnd->hgn", q.double().view(hkv, -1, q.shape[-1]), k.double()) * scale
    p = torch.softmax(x, -1)
    return (torch.einsum("hgn,hnd->hgd", p, v.double()).reshape(q.shape),
            torch.einsum("hgn,hnd->hgd", p, v.double().abs()).reshape(q.shape))


def assert_within(got: torch.Tensor, ref: torch.Tensor, weight: torch.Tensor, what: str = "",
                  half: float | None = None) -> None:
    """got [Hq, D] against ref, weight = sum(p |v|) of the same shape. Allowed: half a step of
    the output type at ref (``half``, by default got's type); half a step of fp16 (2^-11) in
    every probability, 2^-11 weight, with 10% on top for the fp32 sums and exponentials
    (2^-15 relative) and for the output's rounding starting from a value that is off; and for
    probabilities below fp16's normal range 2^-25 each, at most n 2^-32 (n <= 2048 keys:
    2^-21) of the largest p max|v|, which is at most the row's largest weight."""
    if half is None:
        half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = half * ref.abs() + 1.1 * 2.0**-11 * weight + 2.0**-21 * weight.amax(-1, keepdim=True) + 1e-12
    bad = ~(err <= bound)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; at {i} got "
                             f"{float(got[i])} ref {float(ref[i])} bound {float(bound[i])}")
