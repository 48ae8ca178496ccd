"""Plain statements of the rotary and 8-bit-cache operators for the tests: torch on
the CPU, float64 (float32 where a rounding step is part of the definition)."""
from __future__ import annotations

import math

import torch

PAGE, BLOCK, RING = 64, 16, 32
TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def rope(x, pos, freq, layout, factor):
    """x [T, heads, dim] -> float64."""
    y = x.double().clone()
    half = freq.numel()
    t = pos.double()[:, None] * freq.double()[None]
    c, s = torch.cos(t)[:, None] * factor, torch.sin(t)[:, None] * factor
    ia = torch.arange(half) if layout == "half" else 2 * torch.arange(half)
    ib = ia + half if layout == "half" else ia + 1
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def quantise(rows, code):
    """Blocks [..., 16, D] -> (codes, scales [...]): the largest magnitude over top, rounded
    to float32, and the exact quotients x top / amax rounded to codes."""
    x = rows.float()
    most = x.abs().amax((-1, -2))
    fine = torch.isfinite(most)
    top = TOP[code]
    scale = torch.where(fine, most / top, torch.full_like(most, math.nan))
    r = (x.double() * top / most.double()[..., None, None]).float()
    r = torch.where((fine & (most > 0))[..., None, None], r, torch.zeros_like(r))
    return (r.round() if code == "int8" else r).to(CODE[code]), scale


class Model:
    """What the cache should hold: each sequence's 16-bit rows [n, H, D] (the whole
    history); the codes follow from them."""

    def __init__(self, seqs, heads, dim, code, dtype):
        self.rows = [[torch.zeros(0, heads, dim, dtype=dtype) for _ in range(seqs)] for _ in range(2)]
        self.code = code

    def append(self, b, k, v):
        self.rows[0][b] = torch.cat([self.rows[0][b], k])
        self.rows[1][b] = torch.cat([self.rows[1][b], v])

    def cut(self, b, n):
        for s in range(2):
            self.rows[s][b] = self.rows[s][b][:n]

    def blocks(self, side, b):
        x = self.rows[side][b]
        n, H, D = x.shape
        x = torch.cat([x, torch.zeros(-n % BLOCK, H, D, dtype=x.dtype)])
        return quantise(x.reshape(-1, BLOCK, H, D).transpose(1, 2), self.code)       # [nb, H, 16, D], [nb, H]

    def values(self, side, b):
        """[n, H, D] float32: code * scale, one rounding (what a read returns)."""
        n = self.rows[side][b].shape[0]
        code, scale = self.blocks(side, b)
        x = code.float() * scale[..., None, None]
        return x.transpose(1, 2).reshape(-1, *self.rows[side][b].shape[1:])[:n]


def attend(q, k, v, scale, window=0):
    """q [n, heads, D] at the last n positions over k, v [len, H, D]: out and lse, float64,
    and for each key and kv head the weights' sum over rows and heads [H, len]."""
    n, heads, D = q.shape
    L, H = k.shape[0], k.shape[1]
    G = heads // H
    s = torch.einsum("nhgd,lhd->hgnl", q.double().reshape(n, H, G, D), k.double()) * scale
    p = torch.arange(n) + L - n
    j = torch.arange(L)
    seen = j[None] <= p[:, None]
    if window:
        seen &= j[None] > p[:, None] - window
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1) if L else torch.full((H, G, n), -math.inf, dtype=torch.float64)
    w = torch.where(seen, torch.exp(s - lse[..., None]), torch.zeros_like(s))
    vv = v.double()[None, :].expand(1, L, H, D)[0]
    # a key that a row does not see adds nothing, whatever its value
    o = torch.zeros(n, H, G, D, dtype=torch.float64)
    for i in range(n):
        sel = seen[i]
        o[i] = torch.einsum("hgl,lhd->hgd", w[:, :, i][:, :, sel], vv[sel])
    return o.reshape(n, heads, D), lse.permute(2, 0, 1).reshape(n, heads), w.sum((1, 2))


def attend_bound(q, k, v, scale, dtype, ref):
    """How far an output may be from `ref`, elementwise.  The kernels' steps: the score
    is a float32 sum of D products (at most D + 4 roundings of the magnitudes' sum A:
    the products, the sums, two scalings), a row in 16 bits may be scaled by a power
    of two into F16 (2^-25 of its largest entry per entry, inside the same bound with
    one more rounding of A); exp adds a few units; the running sums over L keys and the
    join of the parts at most L + 16 roundings, and the weights may be rounded to F16
    before the product with V (2^-11 relative, 2^-24 absolute below F16's range).
    The output's own rounding is half a step."""
    n, heads, D = q.shape
    L, H = k.shape[0], k.shape[1]
    if L == 0:
        return torch.zeros_like(ref)
    G = heads // H
    A = torch.einsum("nhgd,lhd->nhgl", q.double().abs().reshape(n, H, G, D), k.double().abs()).amax(-1) * abs(scale)
    u = 2.0 ** -24
    ds = (D + 6) * u * A
    rel = 2 * ds + (L + 32) * u + 2.0 ** -11
    vmax = v.double().abs().amax(0)[None, :, None]                                   # [1, H, 1, D]
    b = rel[..., None] * vmax
    return b.reshape(n, heads, D) + torch.finfo(dtype).eps / 2 * (ref.abs() + b.reshape(n, heads, D)) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def score_bound(q, k, scale):
    """How far lse may be, [n, heads]."""
    n, heads, D = q.shape
    L, H = k.shape[0], k.shape[1]
    if L == 0:
        return torch.zeros(n, heads, dtype=torch.float64)
    A = torch.einsum("nhgd,lhd->nhgl", q.double().abs().reshape(n, H, heads // H, D), k.double().abs()).amax(-1) * abs(scale)
    u = 2.0 ** -24
    return ((D + 6) * u * A + (L + 32) * u + 2 * u * (A + math.log(L))).reshape(n, heads)


def keep(weight, n, budget, sinks, recent):
    """Positions that stay of one (sequence, head): the definition, by sorting."""
    if n <= budget:
        return list(range(n))
    w = weight.tolist()
    order = sorted(range(sinks, n - recent), key=lambda i: (0, 0, i) if math.isnan(w[i]) else (1, -w[i], i))
    return sorted(list(range(sinks)) + order[: budget - sinks - recent] + list(range(n - recent, n)))


def requantise(code_rows, scales, code):
    """Codes [N, D] (as float) with their scales [N], N a multiple of 16 -> new (codes, scales [N / 16])."""
    top = TOP[code]
    x = code_rows.float().reshape(-1, BLOCK, code_rows.shape[-1])
    s = scales.float().reshape(-1, BLOCK)
    new = (s * (x.abs().amax(-1) / top)).amax(-1)
    ratio = torch.where(new[:, None] > 0, s / new[:, None], torch.zeros_like(s))
    r = (x * ratio[..., None]).clamp(-top, top)
    return (r.round() if code == "int8" else r).to(CODE[code]), new
