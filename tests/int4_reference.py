"""Plain 64-bit forms of the 4-bit pool's operators, and pools to run them on (torch on the CPU)."""

from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def quantize(x: torch.Tensor):
    """``(codes [..., D] uint8, step [..., 1], mid [..., 1])`` of rows ``x`` (the
    format's own fp32 operations; step and mid in x's type)."""
    f = x.float()
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    mid = (lo / 2 + hi / 2).to(x.dtype)
    step = (torch.maximum(hi - mid.float(), mid.float() - lo) / 7.5).to(x.dtype)
    code = torch.where(step > 0, (torch.floor((f - mid.float()) / step.float()) + 8).clamp(0, 15),
                       torch.full_like(f, 8.0))
    ok = torch.isfinite(f).all(-1, keepdim=True)
    nan = torch.full_like(mid, math.nan)
    return (torch.where(ok, code, torch.full_like(code, 8.0)).to(torch.uint8),
            torch.where(ok, step, torch.zeros_like(step)), torch.where(ok, mid, nan))


def pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def values(kv_codes: torch.Tensor, kv_params: torch.Tensor) -> torch.Tensor:
    """float64 values of a pool (or rows of one): ``[..., D]``."""
    c = torch.stack([kv_codes & 15, kv_codes >> 4], -1).flatten(-2).double()
    p = kv_params.double()
    return p[..., 1:2] + p[..., 0:1] * (c - 7.5)


def make_pool(gen, layers, blocks, hkv, bs, d, dtype, spread=None):
    """A pool of quantised normal rows; ``spread``: rows scaled by powers of
    two up to 2^spread, with offsets, so that steps and mids vary."""
    x = torch.randn(layers, blocks, hkv, 2, bs, d, generator=gen)
    if spread:
        x = x * torch.exp2(torch.randint(-spread, spread + 1, x.shape[:-1] + (1,), generator=gen).float())
        x = x + torch.randn(x.shape[:-1] + (1,), generator=gen)
    code, step, mid = quantize(x.to(dtype))
    return pack(code), torch.cat([step, mid], -1)


def shuffled_tables(gen, lens, bs, spare=3, extra_cols=2):
    """Tables of a shuffled pool for ``lens`` (unused entries point past the
    pool's end, which nothing may read) and the number of blocks."""
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need + [0]) + extra_cols), 1 << 30, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    return table, blocks


def poison(kv_codes, kv_params, layer, table, lens, bs):
    """Copies whose rows outside the sequences hold NaN parameters (codes keep
    whatever they were)."""
    params = torch.full_like(kv_params, math.nan)
    for b, n in enumerate(lens):
        for j in range(-(-n // bs)):
            blk, rows = int(table[b, j]), min(bs, n - j * bs)
            params[layer, blk, :, :, :rows] = kv_params[layer, blk, :, :, :rows]
    return kv_codes.clone(), params


def sequence_rows(kv_codes, kv_params, layer, blocks, n, bs):
    """(values [Hkv, n, D], deviations from mid [Hkv, n, D], step, |mid| [Hkv, n]) for K and for V."""
    pos = torch.arange(n)
    blk, off = blocks.long()[pos // bs], pos % bs
    c, p = kv_codes[layer, blk, :, :, off], kv_params[layer, blk, :, :, off]  # [n, Hkv, 2, .]
    v = values(c, p)
    dev = v - p[..., 1:2].double()
    out = []
    for i in range(2):
        out.append(tuple(t.transpose(0, 1) for t in (v[:, :, i], dev[:, :, i], p[:, :, i, 0].double(),
                                                      p[:, :, i, 1].double().abs())))
    return out


def attend(q, kv_codes, kv_params, layer, blocks, n, bs, first, scale, keep=None):
    """Attention of query rows ``q [R, Hq, D]`` (row r sees positions 0 ..
    first + r of a sequence of n tokens) in 64 bits, and a bound of what an
    fp32 evaluation with ``step * probability`` rounded to q's type may be off
    by.  ``keep [n]``: positions that exist (False: a block outside the pool).

    Bound, with h half a step of the type (2^-24 for fp32):
      h |out|                     the output's own rounding;
      h sum p |v - mid|           step * p rounded before the product with the codes (16-bit types);
      2 d sum p |v|               a relative error of each probability of at most d = the error of a score:
                                  sums of D + 8 fp32 products of q with codes offset by at most 272 and of the
                                  offset's correction, 2^-23 each relative to sum |q| (272 step + |mid|) scale,
                                  and 2^-22 of the score for the exponential's argument;
      (n + 64) 2^-23 sum p |v|    the fp32 sums over n tokens.
    """
    r, hq, d = q.shape
    hkv = kv_codes.shape[2]
    group = hq // hkv
    out = torch.zeros(r, hq, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    h = HALF_STEP[q.dtype]
    if n == 0:
        return out, tol
    (k, _, kst, kmid), (v, vdev, _, _) = sequence_rows(kv_codes, kv_params, layer, blocks, n, bs)
    seen = torch.arange(n)[None, :] <= first + torch.arange(r)[:, None]
    if keep is not None:
        seen = seen & keep[None, :]
    offset = 0.0 if q.dtype == torch.float32 else 272.0
    for a in range(hq):
        kh = a // group
        qd = q[:, a].double()
        s = (qd @ k[kh].T) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), 0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        vv = torch.where(seen.any(0)[:, None], v[kh], 0.0)
        dd = torch.where(seen.any(0)[:, None], vdev[kh], 0.0)
        out[:, a] = p @ vv
        size = qd.abs().sum(-1, keepdim=True) * (offset * kst[kh].abs() + kmid[kh] + 8 * kst[kh].abs())[None, :] * abs(scale)
        ds = torch.where(seen, size * (d + 8) * 2.0 ** -23, 0.0).amax(-1, keepdim=True)
        ds = ds + torch.where(seen, s.abs(), 0.0).amax(-1, keepdim=True) * 2.0 ** -21
        mass = p @ vv.abs()
        tol[:, a] = h * out[:, a].abs() + (h if q.dtype != torch.float32 else 0.0) * (p @ dd.abs()) \
            + (2 * ds + (n + 64) * 2.0 ** -23) * mass + 1e-12
    if q.dtype == torch.float16:
        tol += 2.0 ** -25  # half a step of the subnormals
    return out, tol


def rotate(x, cos, sin):
    """x cos + rotate_half(x) sin with each product and the sum rounded to x's type."""
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    a = (x.double() * cos.double()).to(x.dtype).double()
    b = (turned.double() * sin.double()).to(x.dtype).double()
    return (a + b).to(x.dtype)
