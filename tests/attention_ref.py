"""Float64 definitions of the attention operators for the tests (torch on the CPU), written
from the formulas, with the error bounds that the kernels' roundings allow.

Bounds.  With u the half-step of the output type (eps / 2) and A = sum_j p_j |v_j| (p the
softmax weights, the sink's share left out of the sum but kept in the denominator):
  - the output's own rounding: u |out|;
  - the weights p_j are rounded to 16 bits before they meet V: at most u' A, u' the half-step
    of the type the products run in (the output's own, or f16 over an E4M3 cache, which is finer);
  - a score's float32 dot product of D terms, the scale and the log2e factor: at most
    (D + 8) 2^-24 S, S the largest |scale| |q|_max sum|k|, and the same for the 2^-25 |q|_max
    a bf16 query loses as an f16 operand; a weight then carries a relative error of twice that
    (its own score and the denominator's), and so the output 2 (D + 8) 2^-24 S A;
  - exponentials, sums of n terms and the division in float32: (2^-20 + n 2^-24) A.
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotated(x, pos, freq, conc):
    """Rows [n, heads, d] at positions pos in float64, rounded to float32."""
    half = x.shape[-1] // 2
    ang = (pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64))[:, None]
    c, s = torch.cos(ang) * conc, torch.sin(ang) * conc
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat((a * c - b * s, b * c + a * s), -1).float()


def e4m3(rows):
    """float32 rows -> (codes as float8_e4m3fn, scale bytes), one exponent a row."""
    codes = torch.empty(rows.shape, dtype=torch.float8_e4m3fn)
    scale = torch.empty(rows.shape[:-1], dtype=torch.uint8)
    flat, fc, fs = rows.reshape(-1, rows.shape[-1]), codes.view(-1, rows.shape[-1]), scale.view(-1)
    top = flat.abs().amax(-1).double()
    e = torch.zeros_like(top)
    ok = torch.isfinite(flat).all(-1)
    pos = ok & (top > 0)
    e[pos] = torch.ceil(torch.log2(top[pos] / 448))
    for _ in range(2):  # the logarithm may be off by one at a border
        e = torch.where(pos & (top > 448 * torch.exp2(e)), e + 1, e)
        e = torch.where(pos & (top <= 448 * torch.exp2(e - 1)), e - 1, e)
    e = e.clamp(-127, 127)
    fc.copy_((flat.double() * torch.exp2(-e)[:, None]).float().to(torch.float8_e4m3fn))
    fs.copy_((e + 127).to(torch.uint8))
    fs[~ok] = 255
    return codes, scale


def values(codes, scale):
    """What stored rows stand for, float64."""
    x = codes.double()
    if scale is None:
        return x
    by = torch.exp2(scale.double() - 127)
    by[scale == 255] = math.nan
    return x * by[..., None]


def rows_of(pages, scale, table, first, count):
    """`count` rows from position `first` of the sequence whose page ids `table` lists: [count, heads, d]."""
    page = pages.shape[2]
    pos = torch.arange(first, first + count)
    ids = table.long()[pos // page]
    sc = None if scale is None else scale[ids, :, pos % page]
    return values(pages.view(torch.uint8)[ids, :, pos % page].view(pages.dtype) if scale is not None
                  else pages[ids, :, pos % page], sc)


def attention(q, k, v, sinks=None, window=0, scale=None, out_type=None):
    """(out, bound): the last len(q) of len(k) positions attend causally.  float64."""
    n, heads, d = q.shape
    m, kv = k.shape[0], k.shape[1]
    scale = scale or 1 / math.sqrt(d)
    out_type = out_type or q.dtype
    q, k, v = q.double(), k.double(), v.double()
    out, bound = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, d, dtype=torch.float64)
    at, key = torch.arange(m - n, m)[:, None], torch.arange(m)[None]
    seen = key <= at
    if window:
        seen &= key > at - window
    u = half_step(out_type)
    any_seen = seen.any(1)
    for h in range(heads):
        kk, vv = k[:, h * kv // heads], v[:, h * kv // heads]
        s = (q[:, h] @ kk.T * scale).masked_fill(~seen, -math.inf)
        top = s.amax(1) if m else torch.full((n,), -math.inf)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        top = torch.where(any_seen, top, torch.zeros_like(top))
        p = torch.exp(s - top[:, None])
        total = p.sum(1) + (torch.exp(sinks[h].double() - top) if sinks is not None else 0)
        p = p / torch.where(any_seen, total, torch.ones_like(total))[:, None]
        p = p.masked_fill(~seen, 0)
        # a masked key contributes nothing, whatever its value
        vis = [torch.nan_to_num(vv, 0, 0, 0) if not torch.isfinite(vv).all() else vv]
        out[:, h] = p @ vis[0]
        if vis[0] is not vv:
            bad = ~torch.isfinite(vv)
            for i in range(n):
                hit = seen[i][:, None] & bad
                if hit.any():
                    out[i, h] = torch.where(hit.any(0), torch.where(seen[i][:, None], p[i][:, None] * vv, 0.0).sum(0),
                                            out[i, h])
        big = (q[:, h].abs().amax(1, keepdim=True) * torch.nan_to_num(kk, 0, 0, 0).abs().sum(1)[None] * scale)
        big = big.masked_fill(~seen, 0).amax(1) if m else torch.zeros(n)
        soft = 2 * (d + 8) * 2.0 ** -24 * big + 2.0 ** -20 + m * 2.0 ** -24
        bound[:, h] = u * out[:, h].abs() + (u + soft)[:, None] * (p @ vis[0].abs())
    # the smallest steps of the output type and a margin for second-order terms
    return out, bound * 1.01 + torch.finfo(out_type).smallest_normal * torch.finfo(out_type).eps


def close(got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got[bad]), torch.isnan(want[bad]))
    fine = ~bad
    assert torch.isfinite(got[fine]).all()
    off = ((got - want).abs() - bound)[fine]
    if off.numel():
        assert off.max() <= 0, (float(off.max()), float((got - want).abs()[fine].max()))
