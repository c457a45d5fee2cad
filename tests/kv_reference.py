"""Plain 64-bit forms of the quantised paged KV cache operators (torch, any device)."""
import math

import torch


def quantise(x, bits):
    """(codes [.., D] as integers, scale, zero) of groups over the last axis.
    f32 scale and zero as the cache holds them; codes from exact quotients."""
    x = x.float()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    safe = torch.where(finite, x, torch.zeros_like(x))
    lo, hi = safe.amin(-1, keepdim=True), safe.amax(-1, keepdim=True)
    if bits == 8:
        scale = (safe.abs().amax(-1, keepdim=True).double() / 127).float()
        zero, low, high, mid = torch.zeros_like(scale), -127, 127, 128
    else:
        span = hi - lo
        finite &= torch.isfinite(span)
        scale = (span.double() / 15).float()
        zero, low, high, mid = lo + 8 * scale, -8, 7, 8
    one = torch.ones_like(scale)
    c = (safe.double() - zero.double()) / torch.where(scale > 0, scale, one).double()
    c = torch.where(finite & (scale > 0), c.round().clamp(low, high), torch.zeros_like(c))
    nan = torch.full_like(scale, math.nan)
    scale, zero = torch.where(finite, scale, nan), torch.where(finite, zero, nan)
    return c.to(torch.int64) + mid, scale, zero


def pack(codes, bits):
    codes = codes.to(torch.uint8)
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def held(codes, scale, zero, bits):
    """Values in 64 bits."""
    if bits == 8:
        return scale.double() * (codes.double() - 128)
    return zero.double() + scale.double() * (codes.double() - 8)


def side(codes, scales, bits):
    """(scale * code, zero) of cache buffers, 64 bits: [.., D] and [.., 1]."""
    if bits == 8:
        return scales.double() * (codes.double() - 128), torch.zeros_like(scales[..., :1]).double()
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return scales[..., :1].double() * (c.double() - 8), scales[..., 1:].double()


def attention(q, cache, lens, table, window=0, sinks=0, scale=None):
    """(out, spread, reach, floor) in 64 bits per row [rows, heads, D] / [rows, heads, 1].

    lens: (new tokens, cache length) per sequence, rows in order.  spread is
    sum p (|scale code| + |zero|), what a relative error of the weights can
    move the output by; reach the largest scale * sum|q||k| a row meets, what
    an error of the scores is relative to; floor the largest p * max(scale, |zero|)
    of a row times sum|code|, what an absolute error of the weights can move it by."""
    heads, d = q.shape[1], q.shape[2]
    hkv, page = cache.kv_heads, cache.page_tokens
    group = heads // hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    floor = torch.zeros_like(out)
    reach = torch.zeros((*q.shape[:2], 1), dtype=torch.float64, device=q.device)
    at = 0
    for b, (n, kv) in enumerate(lens):
        rows = slice(at, at + n)
        at += n
        if n == 0 or kv == 0:
            continue
        pos = torch.arange(kv - n, kv, device=q.device)[:, None]
        key = torch.arange(kv, device=q.device)[None]
        seen = key <= pos
        if window:
            seen = seen & ((key > pos - window) | (key < sinks))
        need = seen.any(0)
        tok = torch.nonzero(need).flatten()
        ids = table[b].long()[tok // page]
        for h in range(hkv):
            k0, kz = side(cache.k_codes[ids, h, tok % page], cache.k_scales[ids, h, tok % page], cache.bits[0])
            v0, vz = side(cache.v_codes[ids, h, tok % page], cache.v_scales[ids, h, tok % page], cache.bits[1])
            see = seen[:, tok]
            for g in range(group):
                qq = q[rows, h * group + g].double()
                s = (qq @ k0.T + qq.sum(-1, keepdim=True) * kz.T) * scale
                s = s.masked_fill(~see, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
                p = torch.where(see, p, torch.zeros_like(p))
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                vv = torch.where(need[tok][:, None], v0 + vz, torch.zeros_like(v0))
                hidden_nan = torch.isnan(vv) & ~see.any(0)[:, None]
                vv = torch.where(hidden_nan, torch.zeros_like(vv), vv)
                out[rows, h * group + g] = _times(p, vv, see)
                spread[rows, h * group + g] = _times(p, v0.abs() + vz.abs(), see)
                sv = cache.v_scales[ids, h, tok % page][:, 0].double()
                mag = torch.maximum(sv, vz[:, 0].abs())
                weight = torch.nan_to_num(torch.where(see, p * mag, torch.zeros_like(p))).amax(-1, keepdim=True)
                code = torch.nan_to_num(v0 / sv[:, None]).abs()
                floor[rows, h * group + g] = weight * (see.double() @ code)
                a = (qq.abs() @ k0.abs().T + qq.abs().sum(-1, keepdim=True) * kz.abs().T) * scale
                a = torch.where(see, a, torch.zeros_like(a))
                reach[rows, h * group + g] = a.amax(-1, keepdim=True)
    return out, spread, reach, floor


def _times(p, v, see):
    """p @ v where a row takes nothing from tokens that it does not see, whatever they hold."""
    bad = ~torch.isfinite(v).all(-1)
    clean = p @ torch.where(bad[:, None], torch.zeros_like(v), v)
    touched = (see & bad[None]).any(-1, keepdim=True)
    return torch.where(touched, torch.full_like(clean, math.nan), clean)


def tolerance(ref, spread, reach, floor, dtype):
    """How far an output may be from the 64-bit one, element by element.

    - the output's own rounding: eps / 2 of the value;
    - the weights p * scale are rounded to f16 (2^-11 of each), for f32 queries
      to f16 hi + lo (2^-22, taken as 2^-21);
    - the scores: q as f16 hi + lo (2^-22) and at most 32 f32 roundings of
      2^-23 relative to scale * sum|q||k|, that is 2^-18, in the numerator and
      in the sum: a factor 2 ln 2 < 1.5 of it in base 2;
    - exp2 and the running sums in f32: 2^-18 of everything summed;
    - f16 has no step below 2^-24: the reference puts the largest
      p * max(scale, |zero|) of a row at 2^3 or more, so each weight, and the lo
      half for f32 queries, is off by up to 2^-25 / 2^3 = 2^-28 of the largest
      whatever its own size (a dimension in which the largest weight meets code
      zero shows that alone)."""
    w = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    return torch.finfo(dtype).eps / 2 * ref.abs() + (w + 1.5 * 2.0 ** -18 * reach + 2.0 ** -18) * spread \
        + 2.0 ** -28 * floor + 1e-30
