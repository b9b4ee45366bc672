"""The 8-bit cache's format and attention over it, from their definitions, in 64 bits (plain torch, any device).

A row's scale is 2^e with e the smallest integer of [-100, 119] for which max|x| <= 448 * 2^e; its numbers are x * 2^-e rounded to the
nearest e4m3 number, ties to the even one, at most 448 in size.  A row with an infinity or a NaN has scale byte 255 and reads as NaN."""
import math

import torch

PAGE = 64


def code_values(device="cpu"):
    """What each of the 256 codes stands for."""
    out = []
    for b in range(256):
        exponent, fraction = (b >> 3) & 15, b & 7
        x = math.ldexp(fraction, -9) if exponent == 0 else math.ldexp(8 + fraction, exponent - 10)
        out.append(math.nan if b & 127 == 127 else -x if b & 128 else x)
    return torch.tensor(out, dtype=torch.float64, device=device)


def quantise(x):
    """Rows [..., hd] -> (codes uint8 [..., hd], scale bytes uint8 [...])."""
    x = x.double()
    finite = torch.isfinite(x).all(dim=-1)
    y = torch.where(finite[..., None], x, torch.zeros_like(x))
    amax = y.abs().amax(dim=-1)
    e = torch.full_like(amax, -100.0)
    for k in range(-100, 119):                       # the smallest that holds the row, by the definition
        e = torch.where(amax > 448.0 * 2.0 ** k, torch.full_like(e, k + 1.0), e)
    y = (y * torch.exp2(-e)[..., None]).clamp(-448.0, 448.0)
    positive = code_values(x.device)[:127]           # rising
    mag = y.abs()
    up = torch.searchsorted(positive, mag.contiguous()).clamp(max=126)
    low = (up - 1).clamp(min=0)
    below, above = mag - positive[low], positive[up] - mag
    code = torch.where((below < above) | ((below == above) & (low % 2 == 0)), low, up)       # even codes have an even last bit
    code = torch.where(mag == 0, torch.zeros_like(code), code)
    code = code + 128 * torch.signbit(y)
    code = torch.where(finite[..., None], code, torch.zeros_like(code))
    return code.to(torch.uint8), torch.where(finite, e + 127, torch.full_like(e, 255.0)).to(torch.uint8)


def values(codes, scale):
    s = torch.exp2(scale.double() - 127.0)
    s = torch.where(scale == 255, torch.full_like(s, math.nan), s)
    return code_values(codes.device)[codes.long()] * s[..., None]


def visible(positions, n_keys, window=0, keep_first=0, chunk=0):
    """bool [rows, n_keys]"""
    p = positions.long()[:, None]
    j = torch.arange(n_keys, device=positions.device)[None, :]
    seen = j <= p
    if window:
        seen = seen & ((p - j < window) | (j < keep_first))
    if chunk:
        seen = seen & (j >= (p // chunk) * chunk)
    return seen


def attention(q, k, v, seen, scale, sinks=None, softcap=0.0):
    """One sequence: q [rows, H, hd], k and v [keys, KV, hd], seen [rows, keys].  Returns (out, bound), both [rows, H, hd]: bound is how far a
    16-bit result may be off, from these roundings:
      the score in float32, hd products and sums of numbers up to |q||k|, and what scales and shifts it: (hd + 8) 2^-24 of |q|.|k| scale,
        and the exponential's own error, 2^-21 (two units of a float32 exponential's argument of up to 2^2 and its result's two);
        a score off by d makes its weight off by d of itself, and numerator and denominator both: 2 d;
      the weight as the second product's operand, half a step of bfloat16 at most: 2^-8; where it is below float16's normal numbers
        2^-25 of the largest weighted row instead;
      the result's own rounding: 2^-8."""
    rows, H, hd = q.shape
    group = H // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    raw = torch.einsum("rhd,khd->hrk", q, k) * scale
    size = torch.einsum("rhd,khd->hrk", q.abs(), k.abs()) * scale
    s = softcap * torch.tanh(raw / softcap) if softcap else raw
    s = s.masked_fill(~seen, -math.inf)
    off = ((hd + 8) * 2.0 ** -24 * size + 2.0 ** -21 + 2.0 ** -22 * max(softcap, 0.0)).masked_fill(~seen, 0.0)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    nothing = (total == 0).expand(-1, -1, 1)
    if sinks is not None:
        total = total + torch.exp(sinks.double()[:, None, None] - top)
    w = w / total
    w = torch.where(nothing, torch.zeros_like(w), w)
    vv = torch.where(seen.any(0)[:, None, None], v, torch.zeros_like(v))       # what nobody sees may be anything
    out = torch.einsum("hrk,khd->rhd", w, vv)
    size_out = torch.einsum("hrk,khd->rhd", w, vv.abs())
    d = off.amax(-1).transpose(0, 1)[..., None]                               # [rows, H, 1]
    small = seen.sum(-1).double()[:, None, None] * 2.0 ** -24 * (w * vv.abs().amax(-1).transpose(0, 1)[:, None, :]).amax(-1).transpose(0, 1)[..., None]
    e = (2.0 ** -8 + 2 * d) * size_out + small
    return out, e + 2.0 ** -8 * (out.abs() + e) + 1e-37
