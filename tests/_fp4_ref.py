"""Plain 64-bit forms of the FP4 operators for the tests: the format's definition on tensors, without the library."""
import math

import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantize(x):
    """(codes uint8, scale bytes uint8) of x [..., 32 g], by search over the format's scales and magnitudes."""
    x = x.double().cpu().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    exps = torch.arange(-125, 126)
    fits = top.unsqueeze(-1) <= 7 * torch.exp2(exps.double())
    at = fits.to(torch.int8).argmax(-1)   # the least scale that fits
    bad = ~torch.isfinite(top) | ~fits.any(-1)
    e = exps[at]
    a = x.abs() / torch.exp2(e.double()).unsqueeze(-1)
    # nearest magnitude; of two as near the even code
    d = (a.unsqueeze(-1) - GRID).abs() * 2 + (torch.arange(8) % 2) * 1e-12
    code = d.argmin(-1).to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)
    code[bad] = 0
    byte = (e + 127).to(torch.uint8)
    byte[bad] = 255
    return code.flatten(-2), byte


def values(code, byte):
    """float64 values of codes [..., 32 g]."""
    v = GRID[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.exp2(byte.double() - 127)
    s[byte == 255] = math.nan
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def halves(code):
    return (code[..., 0::2] | code[..., 1::2] << 4).contiguous()


def rounded(x):
    """Values of x after quantisation."""
    return values(*quantize(x))


def norm_rope(x, w, eps, pos, theta, rope_scale=1.0):
    """x [S, heads, hd] normed per head by w [hd] (or None), then rotated at pos [S, hd / 2] (or None)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if pos is None:
        return x
    half = x.shape[-1] // 2
    ang = pos.double() * theta ** (-torch.arange(half, dtype=torch.float64) / half) / rope_scale
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attention(q, k, v, causal):
    """(output, bound of its error) of q [n, hq, hd] over k, v [kv, hkv, hd], all float64.

    The bound counts what a kernel may round: the output (2^-8 of it), each weight to bf16 (2^-8 of its share), and the
    scores' fp32 sums: hd / 32 + 32 additions of products, the scaling and the exponential's argument, 2^-23 each, of
    the sum of magnitudes. An error d of a score changes its weight, and through the sum all weights, by 2 d. Weights under
    2^-126 are subnormal in bf16 and fp32, where the relative bounds end: each may be lost whole, 2^-126 of its value."""
    n, hq, hd = q.shape
    kv, hkv, _ = k.shape
    out, tol = torch.zeros(n, hq, hd, dtype=torch.float64), torch.zeros(n, hq, hd, dtype=torch.float64)
    if kv == 0:
        return out, tol
    seen = torch.arange(kv)[None] <= torch.arange(n)[:, None] + (kv - n) if causal else torch.ones(n, kv, dtype=torch.bool)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
        s = (q[:, h] @ kh.T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
        mag = (q[:, h].abs() @ kh.abs().T / math.sqrt(hd)).masked_fill(~seen, 0)
        p = torch.softmax(s, -1)
        out[:, h] = p @ vh
        d = (hd / 32 + 40) * 2.0 ** -23 * mag.amax(-1, keepdim=True)
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + (p @ vh.abs()) * (2.0 ** -8 + 2 * d + 2.0 ** -18)
        tol[:, h] += kv * 2.0 ** -126 * vh.abs().amax()
    return out, tol
