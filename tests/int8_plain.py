"""Plain forms of the operators of 8-bit codes, on the CPU, and how far a kernel's results may be from them."""
import math

import torch

PAGE = 64


def codes_of(x):
    """float32 rows (the last dimension) -> int8 codes and float32 scales, each step rounded as float32 is."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    zero = top < 2.0 ** -100
    most = torch.full_like(top, 127.0)  # (a quotient of two tensors is rounded once; by a number it is a product with a reciprocal)
    inverse = torch.where(zero, torch.zeros_like(top), most / top)
    codes = torch.round(x * inverse)
    scales = torch.where(zero, torch.zeros_like(top), top / most)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, torch.zeros_like(codes), codes).to(torch.int8), torch.where(bad, torch.full_like(top, math.nan), scales)[..., 0]


def rotate(x, cos, sin):
    """Halves of the last dimension turned, each product and sum rounded by itself, the result to x's type."""
    half, y = x.shape[-1] // 2, x.float()
    a, b = y[..., :half], y[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)


def angles(positions, d):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return torch.cos(a).float(), torch.sin(a).float()


def store(pages, kv_heads, d, gen):
    """Random codes and scales."""
    x = torch.randn((pages, kv_heads, PAGE, d), generator=gen)
    codes, scales = codes_of(x)
    return codes, scales * (0.5 + torch.rand(scales.shape, generator=gen))


def attention(q, k, v, k_scales, v_scales, positions, seqs, table, heads, kv_heads, window, scale, exact_q=True):
    """float64 (out, bound) of every row: ``bound`` is how far a kernel may be, output rounding included.

    Of a score: sums and products of float32 are (d + 4) roundings of at most 2^-24 of the magnitudes' sum; a query held in
    16-bit codes (``exact_q`` False) is off by at most half a step, top / 65,024, per value.  A weight's relative error is that
    of its exponent, twice (its own and the maximum's), two roundings of 2^-11 where it is held in 16 bits (else of 2^-22, an
    exponential's), and as much again through the sum that it is divided by; what a weight times its value's scale is below 2^-29 of
    the largest times the largest is held to 2^-39 of it (float16 behind a factor of 2^15, next to a power of two above the scales).
    The output is rounded to half a step of its type."""
    n, d = q.shape[0], q.shape[1] // heads
    per, dtype = heads // kv_heads, q.dtype
    out, bound = torch.zeros((n, heads, d), dtype=torch.float64), torch.zeros((n, heads, d), dtype=torch.float64)
    for r in range(n):
        pos, seq = positions[r], seqs[r]
        if pos < 0 or not 0 <= seq < len(table):
            continue
        first = max(0, pos - window + 1) if window else 0
        at = [(table[seq][t // PAGE], t % PAGE) for t in range(first, min(pos + 1, len(table[seq]) * PAGE))]
        at = [(p, s) for p, s in at if 0 <= p < k.shape[0]]
        if not at:
            continue
        page, slot = (torch.tensor(x) for x in zip(*at))
        for h in range(heads):
            keys = k[page, h // per, slot].double() * k_scales[page, h // per, slot].double()[:, None]
            values = v[page, h // per, slot].double() * v_scales[page, h // per, slot].double()[:, None]
            x = q[r, h * d:(h + 1) * d].double()
            scores = keys @ x * scale
            p = torch.softmax(scores, 0)
            out[r, h] = p @ values
            off = (d + 4) * 2.0 ** -24 * (keys.abs() @ x.abs()).max() * scale
            if not exact_q:
                off = off + x.abs().max() / 65024 * keys.abs().sum(1).max() * scale
            rounding = 2.0 ** -22 if exact_q else 2.0 ** -11
            relative = 2 * (math.expm1(2 * float(off)) + 2 * rounding + len(at) * 2.0 ** -24)
            small = 2.0 ** -38 * float(p.max()) * float(v_scales[page, h // per, slot].max())
            bound[r, h] = relative * p @ values.abs() + small * v[page, h // per, slot].double().abs().sum(0) + torch.finfo(dtype).eps / 2 * out[r, h].abs() + 1e-30
    return out.reshape(n, -1), bound.reshape(n, -1)


def product(x, w, k, w_scales, bias, gated):
    """float64 (y, bound) of codes w [rows, width] and rows x [m, k]: the sums are exact, then come at most four roundings of float32,
    of a gated product those of its exponential and quotient too (the error of exp(-g) grows with g: |g| 2^-23), and the output's."""
    codes, scales = codes_of(x)
    a = (codes.double() @ w[:, :k].double().T) * scales.double()[:, None] * w_scales.double()
    y = a + (bias.double() if bias is not None else 0.0)
    off = 4 * 2.0 ** -24 * (a.abs() + y.abs())
    if not gated:
        return y, off + torch.finfo(x.dtype).eps / 2 * y.abs() + 1e-37
    n = y.shape[1] // 2
    gate, up, silu = y[:, :n], y[:, n:], y[:, :n] * torch.sigmoid(y[:, :n])
    out = silu * up
    # silu's slope is at most 1.1
    off = 1.1 * off[:, :n] * up.abs() + silu.abs() * off[:, n:] + (8 + 2 * gate.abs()) * 2.0 ** -23 * out.abs()
    return out, off * 1.01 + torch.finfo(x.dtype).eps / 2 * out.abs() + 1e-37
