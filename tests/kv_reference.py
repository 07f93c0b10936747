"""The key/value cache operators in 64 bits (NumPy-style torch on the CPU), from
their definition in include/q4rdna.h, and the tolerances of the tests.

Tolerances (u = 2^-24, half a step of f32; e = half a step of the output type):

* rotated q and k, f32 arithmetic: the norm's factor comes from a sum of D
  squares (a lane's own up to 8 and 5 shuffle steps: under 14 u, halved by the
  root), rsqrtf (2 ulp = 4 u) and two products: under 14 u; the reduced angle
  is rounded once (pi u) and sincosf is within 2 ulp (4 u): under 8 u for each of
  the two terms, which are then rounded twice more.  Altogether |error| <=
  32 u (|a| + |b|) for the pair (a, b), and e |y| for the output type.
* a scale: the same 32 u sqrt(2) relative, for the largest |x| of a tile, and a
  division: 48 u.
* a code: x / s is off by 32 u sqrt(2) relative to the tile's largest value (and
  the rounding of 1 / s and of the product), under 64 u * top of a step; so
  |code - x / s| <= 1/2 + 64 u top for int8, and half a step of e4m3 (2^-4
  relative, 2^-10 below the normal numbers) likewise.
* attention: scores are exact products of codes summed in f32, with q in at
  least 22 bits: |error| <= 2^-19 A, A = scale * sum |q k| of the row's largest
  key, in the exponent; the same for the sum, so twice, and 2^-19 for the
  exponential, the sums over tokens in f32 and the join of pieces.  16-bit types
  hold the weights in 11 bits: 2^-11 more.  All relative to sum p |v|, and e |y|.
"""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
CODE = {0: torch.int8, 1: torch.float8_e4m3fn}
TOP = {0: 127.0, 1: 448.0}


def parts(tiles, D, fmt):
    """Views of the tiles: scales [..., 2], key and value codes [..., 16, D]."""
    t = CODE[fmt]
    return (tiles[..., :8].view(torch.float32), tiles[..., 16:16 + 16 * D].view(t).unflatten(-1, (16, D)),
            tiles[..., 16 + 16 * D:].view(t).unflatten(-1, (16, D)))


def numbers(tiles, D, fmt):
    """(k, v) f64 [pages, heads, page_tokens, D]."""
    s, k, v = parts(tiles, D, fmt)
    return tuple((c.float() * s[..., i, None, None]).double().flatten(2, 3) for i, c in ((0, k), (1, v)))


def fill(tiles, D, fmt, seed, k_scale=1.0, v_scale=1.0):
    """Random codes and scales everywhere (tiles on the CPU)."""
    g = torch.Generator().manual_seed(seed)
    s, k, v = parts(tiles, D, fmt)
    for i, (c, f) in enumerate(((k, k_scale), (v, v_scale))):
        x = torch.randn(c.shape, generator=g) * f
        sc = x.abs().amax((-1, -2)) / TOP[fmt]
        s[..., i] = sc
        x = x / sc[..., None, None]
        c.copy_((x.round() if fmt == 0 else x.clamp(-TOP[fmt], TOP[fmt])).to(CODE[fmt]))
    return tiles


def attention(tiles, D, fmt, table, lengths, news, q, window=0, scale=0.0):
    """(out, mag, A) f64: mag = sum p |v|, A = the largest scale * sum |q k| of a
    row; news[s] rows of sequence s, all of them rows of q [T, heads, D]."""
    kk, vv = numbers(tiles, D, fmt)
    H = tiles.shape[1]
    T, Hq, _ = q.shape
    G = Hq // H
    scale = scale or 1 / math.sqrt(D)
    out, mag, big = (torch.zeros((T, Hq, D), dtype=torch.float64) for _ in range(3))
    row = 0
    for s, n in enumerate(news):
        L = int(lengths[s])
        pages = table[s, : -(-L // (kk.shape[2]))].long()
        K, V = (x[pages].transpose(0, 1).flatten(1, 2)[:, :L] for x in (kk, vv))  # [H, L, D]
        for i in range(n):
            p = L - n + i
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                continue
            x = q[row + i].double().reshape(H, G, D)
            k, v = K[:, lo:p + 1], V[:, lo:p + 1]
            w = torch.softmax(x @ k.transpose(-1, -2) * scale, -1)
            out[row + i] = (w @ v).reshape(Hq, D)
            mag[row + i] = (w @ v.abs()).reshape(Hq, D)
            big[row + i] = ((x.abs() @ k.abs().transpose(-1, -2)) * scale).amax(-1).reshape(Hq, 1)
        row += n
    return out, mag, big


def check_attention(y, ref, dtype, what=""):
    out, mag, big = ref
    y = y.double().cpu()
    assert torch.isfinite(y).all(), f"{what}: not finite"
    rel = 2 * (big * 2.0 ** -19) + 2.0 ** -19 + (0.0 if dtype == torch.float32 else 2.0 ** -11)
    bound = mag * rel + HALF[dtype] * (out.abs() + mag * rel) + 1e-30
    worst = ((y - out).abs() / bound).max().item() if y.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"
    return worst


def turned(x, w, pos, inv_freq, rot, neox, eps):
    """(y, mag) f64 of [rows, heads, D]: norm, rotation; mag = |a| + |b|."""
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y, mag = x.clone(), x.abs()
    if inv_freq is not None:
        rot = rot or D
        h = rot // 2
        ang = pos.double()[:, None] * inv_freq.double()
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        ia, ib = (torch.arange(h), torch.arange(h) + h) if neox else (2 * torch.arange(h), 2 * torch.arange(h) + 1)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        mag = mag.clone()
        mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def check_append(before, after, D, fmt, table, lengths, news, k, v, what=""):
    """The tiles after an append of k, v (f64 [T, H, D], already turned) against
    the definition, step by step: scales, new codes, older codes, all else
    untouched.  before / after: tiles on the CPU."""
    P = after.shape[2] * 16
    top = TOP[fmt]
    half_step = (lambda x: torch.full_like(x, 0.5)) if fmt == 0 else (
        lambda x: torch.maximum(x.abs() * 2.0 ** -4, torch.full_like(x, 2.0 ** -10)))
    want = before.clone()
    s0, c0 = parts(before, D, fmt)[0], parts(before, D, fmt)[1:]
    s1, c1 = parts(after, D, fmt)[0], parts(after, D, fmt)[1:]
    row = 0
    for s, n in enumerate(news):
        L = int(lengths[s])
        for b in range(max(0, L - n) // 16, -(-L // 16)):
            lo, hi = max(L - n, 16 * b, 0), min(L, 16 * b + 16)
            if lo >= hi:
                continue
            at = (int(table[s, 16 * b // P]), slice(None), b % (P // 16))
            rows = slice(row + lo - (L - n), row + hi - (L - n))
            for z, x in ((0, k), (1, v)):
                x = x[rows].transpose(0, 1)  # [H, tokens, D]
                amax = x.abs().amax((-1, -2)) / top
                old = s0[at][:, z].double() if lo > 16 * b else torch.zeros_like(amax)
                got = s1[at][:, z].double()
                ref = torch.maximum(amax, old)
                assert ((got - ref).abs() <= 48 * U * ref).all(), f"{what}: scale of block {b}"
                sc = got[:, None, None]
                y = x / sc
                off = (c1[z][at].double()[:, lo - 16 * b:hi - 16 * b] - y).abs()
                assert (off <= half_step(y) * (1 + 2.0 ** -20) + 64 * U * top).all(), f"{what}: codes of block {b}"
                was = c0[z][at].double()[:, : lo - 16 * b]
                y = was * (old / got)[:, None, None]
                off = (c1[z][at].double()[:, : lo - 16 * b] - y).abs()
                grown = (got > old)[:, None, None]
                lim = torch.where(grown, half_step(y) * (1 + 2.0 ** -20) + 64 * U * top, torch.zeros_like(y))
                assert (off <= lim).all(), f"{what}: older codes of block {b}"
                ws, wc = parts(want, D, fmt)[0], parts(want, D, fmt)[1 + z]
                ws[at][:, z] = s1[at][:, z]
                wc[at][:, : hi - 16 * b] = c1[z][at][:, : hi - 16 * b]
        row += n
    assert torch.equal(want, after), f"{what}: bytes outside the new tokens changed"
