"""float64 definitions of the paged cache's operators, written from their formulas with numpy and torch on the CPU.

Tolerances: bf16 rounds by at most 2^-8 of the value, e4m3 by 2^-4 of it (2^-10 of
the scale below 2^-6 of the scale), fp32 by 2^-24.
"""
import math

import numpy as np
import torch


def inv_freq(rot, base=10000.0, scaling="none", factor=1.0, original=0):
    """(angle per position of each pair in float64, factor on cos and sin)."""
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    inv = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "by_parts":
        pair = lambda n: rot * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def rotate(x, positions, rot, interleaved, inv, m):
    """(rotated x in float64, sum of the magnitudes of each output's two terms); x [T, H, D]."""
    x = np.asarray(x, dtype=np.float64)
    angle = np.asarray(positions, dtype=np.float64)[:, None] * inv
    c, s = (np.cos(angle) * m)[:, None], (np.sin(angle) * m)[:, None]
    out, mag = x.copy(), np.abs(x)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    u, w = x[..., a], x[..., b]
    out[..., a], out[..., b] = u * c - w * s, w * c + u * s
    mag[..., a] = mag[..., b] = (np.abs(u) + np.abs(w)) * m
    return out, mag


# One rotated value: the phase's rounding to fp32 turns the angle by at most pi 2^-25 = 9.4e-8, sincospif is
# off by at most 2 ulp (2^-23), and the factor, two products and the sum round by 2^-24 each: below 4.6e-7 of
# |u| + |w| together.  numpy's own float64 angles add 2^-53 of the angle (checked at positions below 2^22: 5e-10).
ROPE_ERR = 5e-7


def exponent(amax, limit):
    """The least e with amax <= limit 2^e, clamped to [-100, 120]; 0 for 0.  Exact (python floats)."""
    if amax == 0:
        return 0
    m, e = math.frexp(amax)
    ml, el = math.frexp(limit)
    return max(-100, min(120, e - el + (1 if m > ml else 0)))


def key_limit(mscale):
    limit = 448.0 / (math.sqrt(2.0) * mscale)
    f = np.float32(limit)
    return float(np.nextafter(f, np.float32(0)) if float(f) > limit else f)


def places(q_start, kv_len, page):
    """(token, sequence, position) of every new token of every sequence."""
    for b, n in enumerate(kv_len):
        n_new = q_start[b + 1] - q_start[b]
        for i in range(n_new):
            yield q_start[b] + i, b, n - n_new + i


def values(pages, exps=None):
    """Pages as float64 values (a torch tensor on the CPU)."""
    x = pages.cpu()
    if exps is None:
        return x.double()
    x = x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x
    return x.float().double() * torch.exp2(exps.cpu().double() - 127)[..., None]


def gather(vals, table, b, length):
    """[length, kv_heads, D]: the first positions of sequence b."""
    page = vals.shape[2]
    ids = table[b, :-(-length // page)].long().cpu()
    return vals[ids].transpose(1, 2).flatten(0, 1)[:length]


def attend(q, k, v, n_before, scale):
    """One sequence: q [n, H, D] at positions n_before and on, k, v [L, K, D], all float64.  Returns the outputs, the
    sums of p |v| and the largest sum of |q_d k_d| scale of each row: what the error bound is made of."""
    n, H, D = q.shape
    L, K, _ = k.shape
    out, mag = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    big = torch.zeros(n, H, 1, dtype=torch.float64)
    for i in range(n):
        vis = max(0, min(L, n_before + i + 1))
        if vis == 0:
            continue
        kk = k[:vis].repeat_interleave(H // K, dim=1)
        vv = v[:vis].repeat_interleave(H // K, dim=1)
        s = torch.einsum("hd,jhd->hj", q[i], kk) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hj,jhd->hd", p, vv)
        mag[i] = torch.einsum("hj,jhd->hd", p, vv.abs())
        big[i, :, 0] = torch.einsum("hd,jhd->hj", q[i].abs(), kk.abs()).amax(-1) * abs(scale)
    return out, mag, big


def attention_bound(out, mag, big, D):
    """How far an output may be off: its rounding to bf16, the weights' rounding to 8 bits' mantissa (2^-8 of
    each), fp32 sums of D products in any order (D 2^-24 of the magnitudes, an error of the score and so twice of its
    weight and of the sum they are divided by), 2^-18 for the exponentials and the fp32 sums over positions."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 4 * D * 2.0 ** -24 * big + 2.0 ** -18) * mag + 1e-30
