"""Plain restatements for the tests of the 4-bit cache and of the q/k-normed append: the quantiser in f32 (its
definition), everything else in f64."""
import math

import numpy as np
import torch


def quantize(x):
    """x [..., 128] -> codes 0..15 [..., 128] (uint8), scale and offset [..., 4] (f32 values of f16 numbers)."""
    g = torch.as_tensor(x).float().unflatten(-1, (4, 32))
    nan = torch.isnan(g).any(-1)
    lo, hi = (torch.nan_to_num(t, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-60000, 60000)
              for t in (g.amin(-1), g.amax(-1)))
    s = ((hi - lo) * (torch.ones(()) / 15)).bfloat16().half().float()
    o = (lo + 8 * s).half().float()
    s, o = torch.where(nan, 0.0, s), torch.where(nan, math.nan, o)
    d = torch.where(s[..., None] > 0, (g - o[..., None]) / s[..., None], torch.zeros(()))
    return (d.round().clamp(-8, 7) + 8).to(torch.uint8).flatten(-2), s, o


def held(x):
    """The f32 values that a 4-bit cache holds for rows x [..., 128]."""
    c, s, o = quantize(x)
    return (o[..., None] + (c.float().unflatten(-1, (4, 32)) - 8) * s[..., None]).flatten(-2)


def attend(q, k, v, seen, scale=None):
    """q [rows, Hq, 128], k, v [Hkv, L, 128], row i sees the first seen[i] tokens -> out, lse in f64."""
    q, k, v = (torch.as_tensor(t).double().cpu() for t in (q, k, v))
    rows, hq, hkv = q.shape[0], q.shape[1], k.shape[0]
    out = torch.zeros(rows, hq, 128, dtype=torch.float64)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    for i, n in enumerate(seen):
        if n:
            kk, vv = (t[:, :n].repeat_interleave(hq // hkv, 0) for t in (k, v))
            s = torch.einsum("hd,hld->hl", q[i], kk) * (scale or 1 / math.sqrt(128))
            lse[i] = torch.logsumexp(s, -1)
            out[i] = torch.einsum("hl,hld->hd", torch.softmax(s, -1), vv)
    return out.numpy(), lse.numpy()


def rope_table(theta, n):
    """The library's f32 table (angle = f32 position * f32 inverse frequency)."""
    from oomllama_b200 import compute_rope_freqs
    sin, cos = compute_rope_freqs(128, n, theta)
    return cos.double(), sin.double()


def normed_rope(x, bias, weight, eps, positions, theta, variant):
    """x [T, H, 128] -> bias, norm of every head (weight None: none), rotation at positions [T]; f64."""
    x = torch.as_tensor(x).double()
    if bias is not None:
        x = x + bias.double().view(-1, 128)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    positions = torch.as_tensor(np.asarray(positions))
    c, s = (t[positions][:, None] for t in rope_table(theta, int(positions.max()) + 1))
    y = torch.empty_like(x)
    a, b = (x[..., :64], x[..., 64:]) if variant == "split_half" else (x[..., 0::2], x[..., 1::2])
    lo, hi = a * c - b * s, a * s + b * c
    if variant == "split_half":
        y[..., :64], y[..., 64:] = lo, hi
    else:
        y[..., 0::2], y[..., 1::2] = lo, hi
    return y


def code_bound(x):
    """How far a held value may be from x [..., 128] (f64): half a step, a step's scale rounded to 8 bits (15 s 2^-9),
    and the offset's half-precision rounding, for a group whose bounds are known to f32 accuracy."""
    g = torch.as_tensor(x).double().unflatten(-1, (4, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = (hi - lo) / 15 * (1 + 2.0 ** -8) + 2.0 ** -24
    return (0.53 * s + (lo.abs() + 8 * s) * 2.0 ** -11 + 1e-5 * g.abs().amax(-1, keepdim=True)).expand(g.shape).flatten(-2)
