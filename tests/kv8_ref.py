"""Caches held in 8 bits, restated in 64 bits: the format, the rows of a step, attention with its sums, key weights, eviction.
Plain torch in float64; every rounding is done by arithmetic on the numbers."""
from __future__ import annotations

import math

import torch

from diffgemma_b200 import capi

BLOCK = 128


def low(x):
    """Rounded to bf16 (by way of fp32, as a cast does)."""
    return x.float().to(torch.bfloat16).double()


def scale_exp(top: float) -> int:
    e = -60
    while e < 60 and top > 448.0 * 2.0 ** e:
        e += 1
    return e


def code(x):
    """float64 [n, heads, D] -> the values that the blocks of each head hold."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[0], BLOCK):
        for h in range(x.shape[1]):
            part = x[b:b + BLOCK, h]
            e = scale_exp(float(part.abs().max()))
            y = part * 2.0 ** -e
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            out[b:b + BLOCK, h] = torch.clamp(torch.round(y / step) * step, -448, 448) * 2.0 ** e
    return out


def norm(x, w, eps):
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return x if w is None else x * w.double()


def rope(x, pos, layer):
    """x: [n, heads, D] float64, pos: [n]."""
    half = layer.rotary_dim // 2
    if half == 0:
        return x
    dist = half if layer.rope_pairing == capi.ROPE_SPLIT_HALF else layer.head_dim // 2
    theta = float(torch.tensor(layer.rope_theta, dtype=torch.float32))
    f = theta ** (-2.0 * torch.arange(half, dtype=torch.float64, device=x.device) / layer.head_dim)
    ang = pos.double()[:, None] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    y = x.clone()
    a, b = x[..., :half], x[..., dist:dist + half]
    y[..., :half] = a * c - b * s
    y[..., dist:dist + half] = b * c + a * s
    return y


def step_rows(layer, q, k, v, qw, kw, pos):
    """The rows of one canvas as they enter the attention: q, k normed, rotated and rounded, v normed where the layer does."""
    at = pos + torch.arange(layer.canvas, device=q.device)
    q = low(rope(norm(q, qw, layer.rms_eps), at, layer))
    if k is None:
        return q, None, None
    k = low(rope(norm(k, kw, layer.rms_eps), at, layer))
    return q, k, low(norm(v, None, layer.rms_eps)) if layer.v_norm else v.double()


def visible(layer, n, n_canvas):
    """[C, n + n_canvas]"""
    C, w, m = layer.canvas, layer.window, layer.mask_mode
    out = torch.zeros(C, n + n_canvas, dtype=torch.bool)
    for i in range(C):
        own = n + i if m in (capi.MASK_WINDOW_PER_ROW, capi.MASK_CAUSAL) else n
        lo = max(0, own - (w - 1)) if w and m != capi.MASK_NONE else 0
        out[i, lo:n] = True
        if m == capi.MASK_CAUSAL:
            out[i, max(n, lo):n + min(i + 1, n_canvas)] = True
        else:
            out[i, n:] = True
    return out


# A bf16 number is the sum of two e4m3 codes down to 2^-10 of the largest of its row (query) or block (canvas K, V); below it
# the second code is off by at most half of e4m3's smallest step, 2^-10 times the scale, and the scale is at most 2 / 448 of
# the largest.
TAIL = 2.0 ** -10 * 2 / 448


def attend(layer, q, keys, values, see):
    """q [C, Hq, D], keys / values [T, Hkv, D], see [C, T].  Returns out, lse, mean of |v| under the weights, and of each row
    the largest sum of |q k| and of what the two-term split leaves of a score, all float64 [C, Hq, ...]."""
    C, Hq, D = q.shape
    g = Hq // keys.shape[1]
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((C, Hq), -math.inf, dtype=torch.float64, device=q.device)
    big = torch.zeros(2, C, Hq, dtype=torch.float64, device=q.device)
    hidden = ~see.to(q.device)
    scale = float(torch.tensor(layer.softmax_scale, dtype=torch.float32))
    if keys.shape[0] == 0:
        return out, lse, spread, big
    for h in range(Hq):
        k, v = keys[:, h // g], values[:, h // g]
        s = (q[:, h] @ k.T) * scale
        big[0, :, h] = ((q[:, h].abs() @ k.abs().T) * scale).amax(1)
        big[1, :, h] = scale * TAIL * (q[:, h].abs().amax(1) * k.abs().sum(1).max() + q[:, h].abs().sum(1) * k.abs().max())
        s[hidden] = -math.inf
        lse[:, h] = torch.logsumexp(s, 1)
        p = torch.nan_to_num(torch.softmax(s, 1))
        out[:, h], spread[:, h] = p @ v, p @ v.abs()
    return out, lse, spread, big


def key_weights(layer, q, keys, see, lse):
    C, Hq, D = q.shape
    g = Hq // keys.shape[1]
    scale = float(torch.tensor(layer.softmax_scale, dtype=torch.float32))
    w = torch.zeros(keys.shape[1], keys.shape[0], dtype=torch.float64, device=q.device)
    hidden = ~see[:, :keys.shape[0]].to(q.device)
    for h in range(Hq):
        p = torch.exp((q[:, h] @ keys[:, h // g].T) * scale - lse[:, h, None].double())
        p[hidden] = 0
        p[torch.isinf(lse[:, h])] = 0
        w[h // g] += p.sum(0)
    return w


def keep(weights, n, n_keep, n_recent):
    """Slots kept of each head: [heads, n_keep]."""
    got = []
    for row in weights[:, :n].tolist():
        rank = sorted(range(n - n_recent), key=lambda t: (-row[t] if row[t] == row[t] else math.inf, t))
        nan_last = [t for t in rank if row[t] == row[t]] + [t for t in range(n - n_recent) if row[t] != row[t]]
        got.append(sorted(nan_last[:n_keep - n_recent]) + list(range(n - n_recent, n)))
    return torch.tensor(got, dtype=torch.int32)


# A bf16 output of the kernels against these sums.  Rounding the output: half a bf16 step, 2^-8 of it.  A weight is the sum of
# an e4m3 and an e5m2 number: 2^-4 of it left by the first, 2^-3 of that by the second, 2^-7, after a rounding to f16, 2^-11.
# Weights below 2^-11 of their row's largest are held to 2^-3 of themselves, 2^-19 of that largest at most: values to which no
# larger weight adds anything can be that far off (the bound leaves it out, no case here has such values).  Sums in fp32: 2^-24 of |p v| for each
# of T keys and two passes, far below.
# Canvas values come as two codes: TAIL of the largest for those far below it.
def out_bound(out, spread, T, canvas_top=0.0):
    return 2.0 ** -8 * out.abs() + (2.0 ** -7 + 2.0 ** -11 + (2 * T + 64) * 2.0 ** -24) * spread + 1.01 * TAIL * canvas_top + 1e-30


# Log-sum-exp: a score is the fp32 sum of 2 D products (q in two terms), 2^-24 of the sum of magnitudes for each at most; the
# exponent x = s c - m is rounded at a magnitude of at most 2^8, 2^-16 in base 2; exp2 and the sums add 2^-22 and
# T 2^-24 relative.
def lse_bound(big, D, T):
    return 2 * D * 2.0 ** -24 * big[0] + big[1] + 2.0 ** -16 + 2.0 ** -22 + T * 2.0 ** -24
