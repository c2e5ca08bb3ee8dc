"""Plain implementations in 64 bits of the token-model operators (embed,
layer_norm, the 8-bit tape, expert_mm), and the error bounds their tests use.

A bound is |out - ref| <= u_T |ref| + k u_P scale: one rounding to the array's
type, and k roundings of the sums' type relative to the sum of magnitudes
`scale` of what was added (the standard bound of a sum of n terms in any order
has k = n; the tensor cores' sums truncate, which doubles it).
"""
import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -8,
        torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.float64: 0.0, torch.bfloat16: 2.0 ** -133,
        torch.float16: 2.0 ** -24}


def par(dt):
    return torch.float64 if dt == torch.float64 else torch.float32


def f64(t):
    return t.detach().cpu().double().numpy()


def assert_close(out, ref, scale, k, name=""):
    """out: tensor; ref, scale: float64 arrays; k: roundings of the sums."""
    o = f64(out).reshape(ref.shape)
    assert np.array_equal(np.isnan(o), np.isnan(ref)), f"{name}: NaN in other places"
    ok = ~np.isnan(ref)
    tol = (UNIT[out.dtype] * 1.001 * np.abs(ref) + TINY[out.dtype] +
           k * UNIT[par(out.dtype)] * np.broadcast_to(scale, ref.shape))
    if out.dtype == torch.float16:      # the largest value before infinity
        assert np.all(np.abs(ref[ok]) < 65000), "test inputs must stay in range"
    bad = ok & ~(np.abs(o - ref) <= tol)
    assert not bad.any(), (f"{name}: {bad.sum()} of {ref.size} off, worst "
                           f"{np.nanmax(np.abs(o - ref) / np.maximum(tol, 1e-300)):.2f} x bound")


# ---- embed -------------------------------------------------------------------
def embed(w, ids, scale, base=0):
    v = ids - base
    y = np.zeros((len(ids), w.shape[1]))
    ok = (v >= 0) & (v < w.shape[0])
    y[ok] = scale * w[v[ok]]
    return y


def embed_b(yb, ids, scale, n_v, base=0):
    """(gradient, sum of magnitudes, positions per row)"""
    wb, mag, cnt = np.zeros((n_v, yb.shape[1])), np.zeros((n_v, yb.shape[1])), np.zeros(n_v)
    for s, i in enumerate(ids):
        if 0 <= i - base < n_v:
            wb[i - base] += scale * yb[s]
            mag[i - base] += abs(scale) * np.abs(yb[s])
            cnt[i - base] += 1
    return wb, mag, cnt


# ---- layer_norm ----------------------------------------------------------------
def layer_norm(x, w, b, eps):
    """y, mean, rstd and the magnitude that y's error is relative to"""
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / np.sqrt((d * d).mean(1) + eps)
    w = np.ones(x.shape[1]) if w is None else w
    b = np.zeros(x.shape[1]) if b is None else b
    mag = rstd[:, None] * (np.abs(x) + np.abs(x).mean(1)[:, None]) * np.abs(w) + np.abs(b)
    return d * rstd[:, None] * w + b, mean, rstd, mag


def layer_norm_b(x, w, yb, mean, rstd):
    """xb, wb, bb and the magnitudes of each"""
    w = np.ones(x.shape[1]) if w is None else w
    r = rstd[:, None]
    h, hm = (x - mean[:, None]) * r, (np.abs(x) + np.abs(mean)[:, None]) * r
    g = yb * w
    xb = r * (g - g.mean(1)[:, None] - h * (g * h).mean(1)[:, None])
    ag = np.abs(g)
    mx = r * (ag + ag.mean(1)[:, None] + hm * (ag * hm).mean(1)[:, None])
    return (xb, (yb * h).sum(0), yb.sum(0)), (mx, (np.abs(yb) * hm).sum(0), np.abs(yb).sum(0))


# ---- 8-bit tape ------------------------------------------------------------------
def tape8(x):
    """codes and scale bytes of a float64 array holding the values of x"""
    n_s, n_d = x.shape
    n_g = -(-n_d // 32)
    q, e = np.zeros((n_s, n_d), np.int8), np.zeros((n_s, n_g), np.uint8)
    for s in range(n_s):
        for g in range(n_g):
            v = x[s, 32 * g:32 * g + 32]
            if not np.all(np.isfinite(v)):
                e[s, g] = 255
                continue
            top = np.abs(v).max()
            k = math.frexp(top)[1] - 1 if top > 0 else -1000
            p = max(k - 6, -126)
            e[s, g] = p + 127
            q[s, 32 * g:32 * g + 32] = np.clip(np.rint(np.ldexp(v, -p)), -127, 127)
    return q, e


def tape8_values(q, e):
    n_s, n_d = q.shape
    p = np.repeat(e.astype(np.int64) - 127, 32, axis=1)[:, :n_d]
    v = np.ldexp(q.astype(np.float64), p)
    v[np.repeat(e == 255, 32, axis=1)[:, :n_d]] = np.nan
    return v


_erf = np.vectorize(math.erf)


def act(name, x):
    if name == "relu":
        return np.maximum(x, 0)
    if name == "tanh":
        return np.tanh(x)
    if name == "silu":
        return x / (1 + np.exp(-x))
    return 0.5 * x * (1 + _erf(x / math.sqrt(2)))


def act_slope(name, x):
    if name == "relu":
        return 0.5 * (1 + np.sign(x))
    if name == "tanh":
        return 1 / np.cosh(x) ** 2
    if name == "silu":
        p = 1 / (1 + np.exp(-x))
        return p * (1 + x * (1 - p))
    return 0.5 * (1 + _erf(x / math.sqrt(2))) + x * np.exp(-x * x / 2) / math.sqrt(2 * math.pi)


# ---- expert_mm ---------------------------------------------------------------------
def expert_mm(x, w, off):
    y, mag = np.zeros((len(x), w.shape[2])), np.zeros((len(x), w.shape[2]))
    for e in range(len(w)):
        r = slice(off[e], off[e + 1])
        y[r], mag[r] = x[r] @ w[e], np.abs(x[r]) @ np.abs(w[e])
    return y, mag


def expert_mm_b(x, w, yb, off):
    xb, wb = np.zeros_like(x), np.zeros_like(w)
    mx, mw = np.zeros_like(x), np.zeros_like(w)
    for e in range(len(w)):
        r = slice(off[e], off[e + 1])
        xb[r], mx[r] = yb[r] @ w[e].T, np.abs(yb[r]) @ np.abs(w[e]).T
        wb[e], mw[e] = x[r].T @ yb[r], np.abs(x[r]).T @ np.abs(yb[r])
    return xb, wb, mx, mw
