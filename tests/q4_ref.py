"""Float64 formulas of the rotary plans and of the 4-bit cache (include/pi_attn.h), in numpy, and the
error bounds that the kernels' roundings allow."""
import numpy as np

GROUP = 32


def rotate(x, pos, freqs, m, layout):
    """x [n, heads, D] float64 at positions [n]."""
    half = len(freqs)
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = m * np.cos(a), m * np.sin(a)
    y = np.array(x, np.float64)
    i0, i1 = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if layout == "pairs" else (slice(0, half), slice(half, 2 * half))
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def rms(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)


def scale_of(m):
    """-m / 8 on the format's grid."""
    r = -np.asarray(m, np.float64) / 8
    e = np.floor(np.log2(np.maximum(np.abs(r), 2.0 ** -14)))
    step = np.maximum(np.exp2(e - 6), 2.0 ** -20)
    return np.clip(np.rint(r / step) * step, -904.0, 904.0)


def quantise(x):
    """x [..., D] float64 -> (codes [..., D], scales [..., D / 32])."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    clean = np.clip(np.nan_to_num(g, nan=0.0, posinf=1e300, neginf=-1e300), -1e300, 1e300)
    hi, lo = clean.max(-1), clean.min(-1)
    s = scale_of(np.where(hi >= -lo, hi, lo))
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        t = np.where(s[..., None] == 0, 0.0, clean / s[..., None])
    c = np.clip(np.rint(t), -8, 7) + 8
    return c.reshape(x.shape).astype(np.int64), s


def values(codes, s):
    c = np.asarray(codes, np.float64) - 8
    return (c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP) * np.asarray(s, np.float64)[..., None]).reshape(c.shape)


def unpack(packed):
    """[..., D / 2] bytes -> [..., D] codes, even channel low."""
    p = np.asarray(packed).astype(np.int64)
    return np.stack((p & 15, p >> 4), -1).reshape(*p.shape[:-1], 2 * p.shape[-1])


def pack(codes):
    c = np.asarray(codes).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def head_map(hq, hkv, mode):
    """KV head of each query head (0: modulo, 1: grouped)."""
    return [h % hkv if mode == 0 else h // (hq // hkv) for h in range(hq)]


def attend(q, k, v, pos, kv_of, scale, gate=None, bad=None):
    """q [n, Hq, D], k / v [T, Hkv, D] float64; row i sees keys 0 .. pos[i] that are not `bad` [T]."""
    n, hq, d = q.shape
    out = np.zeros((n, hq, d))
    keys = np.arange(k.shape[0])
    for i in range(n):
        seen = keys <= pos[i]
        if bad is not None:
            seen &= ~bad
        if not seen.any():
            continue
        for h in range(hq):
            s = (k[seen, kv_of[h]] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            out[i, h] = (p / p.sum()) @ v[seen, kv_of[h]]
    if gate is not None:
        out = out / (1 + np.exp(-gate))
    return out


EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def attend_tol(q, k, v, ref, scale, dtype):
    """Largest error of attend()'s rows by the kernels' roundings.

    A score is a sum of D products: f32 accumulation D 2^-24 of sum |q k|, q held in 22 bits for f32 rows (2^-22;
    exact for 16-bit rows); a score error e changes a weight by a factor 2^(e log2 e), and all weights together the
    output by at most 2 e max|v|.  exp2 and the f32 sums add 2^-20, P in 16 bits 2^-11 (f32 rows: 2^-22).
    Last the output's own rounding."""
    if not k.size:
        return np.zeros_like(ref)
    a = np.abs(q).max(-1).max() * np.abs(k).sum(-1).max() * abs(scale)
    e = a * (q.shape[-1] * 2.0 ** -24 + 2.0 ** -22)
    vm = np.abs(v).max()
    p = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    return vm * (2 * e + 2.0 ** -20 + p) + np.abs(ref) * EPS[dtype] + 2.0 ** -24
