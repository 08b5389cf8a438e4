"""The 4-bit cache and its attention in plain numpy, 64 bits, written from the format's description alone."""
import numpy as np


def quantise(x):
    """x [..., hd] fp32 -> codes [..., hd] uint8, d, m [..., hd/64] fp16."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 64)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    with np.errstate(over="ignore"):
        m = g.min(-1).astype(np.float16)
    bad |= np.isinf(m)
    m = np.where(bad, np.float16(0), m)
    d = np.maximum(0.0, (g.max(-1) - m.astype(np.float64)) / 15.0)
    d = np.where(bad, 0.0, d).astype(np.float16)
    dd = np.where(d > 0, d.astype(np.float64), 1.0)[..., None]
    q = np.where(d[..., None] > 0, np.clip(np.rint((g - m.astype(np.float64)[..., None]) / dd), 0, 15), 0)
    q = np.where(bad[..., None], 0, q).astype(np.uint8)
    d, m = np.where(bad, np.float16(np.nan), d), np.where(bad, np.float16(np.nan), m)
    return q.reshape(x.shape), d, m


def values(codes, d, m):
    g = codes.reshape(*codes.shape[:-1], -1, 64).astype(np.float64)
    return (m.astype(np.float64)[..., None] + d.astype(np.float64)[..., None] * g).reshape(codes.shape)


def k_byte(hd, s, D):
    return s * (hd // 2) + 4 * ((D % 32 // 8) * (hd // 32) + D // 32) + D % 8 // 2


def v_byte(hd, s, D):
    p = D // 2
    j, r, h, t, u = p // 8, p % 8, s // 8, s % 8 // 2, s % 2
    return 8 * hd + (j // 4) * 512 + (4 * r + t) * 16 + (j % 4) * 4 + 2 * u + h


def write_rows(cache, hd, pos, k, v):
    """Quantise k, v [n][heads][hd] into cache [heads][blocks][18 hd] (uint8 array) at positions pos [n]."""
    even = np.arange(0, hd, 2)
    for which, x in ((0, k), (1, v)):
        q, d, m = quantise(np.ascontiguousarray(np.transpose(x, (1, 0, 2))))
        at = 16 * hd + which * hd
        scale = np.stack((d, m), -1).astype(np.float16).view(np.uint8).reshape(*d.shape[:2], -1)
        for i, p in enumerate(pos):
            s = p % 16
            cache[:, p // 16, (v_byte if which else k_byte)(hd, s, even)] = q[:, i, 0::2] | (q[:, i, 1::2] << 4)
            n = scale.shape[-1]
            cache[:, p // 16, at + s * n: at + (s + 1) * n] = scale[:, i]


def read_rows(cache, hd, n):
    """float64 K, V [heads][n][hd] of the first n positions."""
    out = []
    D = np.arange(hd)
    for which in (0, 1):
        rows = []
        at = 16 * hd + which * hd
        for p in range(n):
            s = p % 16
            b = cache[:, p // 16, (v_byte if which else k_byte)(hd, s, D - D % 2)]
            q = np.where(D % 2, b >> 4, b & 15)
            sc = np.ascontiguousarray(cache[:, p // 16, at + s * hd // 16: at + (s + 1) * hd // 16]).view(np.float16).reshape(cache.shape[0], -1, 2)
            rows.append(values(q, sc[..., 0], sc[..., 1]))
        out.append(np.stack(rows, 1) if rows else np.zeros((cache.shape[0], 0, hd)))
    return out


def rope(x, pos, rope_type, n_rot, theta, ff=None):
    """x [n][heads][hd] at positions pos [n]; the angle is the fp32 product of position and frequency."""
    out = np.asarray(x, np.float64).copy()
    half = n_rot // 2
    e = (np.float32(-2.0) * np.arange(half, dtype=np.float32)) / np.float32(n_rot)
    f = np.power(np.float64(np.float32(theta)), e.astype(np.float64)).astype(np.float32)
    if ff is not None:
        f = (f / np.asarray(ff, np.float32)).astype(np.float32)
    ang = (np.asarray(pos, np.float32)[:, None] * f).astype(np.float64)[:, None]
    i0 = np.arange(half) if rope_type == 1 else 2 * np.arange(half)
    i1 = i0 + (half if rope_type == 1 else 1)
    a, b = out[..., i0].copy(), out[..., i1].copy()
    out[..., i0], out[..., i1] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
    return out


def attend(q, K, V, first, scale):
    """q [n][n_head][hd] at positions first + i, K, V [n_kv][rows][hd] -> out, and the largest sum_i |q_i k_i| of any score."""
    n, n_head, hd = q.shape
    group = n_head // K.shape[0]
    out, most = np.zeros((n, n_head, hd)), 0.0
    for h in range(n_head):
        k, v = K[h // group], V[h // group]
        for i in range(n):
            L = first + i + 1
            s = (k[:L] @ q[i, h]) * scale
            p = np.exp(s - s.max())
            out[i, h] = (p @ v[:L]) / p.sum()
        most = max(most, float((np.abs(q[:, h]) @ np.abs(k).T).max()))
    return out, most
