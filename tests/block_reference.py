"""The block operators (include/eg2_hip.h) from their definitions in 64 bits,
on the host, and how far a right result may be off: used by the tests of
eg2_hip_linear, _linear_gated, _heads_norm_rope and _window_attention.

Bounds. A sum of n products in 32 bits is off by at most n u times the sum of
the products' magnitudes, u = 2^-23 (half that where every addition rounds to
nearest; the matrix units' own additions are not documented to). A rounding to a type
is off by at most half a step, eps / 2 of the value, or half its smallest step."""
import math

import numpy as np
import torch

U = 2.0 ** -23
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rounding(value, dtype):
    """At most this far does rounding `value` to dtype take it."""
    info = torch.finfo(dtype)
    return np.abs(value) * (info.eps / 2) + info.smallest_normal * info.eps / 2


def activation(z, act):
    if act == "gelu":
        return z / (1.0 + np.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z / (1.0 + np.exp(-z))
    return np.maximum(z, 0.0) if act == "relu" else z


def quantize(w):
    """Q8_0 blocks of the rows of w [m, k] as uint8 [m, 34 k / 32], and the values they stand for."""
    m, k = w.shape
    b = w.reshape(m, k // 32, 32).astype(np.float32)
    d = (np.abs(b).max(2) / 127.0).astype(np.float16)
    q = np.rint(b / np.maximum(d.astype(np.float32), 1e-20)[:, :, None]).clip(-127, 127).astype(np.int8)
    raw = np.concatenate([d[:, :, None].view(np.uint8), q.view(np.uint8)], 2)
    return raw.reshape(m, k // 32 * 34).copy(), (q.astype(np.float64) * d.astype(np.float64)[:, :, None]).reshape(m, k)


def _product(x, w, bias):
    """(x w^T + bias, how far its 32-bit evaluation may be off)."""
    z, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        z, mag = z + bias, mag + np.abs(bias)
    # k products, their sum split and joined and the bias; a Q8_0 block's scale is one more rounding
    return z, (x.shape[1] + 8) * U * mag


def _activated(z, off, act):
    """An activation's slope is at most 1.13. z / (1 + exp(-t)) with t off by 4 u |t|: of the result at most
    |t| 4 u below 0, where it is |z| exp(t) and |t| exp(t) <= 0.37, and less above; exp, the sum and the quotient 4 u more."""
    return activation(z, act), (off if act == "none" else 1.13 * off + (0.0 if act == "relu" else 8 * U * np.abs(z)))


def linear(x, w, bias, act, residual, dtype):
    z, off = _product(x, w, bias)
    y, off = _activated(z, off, act)
    if residual is not None:
        y = y + residual
    off = off + U * np.abs(y)
    return y, off + rounding(np.abs(y) + off, dtype)


def linear_gated(x, gate, up, gate_bias, up_bias, act, dtype):
    g, g_off = _product(x, gate, gate_bias)
    u, u_off = _product(x, up, up_bias)
    a, a_off = _activated(g, g_off, act)
    y = a * u
    off = np.abs(a) * u_off + np.abs(u) * a_off + a_off * u_off + U * np.abs(y)
    return y, off + rounding(np.abs(y) + off, dtype)


def heads_norm_rope(x, w, table, pos, eps, scale, dtype):
    """x [rows, heads, d]. The norm: d + 4 roundings in the sum, halved by the root, and one each of the
    products with 1/rms, w, the angle (two products and a sum) and the scale."""
    d = x.shape[2]
    inv = 1.0 / np.sqrt((x * x).mean(2, keepdims=True) + eps)
    u = x * inv * (1.0 if w is None else w)
    mag = np.abs(u)
    if table is not None:
        half = table.shape[1] // 2
        c, s = (t[:, None, :] for t in (table[pos][:, :half], table[pos][:, half:]))
        a, b, rest = u[..., :half], u[..., half:2 * half], u[..., 2 * half:]
        mag = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c), np.abs(rest)], 2)
        u = np.concatenate([a * c - b * s, a * s + b * c, rest], 2)
    u, off = u * scale, ((d + 4) / 2 + 8) * U * mag * abs(scale)
    return u, off + rounding(np.abs(u) + off, dtype)


def visible(nq, nk, left, right, sinks):
    """[nq, nk] truth values: the keys that each query sees."""
    p = np.arange(nk - nq, nk)[:, None]
    s = np.arange(nk)[None]
    seen = np.ones((nq, nk), bool)
    if right >= 0:
        seen &= s <= p + right
    if left >= 0:
        seen &= (s >= p - left) | (s < sinks)
    return seen


def window_attention(q, k, v, q_offsets, k_offsets, scale, left, right, sinks, k_lengths, dtype):
    """(out, how far it may be off): rows in no sequence are NaN with a bound of 0."""
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    out, off = np.full(q.shape, np.nan), np.zeros(q.shape)
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2  # the weights' own rounding
    for b in range(len(q_offsets) - 1):
        q0, nq, k0 = q_offsets[b], q_offsets[b + 1] - q_offsets[b], k_offsets[b]
        nk = k_offsets[b + 1] - k0 if k_lengths is None else k_lengths[b]
        seen = visible(nq, nk, left, right, sinks)
        for i in range(nq):
            at = k0 + np.flatnonzero(seen[i])
            for h in range(heads):
                if not len(at):
                    out[q0 + i, h] = 0.0
                    continue
                qq, kk, vv = q[q0 + i, h], k[at, h // group], v[at, h // group]
                s = (kk @ qq) * scale
                # The score: d products; the scale, the subtraction and the argument of exp2 (each below
                # twice the largest score), evaluated to a few u.
                s_off = ((d + 4) * U * (np.abs(kk) @ np.abs(qq)) * abs(scale)).max() + 8 * U * np.abs(s).max() + 8 * U
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[q0 + i, h] = p @ vv
                mag = p @ np.abs(vv)
                e = mag * (2 * math.expm1(2 * s_off) + 2 * (len(at) + 8) * U + 2 * eps)
                # a weight below the type's normal numbers loses its last bits: of each at most half the smallest step
                if dtype == torch.float16:
                    e = e + 2.0 ** -25 * np.abs(vv).sum(0) * 2
                off[q0 + i, h] = e + rounding(np.abs(out[q0 + i, h]) + e, dtype)
    return out, off
