"""The KV cache and the attention over it, restated plainly in 64 bits (numpy), from the definitions of include/ktmoe.h:
what the GPU tests compare with, integer for integer."""

from __future__ import annotations

import math

import numpy as np

C0, C1, C2, C3 = 32512.0, 127 * 45435 / 256, 127 * 15874 / 256, 127 * 3605 / 256


def rn24(x):
    """Rounded to 24 significant bits, ties to even (binary32), in float64."""
    with np.errstate(over="ignore", under="ignore"):
        return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def value(scale):
    mant, shift = int(scale[0]), int(np.int32(np.int64(scale[1]) & 0xFFFFFFFF))
    return math.ldexp(mant, -shift) if mant > 0 else 0.0


def rotate(x, table_row, interleaved):
    """x: int codes [..., dim]; table_row: [half][2] or None. The codes after the rotation (int64) and the factor of
    the scale."""
    y = np.asarray(x).astype(np.int64)
    if table_row is None:
        return y, 1.0
    half = table_row.shape[0]
    out = y * (1 << 30)
    ia = 2 * np.arange(half) if interleaved else np.arange(half)
    ib = ia + 1 if interleaved else ia + half
    c, s = table_row[:, 0].astype(np.int64), table_row[:, 1].astype(np.int64)
    out[..., ia] = y[..., ia] * c - y[..., ib] * s
    out[..., ib] = y[..., ib] * c + y[..., ia] * s
    return out, 2.0 ** -30


def quantise_row(y, s):
    """A cached row: (int8 codes, sigma)."""
    top = float(max(abs(int(v)) for v in y))
    t = min(max(top * s / 127.0, 2.0 ** -64), 2.0 ** 63)
    m, e = math.frexp(t)
    sigma = math.ldexp(math.ceil(m * 256), e - 8)
    codes = np.rint(y.astype(np.float64) * (s / sigma))
    return np.clip(codes, -127, 127).astype(np.int8), sigma


def rows_of(begin, kv_len):
    """(row, sequence, position) of every new token."""
    for b in range(len(kv_len)):
        for t in range(begin[b], begin[b + 1]):
            yield t, b, int(kv_len[b]) - (begin[b + 1] - t)


def append(k, v, scale, begin, kv_len, write, table=None, interleaved=False, v_scale=None):
    """Calls write(which, sequence, position, head, codes, sigma) for each new row; k, v: [rows][heads][dim]; scale (and
    v_scale, when the values have their own): [rows][2] or [2]."""
    v_scale = scale if v_scale is None else v_scale
    for t, b, pos in rows_of(begin, kv_len):
        if pos < 0:
            continue
        s = value(scale[t] if np.ndim(scale) == 2 else scale)
        for h in range(k.shape[1]):
            y, f = rotate(k[t, h], None if table is None else table[pos], interleaved)
            write("k", b, pos, h, *quantise_row(y, s * f))
            write("v", b, pos, h, *quantise_row(v[t, h].astype(np.int64), value(v_scale[t] if np.ndim(v_scale) == 2 else v_scale)))


def weights(dots, sigma_k, theta):
    """w_j of the visible keys (float64, exact)."""
    x = rn24(dots * sigma_k)
    d = rn24(x.max() - x)
    z = np.minimum(np.rint(d * theta * 1024), 32 * 1024)
    n = np.rint(z / 1024)
    r = n - z / 1024
    e = rn24(rn24(rn24(C3 * r + C2) * r + C1) * r + C0)
    return np.ldexp(e, -n.astype(np.int64))


def attention(q, scale, begin, kv_len, keys, out, out_scale, softmax_scale, window=0, sinks=0, table=None,
              interleaved=False):
    """keys(sequence, head) -> (k codes [n][dim], sigma_k [n], v codes, sigma_v) of a sequence's positions; q: [rows]
    [heads][dim]; fills out [rows][heads][dim] and out_scale [rows][kv heads][2] (mant, shift)."""
    n_kv = out_scale.shape[1]
    group = q.shape[1] // n_kv
    soft = softmax_scale * 1.4426950408889634
    for t, b, pos in rows_of(begin, kv_len):
        j = np.arange(pos + 1)
        if window:
            j = j[(j > pos - window) | (j < sinks)]
        out[t], out_scale[t] = 0, 0
        if pos < 0 or j.size == 0:
            continue
        s = value(scale[t] if np.ndim(scale) == 2 else scale)
        y, f = rotate(q[t], None if table is None else table[pos], interleaved)
        for h in range(q.shape[1]):
            k8, sk, v8, sv = (a[j] for a in keys(b, h // group))
            top = float(max(abs(int(c)) for c in y[h]))
            if top:
                q8 = np.rint(y[h].astype(np.float64) * (127.0 / top))
                theta = float(rn24(min(top * (s * f) / 127.0 * soft, 2.0 ** 60)))
            else:
                q8, theta = np.zeros(y.shape[1]), 0.0
            w = weights(k8.astype(np.float64) @ q8, sk, theta)
            m, e = np.frexp(sv.max())
            e = int(e) - (1 if m == 0.5 else 0)
            total = int(np.rint(w).sum())
            num = np.rint(w * np.ldexp(sv, -e)) @ v8.astype(np.float64)
            out[t, h] = np.rint(num * (2097152.0 / total)).astype(np.int32)
            out_scale[t, h // group] = (1, 21 - e)
