"""Serving many requests: rotary positions, a KV cache in pages and its attention, and low-rank adapters, from their definitions
in numpy and 64 bits (include/lowbit_decode_hip.h).  Test infrastructure only."""
import numpy as np


def turned(x, position, frequencies, pairs='half', scale=1.0, back=False):
    """x [.., seq, heads, D] at positions [.., seq]."""
    x = np.asarray(x, np.float64)
    n = len(frequencies)
    angle = (np.asarray(position, np.float64)[..., None] * np.asarray(frequencies, np.float64))[..., None, :]
    c, s = scale * np.cos(angle), scale * np.sin(angle) * (-1.0 if back else 1.0)
    y = x.copy()
    first = (slice(0, n), slice(n, 2 * n)) if pairs == 'half' else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., first[0]], x[..., first[1]]
    y[..., first[0]], y[..., first[1]] = a * c - b * s, b * c + a * s
    return y


def partner_sizes(x, n, pairs='half'):
    """|a| + |b| of each value's pair (0 where a value does not turn): what the errors of a rotation are parts of."""
    x = np.abs(np.asarray(x, np.float64))
    y = np.zeros_like(x)
    first = (slice(0, n), slice(n, 2 * n)) if pairs == 'half' else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    y[..., first[0]] = y[..., first[1]] = x[..., first[0]] + x[..., first[1]]
    return y


def values_by_slot(values):
    """[.., page / 16, D, 16] as [.., page, D]."""
    *lead, chunks, dim, slots = values.shape
    return np.moveaxis(values, -1, -2).reshape(*lead, chunks * slots, dim)


def held(keys, values, pages, length):
    """Keys and values [kv_heads, length, D] in 64 bits of a sequence with these pages."""
    k = np.concatenate([keys[p] for p in pages], 1)[:, :length].astype(np.float64)
    v = np.concatenate([values_by_slot(values[p]) for p in pages], 1)[:, :length].astype(np.float64)
    return k, v


def attention(q, k, v, scale):
    """One token: q [heads, D] over k, v [kv_heads, n, D].  Returns the output, the weighted mean of |v|, and the largest sum of
    |q k| scale of a score, [heads, D], [heads, D], [heads]."""
    q = np.asarray(q, np.float64)
    group = len(q) // len(k)
    out, mean, size = np.empty_like(q), np.empty_like(q), np.empty(len(q))
    for h in range(len(q)):
        s = k[h // group] @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mean[h] = p @ v[h // group], p @ np.abs(v[h // group])
        size[h] = (np.abs(k[h // group]) @ np.abs(q[h])).max() * abs(scale)
    return out, mean, size


def adapters(y, x, down, up, index, scales=None):
    """y + s (x A^T) B^T, row by row.  Returns the output and the sums of magnitudes that errors are parts of: those of the
    products with A (carried through |B|), and of the largest |z| of the row."""
    y, x = np.asarray(y, np.float64), np.asarray(x, np.float64)
    out, products, tops = y.copy(), np.zeros_like(y), np.zeros_like(y)
    for m, a in enumerate(index):
        if a == -1:
            continue
        if not 0 <= a < len(down):
            out[m] = np.nan
            continue
        s = 1.0 if scales is None else float(scales[a])
        A, B = np.asarray(down[a], np.float64), np.asarray(up[a], np.float64)
        z = A @ x[m]
        out[m] += s * (B @ z)
        products[m] = abs(s) * (np.abs(B) @ (np.abs(A) @ np.abs(x[m])))
        tops[m] = abs(s) * np.abs(B).sum(1) * np.abs(z).max()
    return out, products, tops
