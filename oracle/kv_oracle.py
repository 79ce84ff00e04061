"""The 8-bit KV cache in 64 bits (include/lowbit_decode_hip.h, lb_kv_cache): what a cache of given rows holds, and
attention over it.  numpy only; written from the definitions, row by row where that is the definition."""
import numpy as np

BLOCK = 64
LIMIT = {'int8': 127.0, 'fp8': 448.0}


def e4m3(x):
    """x rounded to the nearest e4m3fn value (ties to even), |x| <= 448: 4 significant bits, steps of 2^-9 at the least."""
    x = np.asarray(x, dtype=np.float64)
    _, exponent = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(exponent - 4, -9))
    return np.rint(x / step) * step


def e4m3_bits(x):
    """Bytes of e4m3fn values."""
    x = np.asarray(x, dtype=np.float64)
    sign = np.where(np.signbit(x), 0x80, 0)
    mag = np.abs(x)
    _, exponent = np.frexp(mag)
    exponent = np.maximum(exponent - 1, -6)
    mantissa = np.rint(np.ldexp(mag, 3 - exponent)).astype(np.int64)   # 8..15, below 8 where subnormal
    return (sign | np.where(mantissa >= 8, (exponent + 7) * 8 + mantissa - 8, mantissa)).astype(np.uint8)


def quantise(block, format):
    """(values of the codes float64, scale float32) of one block [64, D] of fp16 rows."""
    x = np.asarray(block, dtype=np.float64)
    if not np.isfinite(x).all():
        return np.zeros_like(x), np.float32(np.nan)
    top = np.abs(x).max()
    scale = np.float32(top) / np.float32(LIMIT[format])
    if top == 0:
        return np.zeros_like(x), scale
    unit = x * LIMIT[format] / top   # exact ties stay exact: x and top have 11 bits, the quotient is rounded once
    return (np.rint(unit) + 0.0 if format == 'int8' else e4m3(unit)), scale   # (an int8 code has no negative zero)


def poison(k, v):
    """Rows [n, D] as they are held: a key of NaNs where the key or the value is not finite."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    k = np.array(k, copy=True)
    k[bad] = np.nan
    return k, v


def held(rows, format):
    """float64 values that a cache of these fp16 rows [n, D] holds: whole blocks as code * scale, the others as they are."""
    out = np.array(rows, dtype=np.float64)
    for at in range(0, len(rows) // BLOCK * BLOCK, BLOCK):
        codes, scale = quantise(rows[at:at + BLOCK], format)
        with np.errstate(invalid='ignore'):
            out[at:at + BLOCK] = codes * np.float64(scale)
    return out


def read(rows, format):
    """fp16 values that reading such a cache gives: the fp32 product of code and scale (8 and 24 bits: rounded once there)
    rounded to fp16."""
    out = np.array(rows, dtype=np.float16)
    for at in range(0, len(rows) // BLOCK * BLOCK, BLOCK):
        codes, scale = quantise(rows[at:at + BLOCK], format)
        with np.errstate(invalid='ignore'):
            out[at:at + BLOCK] = (codes.astype(np.float32) * scale).astype(np.float16)
    return out


def rotate(t, cos, sin):
    """RoPE of fp16 rows [n, .., D] with the tables' rows [n, .., D], at the framework's rounding points."""
    t, half = np.asarray(t, dtype=np.float16), t.shape[-1] // 2
    turned = np.concatenate((-t[..., half:], t[..., :half]), -1)
    with np.errstate(over='ignore', invalid='ignore'):
        return ((t.astype(np.float32) * cos.astype(np.float32)).astype(np.float16).astype(np.float32)
                + (turned.astype(np.float32) * sin.astype(np.float32)).astype(np.float16).astype(np.float32)).astype(np.float16)


def attend(q, k, v, first, scale):
    """(out, weight of |v|, largest |q||k| sum) of query rows q [s, D] at slots first .. over values k, v [n, D]."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    out, weight, reach = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros(len(q))
    for i in range(len(q)):
        seen = first + i + 1
        with np.errstate(invalid='ignore', over='ignore'):
            t = (k[:seen] @ q[i]) * scale
            p = np.exp(t - t.max())
            p /= p.sum()
            out[i] = p @ v[:seen]
            weight[i] = p @ np.abs(v[:seen])
            reach[i] = (np.abs(k[:seen]) @ np.abs(q[i])).max() * scale
    return out, weight, reach


def place(slot):
    """Where a slot of a block lies in a value row."""
    return 16 * (slot % 16 // 4) + 4 * (slot // 16) + slot % 4
