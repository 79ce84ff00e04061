"""lb_kv_attention at scores far from zero, and with many small probabilities: scores of 2^12 to 2^40 (in units of log2), where
one step of fp32 is more than a score's distance from the maximum that still counts, equal and evenly rising scores of that
size, and thousands of slots of 2^-25 of the largest probability.

Bounds are derived at each test; half = 2^-11 is half a step of fp16.
"""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import kv_oracle as ko
from test_gpu_kv import check_attention, dev, fresh, ints, rows_of

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11
LOG2E = np.float32(1.44269504088896340736)
# Query rows of a KV head: 2 and 24 (16 and 32 rows a workgroup, slots split over its waves), 140 (tiles of 128).
SEQS = [1, 12, 70]
KINDS = [('int8', 64), ('fp8', 64), ('int8', 128), ('fp8', 128)]


def scale_for(factor):
    """A score scale that times log2(e) is the power of two `factor` in fp32."""
    at = np.float32(factor / 1.44269504088896340736)
    for step in range(-4, 5):
        scale = at
        for _ in range(abs(step)):
            scale = np.nextafter(scale, np.float32(np.inf if step > 0 else 0))
        if np.float32(scale * LOG2E) == np.float32(factor):
            return float(scale)
    raise AssertionError(factor)


def held_by(device, format, k, v, capacity):
    """A cache of rows k, v [batch, n, kv_heads, D], NaN wherever nothing is held."""
    batch, n, kv_heads, dim = k.shape
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints([n] * batch, device))
    return cache


@pytest.mark.parametrize('power', [12, 20, 24, 25, 26, 27, 28, 30, 40])
@pytest.mark.parametrize('seq', SEQS)
@pytest.mark.parametrize('format,dim', KINDS)
def test_one_score_far_above_the_others(device, format, dim, seq, power):
    """Scores of both signs up to 2^power: each row's output is the value of its largest score.

    Where the largest score is more than 40 (in log2) and twice the error of fp32 scores ahead of the next, the others have
    n 2^-40 together, and what is left is fp32 products (six of 2^-24 at the most) and the output's rounding."""
    announce('kv large scores', format, dim, seq, power)
    clear_scores(device, format, dim, seq, power, 500)


@pytest.mark.parametrize('power', [12, 27, 40])
@pytest.mark.parametrize('format,dim', KINDS)
def test_one_score_far_above_the_others_in_parts(device, format, dim, power):
    """The same in tiles whose slots are taken in several parts (of eight blocks at the least): the parts' maxima meet."""
    announce('kv large scores in parts', format, dim, power)
    clear_scores(device, format, dim, 70, power, 2100)


def clear_scores(device, format, dim, seq, power, n):
    heads, kv_heads, batch = 2, 1, 3
    k, v = rows_of(200, batch, n, kv_heads, dim, spread=200), rows_of(201, batch, n, kv_heads, dim)
    q = rows_of(202, batch, seq, heads, dim, spread=200)
    k[1], q[1] = -np.abs(k[1]), np.abs(q[1])            # all scores below zero
    k[2, ::2] *= np.float16(0.01)                       # rows and blocks of very different sizes
    q[2, ::2] *= np.float16(0.03)
    first = n - seq
    held = [[ko.held(t[b, :, 0], format) for t in (k, v)] for b in range(batch)]
    dots = [np.einsum('shd,nd->shn', q[b].astype(np.float64), held[b][0]) for b in range(batch)]
    scale = float(np.float32(2.0 ** power * 0.9 / max(np.abs(d).max() for d in dots) / 1.4426950408889634))
    assert 0 < scale <= 65536
    cache = held_by(device, format, k, v, (n + 63) // 64 * 64)
    got = lb.kv_attention(dev(q, device), cache, ints([first] * batch, device), scale=scale).float().cpu().numpy().astype(np.float64)
    clear = 0
    for b in range(batch):
        reach = np.einsum('shd,nd->shn', np.abs(q[b]).astype(np.float64), np.abs(held[b][0])).max(-1) * scale * 1.4427
        for i in range(seq):
            for h in range(heads):
                t = dots[b][i, h, :first + i + 1] * scale * 1.4426950408889634
                order = np.argsort(t)
                if t[order[-1]] - t[order[-2]] <= 40 + 4 * (dim + 8) * 2.0 ** -24 * reach[i, h]:
                    continue
                clear += 1
                want = held[b][1][order[-1]]
                limit = np.abs(want) * (HALF + 6 * 2.0 ** -24) + 2.0 ** -25 + n * 2.0 ** -40 * np.abs(v[b]).max()
                off = np.abs(got[b, i, h] - want)
                assert (off <= limit).all(), (b, i, h, t[order[-1]], got[b, i, h][:4], want[:4])
    assert clear >= (0.6 if power >= 20 else 0.3) * batch * seq * heads, clear


@pytest.mark.parametrize('factor', [2.0 ** p for p in (-20, -8, -3, 0, 1, 2, 3, 4, 5, 7, 14)])
@pytest.mark.parametrize('seq', SEQS)
@pytest.mark.parametrize('format,dim', KINDS)
def test_equal_scores_however_large(device, format, dim, seq, factor):
    """Keys that are all one row: every probability is the same, whatever the blocks' scales and the score (up to 2^36).

    Keys of +- 127 c or 448 c, c a power of two, and queries of whole numbers: codes, fp16 rows and their fp32 scores are exact
    and the same.  With A = mean |v|: a probability's rounding to fp16 in the sum with V and in the total (2 half A), ratios
    of scales and sums in fp32 (2^-18 A), up to scores of 2^10 the sum of a maximum and an exponent (2^-13 A), the output's
    rounding."""
    announce('kv equal scores', format, dim, seq, factor)
    heads, kv_heads, n, batch = 2, 1, 460, 2
    rng = np.random.default_rng(210)
    unit = 127.0 if format == 'int8' else 448.0
    sign = rng.choice([-1.0, 1.0], dim)
    k = np.broadcast_to((sign * unit * 0.25).astype(np.float16), (batch, n, kv_heads, dim)).copy()
    k[1] *= 2
    v = rows_of(211, batch, n, kv_heads, dim).astype(np.float64)
    v *= np.exp2(rng.uniform(-6, 6, (n + 63) // 64))[np.arange(n) // 64][None, :, None, None]
    v = v.astype(np.float16)
    q = (sign * rng.integers(1, 300, (batch, seq, heads, dim))).astype(np.float16)
    q[:, ::3] *= -1                                     # (largest scores far below zero as well)
    scale = scale_for(factor)
    cache = held_by(device, format, k, v, 512)
    first = n - seq
    got = lb.kv_attention(dev(q, device), cache, ints([first] * batch, device), scale=scale).float().cpu().numpy().astype(np.float64)
    for b in range(batch):
        hv = ko.held(v[b, :, 0], format)
        for i in range(seq):
            seen = hv[:first + i + 1]
            want, weight = seen.mean(0), np.abs(seen).mean(0)
            limit = weight * (2 * HALF + 2.0 ** -18 + 2.0 ** -13) + HALF * np.abs(want) + 2.0 ** -25
            for h in range(heads):
                off = np.abs(got[b, i, h] - want)
                assert (off <= limit).all(), (b, i, h, float((off / limit).max()), got[b, i, h][:4], want[:4])


@pytest.mark.parametrize('factor', [2.0 ** p for p in (-6, 0, 1, 2, 3, 4)])
@pytest.mark.parametrize('seq', SEQS)
@pytest.mark.parametrize('rise', [1, -1])
@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_scores_that_rise_by_a_little(device, format, rise, seq, factor):
    """Large scores, from block to block four units (or one step of fp32 where that is more) higher or lower: a running
    maximum that is not raised for each must not let probabilities run over.  Scores are exact: 63 dims of +-127 c (or 448 c)
    and one whose code counts the blocks, times whole numbers.  The bound is that of equal scores, with the exact weights."""
    announce('kv rising scores', format, rise, seq, factor)
    heads, kv_heads, dim, n = 1, 1, 64, 500
    unit = 127.0 if format == 'int8' else 448.0
    blocks = (n + 63) // 64
    sign = np.random.default_rng(220).choice([-1.0, 1.0], dim)
    k = np.broadcast_to(sign * unit, (n, dim)).copy()
    level = np.arange(n) // 64 if rise > 0 else blocks - 1 - np.arange(n) // 64
    k[:, 5] = level                                     # 0 .. 7: exact in both formats
    k = k.astype(np.float16)[None, :, None]
    v = rows_of(221, 1, n, kv_heads, dim)
    step = max(1.0, 4.0 / factor)                       # raw score a level: times factor 4, or factor
    q = np.broadcast_to(sign * (1000.0 if format == 'int8' else 280.0), (1, seq, heads, dim)).copy()
    q[..., 5] = step
    q = q.astype(np.float16)
    raw = np.einsum('d,nd->n', q[0, 0, 0].astype(np.float64), k[0, :, 0].astype(np.float64))
    assert np.abs(raw).max() < 2 ** 24 and (raw == np.rint(raw)).all() and np.float64(q[0, 0, 0, 5]) == step
    t = raw * factor
    assert (t.astype(np.float32) == t).all()
    scale = scale_for(factor)
    cache = held_by(device, format, k, v, 512)
    first = n - seq
    got = lb.kv_attention(dev(q, device), cache, ints([first], device), scale=scale).float().cpu().numpy().astype(np.float64)
    hv = ko.held(v[0, :, 0], format)
    for i in range(seq):
        p = np.exp2(t[:first + i + 1] - t[:first + i + 1].max())
        p /= p.sum()
        want, weight = p @ hv[:first + i + 1], p @ np.abs(hv[:first + i + 1])
        limit = weight * (2 * HALF + 2.0 ** -18 + 2.0 ** -13) + HALF * np.abs(want) + 2.0 ** -25 + n * 2.0 ** -32 * np.abs(hv).max()
        off = np.abs(got[0, i, 0] - want)
        assert (off <= limit).all(), (i, float((off / limit).max()), got[0, i, 0][:4], want[:4])


@pytest.mark.parametrize('seq,heads', [(1, 2), (8, 2), (70, 2)])
@pytest.mark.parametrize('format,dim', [('int8', 64), ('fp8', 128)])
def test_small_probabilities_count(device, format, dim, seq, heads):
    """Thousands of slots whose probabilities lie between 2^-14 and 2^-40 of the largest.

    The bound is that of test_gpu_kv.py but for the probabilities that fp16 holds with fewer bits.  Lifted by 2^10 (2^9 in
    tiles of 128 rows, where a ratio of value scales of up to 2^2 comes in) they are off by 2^-25
    of that: n 2^-35 max|v| in the sum and in the total, n 2^-32 in tiles."""
    announce('kv small probabilities', format, dim, seq, heads)
    kv_heads, starts = 1, [9000, 4097]
    batch, capacity = len(starts), 9152
    total = max(starts) + seq
    k, v = rows_of(230, batch, total, kv_heads, dim), rows_of(231, batch, total, kv_heads, dim)
    q = rows_of(232, batch, seq, heads, dim)
    # Values of 600, but of 0.01 where the first query's probability is above 2^-14 of the largest: the small ones are its sum.
    t = np.einsum('bd,bnd->bn', q[:, 0, 0].astype(np.float64), k[:, :, 0].astype(np.float64)) * dim ** -0.5 / np.log(2)
    seen = np.arange(total) <= np.array(starts)[:, None]
    top = np.where(seen, t, -np.inf).max(1, keepdims=True)
    v *= np.where(t > top - 14, 0.01, 600)[:, :, None, None].astype(np.float16)
    assert 0.2 < ((t < top - 14) & (t > top - 40)).mean() < 0.6
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints([s + seq for s in starts], device))
    scale = float(np.float32(dim ** -0.5))
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device), scale=scale).float().cpu().numpy().astype(np.float64)
    small = 2.0 ** (-35 if seq * heads <= 32 else -32)
    worst = 0.0
    for b in range(batch):
        n = starts[b] + seq
        kh, vh = (ko.held(t[b, :n, 0], format) for t in (k, v))
        for h in range(heads):
            out, weight, reach = ko.attend(q[b, :, h], kh, vh, starts[b], scale)
            limit = (weight * (2 * HALF + 2 * (dim + 8) * 2.0 ** -24 * reach[:, None] + n * 2.0 ** -24) + 2 * n * small * np.abs(vh).max()
                     + HALF * np.abs(out) + 2.0 ** -25)
            off = np.abs(got[b, :, h] - out)
            worst = max(worst, float((off / limit).max()))
            assert (off <= limit).all(), (b, h, float((off / limit).max()))
    print(f'[kv small probabilities] {format} {dim} {seq}: {worst:.2f} of the bound', flush=True)


@pytest.mark.parametrize('appended', [False, True])
@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_long_sequences_far_apart_in_a_large_batch(device, format, appended):
    """600 sequences, five of them long enough to be taken in parts: before, at and behind each 256th, where the search for a
    workgroup's sequence goes on to the next 256; the last row in the cache already, or appended by the call."""
    announce('kv large batch in parts', format, appended)
    batch, heads, kv_heads, dim, capacity = 600, 2, 1, 64, 4096
    rng = np.random.default_rng(240)
    starts = [int(x) for x in rng.integers(0, 190, batch)]
    far = {3: 4095, 255: 4031, 256: 3000, 511: 4094, 599: 4032}
    for b, s in far.items():
        starts[b] = s
    some = sorted({*far, 0, 1, 254, 257, 510, 512, 598, *(int(x) for x in rng.integers(0, batch, 20))})
    k, v = rows_of(241, batch, 192, kv_heads, dim), rows_of(242, batch, 192, kv_heads, dim, spread=.3)
    more = [rows_of(243 + i, 1, capacity, kv_heads, dim) for i in range(2)]      # rows 192 .. of the long ones
    q = rows_of(245, batch, 1, heads, dim)
    lengths = [s + (not appended) for s in starts]
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints([min(n, 192) for n in lengths], device))
    wide = [dev(t[:, 192:], device).expand(batch, -1, -1, -1) for t in more]
    lb.kv_append(cache, *wide, ints([192 if b in far else 0 for b in range(batch)], device),
                 rows=ints([lengths[b] - 192 if b in far else 0 for b in range(batch)], device))
    full = [np.concatenate((x[some], np.repeat(t[:, 192:], len(some), 0)), 1) for x, t in zip((k, v), more)]
    last = {}
    if appended:
        rows = [np.stack([(x[b] if s < 192 else t[0])[s] for b, s in enumerate(starts)])[:, None] for x, t in zip((k, v), more)]
        last = dict(k=dev(rows[0], device), v=dev(rows[1], device))
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device), **last)
    worst = check_attention(got[some], q[some], *full, [starts[b] for b in some], [1] * len(some), format, dim ** -0.5, kv_heads)
    print(f'[kv large batch in parts] {format}: {worst:.2f} of the bound', flush=True)
    assert bool(torch.isfinite(got).all())
