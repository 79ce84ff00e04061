"""lb_paged_attention where the bits of its probabilities and the range of its numbers show, against its definition in 64 bits
(the bounds of test_gpu_paged, but for what is said here)."""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import serve_oracle as so
from test_gpu_paged import check, TYPES, filled, host, ints, rand, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('type', ['fp16', 'bf16'])
@pytest.mark.parametrize('heads,kv,dim', [(4, 2, 64), (8, 8, 128)])
def test_probabilities_keep_their_bits(device, type, heads, kv, dim):
    """Sums over 31 slots that cancel: what is rounded of a probability is then large beside the output.

    The last slot's value is set against the sum of the others, so that of A = sum p |v| hardly anything is left and the output's own
    half step is small.  A probability enters as two numbers of its type: what is left of it is half a step of the second (a quarter
    of the square of the type's step: 2^-22 of it in fp16, 2^-17 in bf16 as test_gpu_paged counts it), and of fp16 half of
    2^-24 relative to a largest one of 2^10 (31 2^-35 of max|v|).  The score: (D + 8) 2^-24 R and the exponential's 2^-22, in the sum
    and in the total.  One unit of slots in one wave: 32 additions of the products, 8 of the waves, the same of the total,
    and a quotient: 96 2^-24.  Rounded to one fp16 number, each p is off by up to 2^-12 of A by itself."""
    announce('paged bits', type, heads, kv, dim)
    n, page, eps = 31, 16, torch.finfo(TYPES[type]).eps
    cache = filled(device, type, 3, kv, page, dim, seed=21, loud=False)
    cache.keys.mul_(0.0625)
    table = ints([[2, 0]], device).int()
    q = rand(device, type, 1, heads, dim, seed=22)
    scale, group = dim ** -0.5, heads // kv
    keys, values = host(cache.keys), host(cache.values)
    k, v = so.held(keys, values, [2, 0], n)
    for h in range(kv):                     # against the sum that the group's first query sees
        s = k[h] @ host(q)[0, h * group].astype(np.float64) * scale
        p = np.exp(s - s.max())
        values[0, h, 0, :, (n - 1) % 16] = -(p[:-1] @ v[h, :-1]) / p[-1]
    cache.values.copy_(torch.from_numpy(values))
    values = host(cache.values)
    k, v = so.held(keys, values, [2, 0], n)
    want, mean, size = so.attention(host(q[0]), k, v, scale)
    out = host(lb.paged_attention(q, cache, table, ints([n - 1], device))[0]).astype(np.float64)
    score = (dim + 8) * 2.0 ** -24 * size[:, None] + 2.0 ** -22
    left, tiny = (2.0 ** -22, n * 2.0 ** -35 * np.abs(v).max()) if type == 'fp16' else (2.0 ** -17, 0.0)
    near = (left + 2 * np.expm1(score) + 2 * 96 * 2.0 ** -24) * mean + 2 * tiny
    bound = near + eps / 2 * (np.abs(want) + near) + 2.0 ** -25 * (type == 'fp16')
    first = np.arange(kv) * group
    worst = float(np.max((np.abs(out - want) / bound)))
    assert float(np.median(np.abs(want[first]) / mean[first])) < eps      # (they do cancel)
    assert worst <= 1, worst


@pytest.mark.parametrize('type', ['fp16', 'bf16'])
@pytest.mark.parametrize('sign', [1, -1])
def test_scores_of_any_size(device, type, sign):
    """Equal scores of 2^5 to 2^34 in units of log2, on either side of zero: the values' mean, however coarse the scores' own steps
    are (16 of those units from 2^27 on).  Then one slot a step above the others: past 2^32, where a step is 512, its value alone.

    All probabilities are equal, so that they cancel exactly from the quotient but for their sums: 2^-16 covers 8 additions a lane of
    each, the joins' and the quotient's, and bf16's second number (2^-17); then the output's half step."""
    announce('paged scores of any size', type, sign)
    n, page, dim = 200, 32, 64
    cache = filled(device, type, 7, 1, page, dim, seed=31)
    table = ints([list(range(7))], device).int()
    _, v = so.held(host(cache.keys), host(cache.values), range(7), n)
    mean, size = v[0].mean(0), np.abs(v[0]).mean(0)
    q = torch.zeros((1, 2, dim), dtype=TYPES[type], device=device)
    q[0, :, 3] = 2.0 ** 11
    half = torch.finfo(TYPES[type]).eps / 2
    cache.keys.zero_()
    for e in range(-17, 13):
        for part in (1.0, 1.25, 1.375):
            cache.keys[..., 3] = sign * 2.0 ** 11 * part
            out = host(lb.paged_attention(q, cache, table, ints([n - 1], device), scale=2.0 ** e))[0].astype(np.float64)
            worst = float(np.max(np.abs(out - mean) / ((half + 2.0 ** -16) * size + 2.0 ** -25)))
            assert worst <= 1, (e, part, worst)
    cache.keys[2, 0, 9, 3] *= 1.0 + sign * torch.finfo(TYPES[type]).eps * 2     # slot 73: the largest by a 512th or more
    out = lb.paged_attention(q, cache, table, ints([n - 1], device), scale=2.0 ** 12)
    assert torch.equal(out[0, 0], cache.values[2, 0, 0, :, 9]) and torch.equal(out[0, 1], out[0, 0])


@pytest.mark.parametrize('heads,kv,dim,lengths', [(4, 2, 64, [300, 5, 3000]), (6, 2, 128, [40, 1200]), (2, 2, 64, [70] * 66)])
@pytest.mark.parametrize('size', [2.0 ** 124, 2.0 ** -100])
def test_values_of_any_size(device, heads, kv, dim, lengths, size):
    """bf16 values near the type's largest and smallest: no sum on the way passes 32 bits' range where the output does not."""
    announce('paged values of any size', heads, kv, dim, size)
    page = 64
    pages = sum(-(-n // page) for n in lengths) + 1
    cache = filled(device, 'bf16', pages, kv, page, dim, seed=41)
    cache.values.mul_(size)
    table, position = table_of(device, lengths, page, pages), [n - 1 for n in lengths]
    q = rand(device, 'bf16', len(lengths), heads, dim, seed=42)
    out = lb.paged_attention(q, cache, table, ints(position, device))
    check(out, q, cache, table.cpu(), position, dim ** -0.5, 'bf16')
    if size > 1:
        top = torch.finfo(torch.bfloat16).max
        cache.values.fill_(top)
        out = lb.paged_attention(q, cache, table, ints(position, device))
        assert bool((out == top).all())


@pytest.mark.parametrize('dim,whole', [(64, 1024), (128, 512)])
@pytest.mark.parametrize('batch', [3, 70])
def test_about_the_longest_that_is_not_split(device, dim, whole, batch):
    """Tables of as many slots as are never split, which take no workspace, and of a page more."""
    announce('paged whole', dim, batch)
    page = 16
    for slots in (whole, whole + page):
        lengths = [slots, slots - 15, 1] + [1 + (b * 7919) % slots for b in range(batch - 3)]
        pages = sum(-(-n // page) for n in lengths) + 1
        cache, table = filled(device, 'fp16', pages, 2, page, dim, seed=51), table_of(device, lengths, page, pages)
        assert table.shape[1] * page == slots
        q, position = rand(device, 'fp16', batch, 6, dim, seed=52), [n - 1 for n in lengths]
        call = lb.PreparedPagedAttention(q, cache, table, ints(position, device), torch.zeros_like(q))
        assert (call.scratch is None) == (slots == whole)
        call.run()
        check(call.out, q, cache, table.cpu(), position, dim ** -0.5, 'fp16')
