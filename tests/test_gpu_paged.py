"""lb_paged_append and lb_paged_attention against their definitions in 64 bits.

Append: values are copied; a turned key has the tolerance of the rotation (2^-20 of its pair's magnitudes, and its own half step).

Attention: with p the probabilities, A = sum p |v|, R the largest sum |q k| scale of a score and n slots, the kernel differs by
  - the rounding of each probability to fp16, half a step of it, in the sum with V and in the total (twice A eps / 2), and of those
    below 2^-14, half of 2^-24 relative to a largest one of 2^10 or more (n 2^-35 max|v|, twice); to two numbers of bf16, half a
    step of the second, which is half a step of the first and less: 2^-17 A (in the sum alone);
  - the score in fp32: D exact products' sums and the scaling (factors of 1 +- (D + 4) 2^-24 R), the reference's subtraction (a score
    is at most R log2(e) in units of log2, its half step 2^-24 of that) and the exponential (2^-22): each on p, in the sum and total;
  - of a turned q (and k): the rotation's 2^-20 (as test_gpu_rotary derives; twice for |a| + |b| against a value of the pair, in
    the sum over dims at most that), and what is left of q as two numbers of the type, 2^-17 (bf16, as above): 2^-17 + 2^-19 R in all;
  - sums of n / 32 steps and of 256 parts in fp32, each a rounding of A: (n / 32 + 300) 2^-24 A, and the total's, twice;
  - the output's own half step.
All are counted at their worst and added.
"""
import copy
import pickle

import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import serve_oracle as so

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def host(t):
    return t.float().cpu().numpy()


def ints(values, device):
    return torch.tensor(values, dtype=torch.int64, device=device)


def table_of(device, lengths, page, pages, seed=0, wide=0):
    """Pages in a random order; -1 behind a sequence's."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(pages)
    longest = max(1, max(-(-n // page) for n in lengths)) + wide
    table, at = np.full((len(lengths), longest), -1, np.int32), 0
    for b, n in enumerate(lengths):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    assert at <= pages
    return torch.from_numpy(table).to(device)


def filled(device, type, pages, kv, page, dim, seed=1, loud=True):
    g = torch.Generator().manual_seed(seed)
    keys = torch.randn((pages, kv, page, dim), generator=g)
    if loud:
        keys[..., ::17] *= 5
    return lb.PagedKVCache(keys.to(TYPES[type]).to(device),
                           torch.randn((pages, kv, page // 16, dim, 16), generator=g).to(TYPES[type]).to(device))


def rand(device, type, *shape, seed=2):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[type]).to(device)


def forget(cache, table, lengths, value=float('nan')):
    """NaN in every slot that no sequence holds."""
    page = cache.page
    live = np.zeros((cache.pages, page), bool)
    for row, n in zip(table.cpu().numpy(), lengths):
        for p in range(n):
            live[row[p // page], p % page] = True
    gone = torch.from_numpy(~live).to(cache.device)
    cache.keys.permute(0, 2, 1, 3)[gone] = value
    by_slot = cache.values.permute(0, 2, 4, 1, 3)     # a view [pages, chunks, 16, kv, D]
    by_slot[gone.view(cache.pages, page // 16, 16)] = value


def check(out, q, cache, table, position, scale, type, turned=False):
    """out [batch, heads, D] against the definition over what the cache holds; q in 64 bits where it is turned."""
    keys, values = host(cache.keys), host(cache.values)
    eps = torch.finfo(TYPES[type]).eps
    for b, at in enumerate(position):
        n, dim = at + 1, cache.head_dim
        k, v = so.held(keys, values, table[b, :-(-n // cache.page)].tolist(), n)
        want, mean, size = so.attention(q[b] if turned else host(q[b]), k, v, scale)
        R = size[:, None]
        score = ((dim + 8) * 2.0 ** -24 + (2.0 ** -17 + 2.0 ** -19 if turned else 0)) * R + 2.0 ** -22
        tiny = 2 * n * 2.0 ** -35 * np.abs(v).max() if type == 'fp16' else 0.0
        near = ((eps if type == 'fp16' else 2.0 ** -17) + 2 * np.expm1(score) + 2 * (n / 32 + 300) * 2.0 ** -24) * mean + tiny
        bound = near + eps / 2 * (np.abs(want) + near) + 2.0 ** -25 * (type == 'fp16')
        got = host(out[b]).astype(np.float64)
        worst = float(np.max(np.abs(got - want) / bound))
        assert worst <= 1, (b, at, worst)    # (a NaN fails too)


CASES = [
    # type, heads, kv_heads, dim, page, lengths
    ('fp16', 9, 3, 64, 16, [1]),
    ('bf16', 9, 3, 64, 64, [2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65]),
    ('fp16', 32, 8, 128, 32, [100, 1, 513]),
    ('bf16', 32, 8, 128, 128, [511, 512, 513, 1025]),
    ('fp16', 8, 8, 64, 16, [700, 40]),
    ('bf16', 16, 1, 128, 64, [600]),
    ('fp16', 24, 1, 64, 32, [520, 3]),
    ('bf16', 40, 1, 128, 16, [530, 17]),
    ('fp16', 5, 5, 128, 1024, [1500, 1024, 1]),
    ('fp16', 9, 3, 64, 64, [5003]),
    ('bf16', 8, 2, 128, 16, [9001, 20]),
    ('fp16', 3, 3, 64, 16, [(b * 37) % 90 + 1 for b in range(70)]),
    ('fp16', 8, 8, 64, 64, [100 + (b * 7919) % 3500 for b in range(18)]),
    ('bf16', 6, 2, 128, 16, [1 + (b * 7919) % 2500 for b in range(40)]),
    ('fp16', 16, 16, 64, 32, [2100, 900] + [1 + b % 40 for b in range(62)]),
    ('bf16', 16, 16, 64, 32, [2100] + [1 + b % 40 for b in range(69)]),
    ('bf16', 4, 1, 64, 32, [1 + (b % 7) * 400 * (b % 31 == 0) + b % 50 for b in range(200)]),
    ('fp16', 16, 8, 128, 32, [1 + (b * 7919) % 1500 for b in range(36)]),
    ('bf16', 24, 1, 64, 64, [26001, 9]),
    ('fp16', 16, 1, 128, 64, [20000]),
    ('bf16', 8, 8, 128, 16, [3000] + [1 + b % 40 for b in range(80)]),
    ('bf16', 12, 12, 128, 64, [513, 512, 1] + [1 + b % 30 for b in range(21)]),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c[:5])) + f'-b{len(c[5])}-n{max(c[5])}')
def test_attention(device, case):
    """Over pages in any order, with NaN in every slot and page that is not held, and -1 in the table behind a sequence's pages."""
    type, heads, kv, dim, page, lengths = case
    announce('paged attention', case[:5], max(lengths))
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = filled(device, type, pages, kv, page, dim)
    table = table_of(device, lengths, page, pages, wide=3)
    forget(cache, table, lengths)
    q = rand(device, type, len(lengths), heads, dim)
    position = [n - 1 for n in lengths]
    out = lb.paged_attention(q, cache, table, ints(position, device))
    check(out, q, cache, table.cpu(), position, dim ** -0.5, type)
    again = lb.paged_attention(q, cache, table, ints(position, device), out=torch.full_like(q, 3.0))
    assert torch.equal(out, again)


@pytest.mark.parametrize('type', ['fp16', 'bf16'])
@pytest.mark.parametrize('scale', [0.0, 1.0, -0.3, 40.0])
def test_scores(device, type, scale):
    """No, large and negative scores; equal ones (scale 0) are a mean."""
    announce('paged scores', type, scale)
    lengths = [900, 77]
    cache = filled(device, type, 70, 2, 16, 64, seed=5)
    table = table_of(device, lengths, 16, 70)
    q = rand(device, type, 2, 6, 64, seed=6)
    out = lb.paged_attention(q, cache, table, ints([899, 76], device), scale=scale)
    check(out, q, cache, table.cpu(), [899, 76], scale, type)


def test_infinite_and_lowest_values(device):
    """A key of -inf scores leaves its slot out; the type's lowest keys are large scores like others; a NaN that is held shows."""
    announce('paged infinities')
    for type in ('fp16', 'bf16'):
        cache = filled(device, type, 3, 1, 64, 64, seed=7)
        table = ints([[0, 1, 2]], device).int()
        q = torch.ones((1, 2, 64), dtype=TYPES[type], device=device)
        cache.keys[0, 0, 5], cache.keys[1, 0, 9] = float('-inf'), float('-inf')
        got = lb.paged_attention(q, cache, table, ints([150], device))
        kept = lb.PagedKVCache(cache.keys.clone(), cache.values.clone())
        kept.keys[0, 0, 5], kept.keys[1, 0, 9] = torch.finfo(TYPES[type]).min, torch.finfo(TYPES[type]).min
        if type == 'bf16':                 # 64 of them pass fp32's range in a sum: a quarter of a dim each
            kept.keys[0, 0, 5], kept.keys[1, 0, 9] = -1e36, -1e36
        low = lb.paged_attention(q, kept, table, ints([150], device))
        assert bool(got.isfinite().all()) and torch.equal(got, low)
        only = lb.PagedKVCache(torch.full_like(kept.keys, -1e4 if type == 'fp16' else -1e34), kept.values)
        out = lb.paged_attention(q, only, table, ints([99], device))     # all scores equal, and far below zero: a mean
        check(out, q, only, table.cpu(), [99], 0.0, type)
        cache.keys[0, 0, 7] = float('nan')
        assert bool(lb.paged_attention(q, cache, table, ints([150], device)).isnan().all())
        assert bool(lb.paged_attention(q, cache, table, ints([6], device)).isfinite().all())


def test_places_without_a_token_and_bad_tables(device):
    """-1: zeros.  Past the table, below -1, or over an entry that is no page: NaN in that sequence alone, nothing read or written."""
    announce('paged bad positions')
    cache = filled(device, 'fp16', 12, 2, 16, 64, seed=8)
    keys, values = cache.keys.clone(), cache.values.clone()
    table = ints([[0, 1], [2, 3], [4, 5], [6, 12], [7, -1], [8, 9], [2 ** 31 - 1, 10]], device).int()
    position = ints([20, -1, 32, 17, 16, 2 ** 40, 3], device)
    q, k, v = rand(device, 'fp16', 7, 4, 64), rand(device, 'fp16', 7, 2, 64, seed=3), rand(device, 'fp16', 7, 2, 64, seed=4)
    for more in ({}, dict(k=k, v=v)):
        out = lb.paged_attention(q, cache, table, position, **more)
        assert bool(out[0].isfinite().all()) and bool((out[1] == 0).all())
        assert all(bool(out[b].isnan().all()) for b in (2, 3, 4, 5, 6))
    position[:] = ints([-2, -(2 ** 63), 5, 15, 15, -1, -1], device)
    out = lb.paged_attention(q, cache, table, position)
    assert bool(out[:2].isnan().all()) and bool(out[2:5].isfinite().all()) and bool((out[5:] == 0).all())
    row = torch.zeros(12, 16, dtype=torch.bool, device=device)
    row[1, 4] = True                       # slot 20 of the first sequence
    assert torch.equal(cache.keys.permute(0, 2, 1, 3)[~row], keys.permute(0, 2, 1, 3)[~row])
    assert torch.equal(cache.keys[1, :, 4], k[0]) and torch.equal(cache.values[1, :, 0, :, 4], v[0])
    other = cache.values.clone()
    other[1, :, 0, :, 4] = values[1, :, 0, :, 4]
    assert torch.equal(other, values)


@pytest.mark.parametrize('type,heads,kv,dim,page,part,pairs', [
    ('fp16', 9, 3, 64, 16, None, 'half'), ('fp16', 9, 3, 64, 64, 64, 'half'), ('bf16', 32, 8, 128, 32, 128, 'neighbours'),
    ('bf16', 24, 1, 64, 16, 40, 'half'), ('fp16', 16, 1, 128, 128, 24, 'neighbours'), ('fp16', 5, 5, 128, 64, 20, 'half')])
def test_step(device, type, heads, kv, dim, page, part, pairs):
    """A token's key and value in the attention's launch: the cache as an append leaves it, and the output over it."""
    announce('paged step', type, heads, kv, dim, page, part, pairs)
    lengths = [1, page, page + 1, 33, 700, 16]
    pages = sum(-(-n // page) for n in lengths) + 1
    rotary = None if part is None else lb.Rotary(lb.rotary_frequencies(part, device=device), pairs=pairs, scale=1.1)
    table = table_of(device, lengths, page, pages)
    position = [n - 1 for n in lengths]
    rows = rand(device, type, len(lengths), heads + 2 * kv, dim, seed=9)        # q, k and v as slices of one projection
    q, k, v = rows.split((heads, kv, kv), 1)
    caches = [filled(device, type, pages, kv, page, dim, seed=10) for _ in range(2)]
    for cache in caches:
        forget(cache, table, position)     # (the new rows' slots among them)
    out = lb.paged_attention(q, caches[0], table, ints(position, device), k=k, v=v, rotary=rotary)
    lb.paged_append(caches[1], k.unsqueeze(1), v.unsqueeze(1), table, ints(position, device), rotary=rotary)
    assert torch.equal(caches[0].values.view(torch.int16), caches[1].values.view(torch.int16))
    a, b = caches[0].keys.float().nan_to_num(77.0), caches[1].keys.float().nan_to_num(77.0)
    # two roundings of one value, formed alike up to how a product and a sum are fused
    assert bool(((a - b).abs() <= torch.finfo(TYPES[type]).eps * torch.maximum(a.abs(), b.abs()) + 2.0 ** -19).all())
    q64 = host(q)
    if rotary is not None:
        q64 = so.turned(host(q)[:, None], np.array(position)[:, None], rotary.frequencies.cpu().numpy(), pairs, 1.1)[:, 0]
    check(out, q64 if rotary is not None else q, caches[0], table.cpu(), position, dim ** -0.5, type, rotary is not None)
    if rotary is None:
        assert torch.equal(a, b)
        held = lb.paged_attention(q, caches[1], table, ints(position, device))
        assert torch.equal(held, out)


APPENDS = [
    # type, kv_heads, dim, page, batch, seq, positions, rows, part, pairs
    ('fp16', 3, 64, 16, 1, 500, [3], None, 64, 'half'),
    ('bf16', 8, 128, 64, 3, 67, [0, 1, 130], [67, 0, 20], 128, 'neighbours'),
    ('fp16', 1, 64, 32, 4, 1, [0, 15, 16, 95], None, None, 'half'),
    ('bf16', 5, 128, 128, 2, 40, [120, 16], [33, 40], 40, 'half'),
    ('fp16', 9, 64, 1024, 1, 90, [7], [90], 6, 'half'),
    ('fp16', 2, 128, 16, 2, 17, [14, 31], None, 100, 'neighbours'),
    ('fp16', 3, 64, 16, 20, 400, [7 * b % 40 for b in range(20)], [400 - 19 * b for b in range(20)], 64, 'half'),
    ('bf16', 11, 128, 32, 6, 600, [0, 5, 16, 31, 600, 2], [600, 599, 600, 1, 0, 593], 128, 'half'),
    ('fp16', 8, 128, 64, 8, 600, [3 * b for b in range(8)], None, 64, 'neighbours'),
]


@pytest.mark.parametrize('case', APPENDS, ids=lambda c: '-'.join(map(str, c[:6])) + f'-{c[8]}-{c[9]}')
@pytest.mark.parametrize('layout', ['slices', 'plain', 'odd'])
def test_append(device, case, layout):
    """Rows at any slot, in whole, ragged and empty batches; what lies around them stays."""
    type, kv, dim, page, batch, seq, positions, rows, part, pairs = case
    announce('paged append', case, layout)
    counts = [seq] * batch if rows is None else rows
    ends = [p + n for p, n in zip(positions, counts)]
    pages = sum(-(-max(1, n) // page) for n in ends) + 2
    table = table_of(device, [max(1, n) for n in ends], page, pages, wide=-(-seq // page))
    cache = filled(device, type, pages, kv, page, dim)
    keys, values = host(cache.keys), host(cache.values)
    if layout == 'slices':
        k, v = rand(device, type, batch, seq, 2 * kv + 1, dim, seed=3)[:, :, 1:].split((kv, kv), 2)
    elif layout == 'plain':
        k, v = rand(device, type, batch, kv, seq, dim, seed=3).transpose(1, 2), rand(device, type, batch, seq, kv, dim, seed=4)
    else:                                  # rows that are not 16-byte pieces
        k = rand(device, type, batch, seq, kv, dim + 3, seed=3)[..., 1:dim + 1]
        v = rand(device, type, dim, batch, seq, kv, seed=4).permute(1, 2, 3, 0)
    rotary = None if part is None else lb.Rotary(lb.rotary_frequencies(part, device=device), pairs=pairs, scale=0.9)
    lb.paged_append(cache, k, v, table, ints(positions, device), rows=None if rows is None else ints(rows, device), rotary=rotary)
    got_k, got_v = host(cache.keys), so.values_by_slot(host(cache.values))
    at = np.array(positions)[:, None] + np.arange(seq)
    k64 = host(k).astype(np.float64)
    part_sizes = np.zeros_like(k64)
    if rotary is not None:
        f = rotary.frequencies.cpu().numpy()
        part_sizes = so.partner_sizes(k64, part // 2, pairs) * 0.9 * 2.0 ** -20
        k64 = so.turned(k64, at, f, pairs, 0.9)
    want_v = so.values_by_slot(values)
    for b in range(batch):
        for i in range(counts[b]):
            p = positions[b] + i
            id, off = int(table[b, p // page]), p % page
            near = part_sizes[b, i]
            bound = near + torch.finfo(TYPES[type]).eps / 2 * (np.abs(k64[b, i]) + near) * (rotary is not None) + 2.0 ** -25
            assert bool(np.all(np.abs(got_k[id, :, off] - k64[b, i]) <= bound)), (b, i)
            keys[id, :, off] = got_k[id, :, off]
            want_v[id, :, off] = host(v[b, i])
    assert np.array_equal(got_k, keys) and np.array_equal(got_v, want_v)


def test_append_in_any_calls(device):
    """Rows split into calls in any way leave the same bits."""
    announce('paged append split')
    kv, dim, page = 3, 64, 32
    k, v = rand(device, 'fp16', 1, 130, kv, dim, seed=3), rand(device, 'fp16', 1, 130, kv, dim, seed=4)
    rotary = lb.Rotary(lb.rotary_frequencies(64, device=device))
    table = ints([[4, 2, 0, 1, 3]], device).int()
    whole = lb.PagedKVCache.empty(5, kv, page=page, device=device)
    lb.paged_append(whole, k, v, table, ints([0], device), rotary=rotary)
    for cuts in ([0, 1, 2, 30, 31, 64, 129, 130], [0, 100, 130], list(range(131))):
        cache = lb.PagedKVCache.empty(5, kv, page=page, device=device)
        for a, b in zip(cuts, cuts[1:]):
            lb.paged_append(cache, k[:, a:b], v[:, a:b], table, ints([a], device), rotary=rotary)
        assert torch.equal(cache.keys, whole.keys) and torch.equal(cache.values, whole.values)
    keys, values = whole.read([4, 2, 0, 1, 3], 130)
    assert torch.equal(values, v[0].transpose(0, 1)) and keys.shape == (3, 130, 64)


def test_append_outside(device):
    """Sequences whose rows do not lie in the table are left alone, as are rows of entries that are no page."""
    announce('paged append outside')
    cache = filled(device, 'fp16', 6, 2, 16, 64)
    keys, values = cache.keys.clone(), cache.values.clone()
    k, v = rand(device, 'fp16', 6, 20, 2, 64, seed=3), rand(device, 'fp16', 6, 20, 2, 64, seed=4)
    table = ints([[0, 1], [0, 1], [0, 1], [0, 1], [-1, 6], [5, -3]], device).int()
    position, rows = ints([-1, 13, 2 ** 62, 0, 0, 10], device), ints([5, 20, 1, 21, 20, 20], device)
    lb.paged_append(cache, k, v, table, position, rows=rows)
    changed = torch.zeros(6, 16, dtype=torch.bool, device=device)
    changed[5, 10:] = True                 # the last sequence's rows that lie in its first page
    assert torch.equal(cache.keys.permute(0, 2, 1, 3)[~changed], keys.permute(0, 2, 1, 3)[~changed])
    assert torch.equal(cache.keys[5, :, 10:].transpose(0, 1), k[5, :6])
    values[5, :, 0, :, 10:] = v[5, :6].permute(1, 2, 0)
    assert torch.equal(cache.values, values)


def test_shared_pages(device):
    """A prefix that three sequences share, and one table row for all of a batch."""
    announce('paged shared')
    cache = filled(device, 'bf16', 9, 2, 16, 128)
    table = ints([[0, 1, 2], [0, 1, 3], [0, 1, 4]], device).int()
    q = rand(device, 'bf16', 3, 8, 128)
    check(lb.paged_attention(q, cache, table, ints([40, 33, 47], device)), q, cache, table.cpu(), [40, 33, 47], 128 ** -0.5, 'bf16')
    one = ints([5, 6, 7, 8], device).int().expand(3, 4)
    assert one.stride(0) == 0
    check(lb.paged_attention(q, cache, one, ints([63, 0, 31], device)), q, cache, one.cpu(), [63, 0, 31], 128 ** -0.5, 'bf16')


def test_capture(device):
    """A captured step reads table and positions at each replay: sequences grow, one ends and another begins in its place.  Two
    calls in one graph share a workspace in turn; eager work goes on between the replays."""
    announce('paged capture')
    kv, heads, dim, page = 2, 4, 64, 16
    cache = filled(device, 'fp16', 260, kv, page, dim)
    start = [2000, 600, 5]
    table = table_of(device, [n + 20 for n in start], page, 200)
    position = ints(start, device)
    q, k, v = rand(device, 'fp16', 3, heads, dim), rand(device, 'fp16', 3, kv, dim, seed=3), rand(device, 'fp16', 3, kv, dim, seed=4)
    out, second = torch.zeros_like(q), torch.zeros_like(q)
    step = lb.PreparedPagedAttention(q, cache, table, position, out, k=k, v=v)
    more = lb.PreparedPagedAttention(q, cache, table, position, second, scale=0.5, workspace=step.scratch)
    step.run()
    more.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
        more.run()
        free = lb.paged_attention(q, cache, table, position)
    for turn in range(4):
        q.copy_(rand(device, 'fp16', 3, heads, dim, seed=20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        eager = lb.paged_attention(q, cache, table, position)
        assert torch.equal(out, eager) and torch.equal(free, eager)
        assert torch.equal(second, lb.paged_attention(q, cache, table, position, scale=0.5))
        check(out, q, cache, table.cpu(), position.tolist(), 0.125, 'fp16')
        position += 1
        if turn == 1:
            position[1] = 0
            table[1, 0] = 230


def test_streams(device):
    """Calls on two streams at once, each with the workspace of its stream."""
    announce('paged streams')
    cache = filled(device, 'fp16', 300, 2, 16, 128)
    table = table_of(device, [3000, 1500], 16, 300)
    position, q = ints([2999, 1499], device), rand(device, 'fp16', 2, 8, 128)
    want = lb.paged_attention(q, cache, table, position)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(lb.paged_attention(q, cache, table, position))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


def test_copies_and_pickles(device):
    """They have buffers of their own, and calls over them read those."""
    announce('paged copies')
    cache, table = filled(device, 'bf16', 5, 2, 32, 64), ints([[4, 1, 3]], device).int()
    rotary = lb.Rotary(lb.rotary_frequencies(64, device=device), pairs='neighbours', scale=1.5)
    q, position = rand(device, 'bf16', 1, 6, 64), ints([80], device)
    want = lb.paged_attention(q, cache, table, position, rotary=rotary)
    for again in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        twin, turns = again(cache), again(rotary)
        assert twin.keys.data_ptr() != cache.keys.data_ptr() and torch.equal(twin.keys, cache.keys) and torch.equal(twin.values, cache.values)
        assert torch.equal(lb.paged_attention(q, twin, table, position, rotary=turns), want)
        twin.keys.zero_()
        assert not torch.equal(lb.paged_attention(q, twin, table, position, rotary=turns), want)
    assert torch.equal(lb.paged_attention(q, cache, table, position, rotary=rotary), want)
    with pytest.raises(AttributeError):
        cache.keys = cache.keys.clone()
    with pytest.raises(AttributeError):
        rotary.scale = 2.0


def test_read(device):
    announce('paged read')
    cache = filled(device, 'fp16', 3, 2, 16, 64)
    keys, values = cache.read([2, 0], 20)
    assert torch.equal(keys[:, :16], cache.keys[2]) and torch.equal(keys[:, 16:], cache.keys[0][:, :4])
    assert torch.equal(values[:, 16:], cache.values[0, :, 0].transpose(1, 2)[:, :4])
    again = cache.read(ints([2, 0, -1], device).int(), 20)       # (a row of a table, with what stands behind the sequence's pages)
    assert torch.equal(again[0], keys) and torch.equal(again[1], values)
    assert cache.read([], 0)[0].shape == (2, 0, 64)
    for pages, length in (([2, 3], 20), ([-1], 1), ([0], 17), ([0], -1)):
        with pytest.raises(ValueError):
            cache.read(pages, length)


def test_far_pages(device):
    """Pages whose offsets pass 32 bits, in elements and in bytes."""
    announce('paged far')
    pages, kv, page, dim = 70000, 8, 64, 128   # 2^32 elements and more
    keys = torch.empty((pages, kv, page, dim), dtype=torch.float16, device=device)
    values = torch.empty((pages, kv, page // 16, dim, 16), dtype=torch.float16, device=device)
    small = filled(device, 'fp16', 4, kv, page, dim)
    far = [69999, 32767, 65535, 65536]
    keys[far], values[far] = small.keys, small.values
    cache = lb.PagedKVCache(keys, values)
    q, k, v = rand(device, 'fp16', 1, 32, dim), rand(device, 'fp16', 1, kv, dim, seed=3), rand(device, 'fp16', 1, kv, dim, seed=4)
    position = ints([200], device)
    out = lb.paged_attention(q, cache, ints([far], device).int(), position, k=k, v=v)
    near = lb.paged_attention(q, small, ints([[0, 1, 2, 3]], device).int(), position, k=k, v=v)
    assert torch.equal(out, near)
    rows = rand(device, 'fp16', 1, 100, kv, dim, seed=5)
    lb.paged_append(cache, rows, rows, ints([far], device).int(), ints([100], device))
    lb.paged_append(small, rows, rows, ints([[0, 1, 2, 3]], device).int(), ints([100], device))
    assert torch.equal(cache.keys[far], small.keys) and torch.equal(cache.values[far], small.values)
