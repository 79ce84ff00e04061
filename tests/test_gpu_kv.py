"""GPU parity of the 8-bit KV cache (lb_kv_append, lb_kv_read, lb_kv_attention) against the 64-bit oracle.

Codes, scales, the fp16 tails and what is read back are compared bit for bit: the definition leaves no rounding open
(the quotient's ties are exact, everything else is rounded once).

Attention: with p the probabilities, A = sum p |v| and n slots, the kernel differs from the 64-bit result by
  - the rounding of each probability to fp16, half a step 2^-11 of it, in the sum with V (A 2^-11) and in the total
    (|out| 2^-11 <= A 2^-11), and of probabilities below 2^-14, half a step of 2^-25 each (n 2^-25 max|v|, twice);
  - the fp32 score: D products and their sum, a scale or two and an exponential, each 2^-24 of at most
    R = max sum |q k| scale, so a factor of 1 +- (D + 8) 2^-24 R on each probability (2 A of that);
  - fp32 sums of n / 64 rescaled blocks of V, n 2^-24 A at the most;
  - the rounding of the output, 2^-11 |out| (2^-25 below 2^-14).
All are counted at their worst and added.
"""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import kv_oracle as ko

pytestmark = pytest.mark.gpu
PLACES = np.array([ko.place(s) for s in range(64)])


def rows_of(seed, *shape, spread=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape) * spread
    x[..., :: 17] *= 6
    return x.astype(np.float16)


def dev(a, device):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device)


def ints(values, device):
    return torch.tensor(values, dtype=torch.int64, device=device)


def fresh(device, batch, heads, capacity, dim, format, fill=0x35):
    """A cache whose memory is full of a pattern, so that writes outside of what a call may write show."""
    cache = lb.QuantizedKVCache.empty(batch, heads, capacity, head_dim=dim, format=format, device=device)
    for t in cache.tensors():
        t.view(torch.uint8).fill_(fill)
    return cache


def expect(fill, k, v, lengths, capacity, format, history=None):
    """The cache's buffers as numpy bytes after rows k, v [batch, slots, heads, D] up to `lengths` were appended.
    Tail slots that no row went to keep the pattern; history [b]: the most slots a sequence ever held."""
    batch, _, heads, dim = k.shape
    blocks = (capacity + 63) // 64
    word = np.frombuffer(bytes([fill] * 4), np.uint32)[0]
    kc = np.full((batch, heads, blocks, 64, dim), fill, np.uint8)
    vc = np.full((batch, heads, blocks, dim, 64), fill, np.uint8)
    ks, vs = (np.full((batch, heads, blocks), word, np.uint32) for _ in range(2))
    kt = np.full((batch, heads, 2, 64, dim), word & 0xFFFF, np.uint16)
    vt = np.full((batch, heads, 2, dim, 64), word & 0xFFFF, np.uint16)
    for b in range(batch):
        n = lengths[b]
        for h in range(heads):
            kr, vr = ko.poison(k[b, :n, h], v[b, :n, h])
            for i in range(n // 64):
                kq, s0 = ko.quantise(kr[64 * i:64 * i + 64], format)
                vq, s1 = ko.quantise(vr[64 * i:64 * i + 64], format)
                bits = (lambda c: c.astype(np.int8).view(np.uint8)) if format == 'int8' else ko.e4m3_bits
                kc[b, h, i] = bits(kq)
                vc[b, h, i][:, PLACES] = bits(vq).T
                ks[b, h, i], vs[b, h, i] = s0.view(np.uint32), s1.view(np.uint32)
            for slot in range(max(0, (n // 64 - 1) * 64), n):
                kt[b, h, slot // 64 % 2, slot % 64] = kr[slot].view(np.uint16)
                vt[b, h, slot // 64 % 2, :, PLACES[slot % 64]] = vr[slot].view(np.uint16)
    return kc, vc, ks, vs, kt, vt


def same(got, want):
    """Bits of two fp16 (or integer) arrays; says where they differ."""
    got, want = (np.ascontiguousarray(a).view(np.uint16) if a.dtype == np.float16 else a for a in (got, want))
    assert got.shape == want.shape, (got.shape, want.shape)
    at = np.argwhere(got != want)
    assert not len(at), (len(at), at[:3].tolist(), got[got != want][:3], want[got != want][:3])


def buffers(cache):
    kinds = (np.uint8, np.uint8, np.uint32, np.uint32, np.uint16, np.uint16)
    return [t.contiguous().view(torch.uint8).cpu().numpy().view(kind).reshape(t.shape)
            for t, kind in zip(cache.tensors(), kinds)]


def canonical(name, a):
    """NaN payloads are not part of the definition."""
    if name.endswith('scales'):
        return np.where((a & 0x7FFFFFFF) > 0x7F800000, 0x7FC00000, a)
    if name.endswith('tail'):
        return np.where((a & 0x7FFF) > 0x7C00, 0x7E00, a)
    return a


def check_buffers(cache, want, only_tail=None):
    for name, got, exp in zip(('key_codes', 'value_codes', 'key_scales', 'value_scales', 'key_tail', 'value_tail'),
                              buffers(cache), want):
        got, exp = canonical(name, got), canonical(name, exp)
        if name.endswith('tail') and only_tail is not None:
            got, exp = got[only_tail(name)], exp[only_tail(name)]
        same(got, exp)


# ---------------------------------------------------------------- append
SPLITS = [(1,), (64,), (63, 1), (130,), (5, 59, 64, 1), (62, 5, 70), (10, 200), (33, 31, 1, 127, 3), (64, 64, 64, 9),
          (20, 300), (127, 2, 130)]


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('split', SPLITS, ids=['+'.join(map(str, s)) for s in SPLITS])
def test_append_holds_what_the_definition_says(device, format, dim, split):
    """However the rows are split into calls, codes, scales and the open block's rows are the same."""
    announce('kv append', format, dim, split)
    batch, heads, total = 2, 3, sum(split)
    capacity = (total + 63) // 64 * 64 + 64
    k, v = rows_of(1, batch, total, heads, dim), rows_of(2, batch, total, heads, dim, spread=.02)
    cache = fresh(device, batch, heads, capacity, dim, format)
    at = 0
    for n in split:
        lb.kv_append(cache, dev(k[:, at:at + n], device), dev(v[:, at:at + n], device), ints([at] * batch, device))
        at += n
    want = expect(0x35, k, v, [total] * batch, capacity, format)

    def only(name):   # a ring half may also hold rows of the block two before; what matters is the last two blocks' rows
        mask = np.zeros((batch, heads, 2, 64, dim), bool)
        for slot in range(max(0, (total // 64 - 1) * 64), total):
            mask[:, :, slot // 64 % 2, slot % 64] = True
        if name == 'value_tail':
            turned = np.zeros((batch, heads, 2, dim, 64), bool)
            turned[..., PLACES] = np.swapaxes(mask, -1, -2)
            return turned
        return mask
    check_buffers(cache, want, only)


@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_append_ragged_and_nothing_else(device, format):
    """Each sequence its own position and rows; sequences without rows, past the capacity or before slot 0 are left alone,
    and so is every byte outside the appended rows' blocks."""
    announce('kv append ragged', format)
    dim, heads, capacity, seq = 64, 2, 192, 100
    starts = [0, 0, 0, 100, -1, 190, 2 ** 40, 0, 0, 92]
    rows = [100, 64, 0, 100, 5, 5, 5, -3, 101, 100]
    good = [0 <= p and 0 <= n <= seq and p + n <= capacity for p, n in zip(starts, rows)]
    assert good == [True, True, True, False, False, False, False, False, False, True]
    batch = len(starts)
    k, v = rows_of(3, batch, seq, heads, dim), rows_of(4, batch, seq, heads, dim)
    cache = fresh(device, batch, heads, capacity, dim, format, fill=0x2A)
    first = buffers(cache.clone())
    # the last sequence holds 92 rows already (in its own cache memory: appended alone, rows of zero elsewhere)
    k0, v0 = rows_of(5, batch, 92, heads, dim), rows_of(6, batch, 92, heads, dim)
    lb.kv_append(cache, dev(k0, device), dev(v0, device), ints([0] * batch, device), rows=ints([0] * 9 + [92], device))
    lb.kv_append(cache, dev(k, device), dev(v, device), ints(starts, device), rows=ints(rows, device))
    full_k, full_v = (np.concatenate((x, np.zeros((batch, 92, heads, dim), np.float16)), 1) for x in (k, v))
    full_k[9] = np.concatenate((k0[9], k[9]))
    full_v[9] = np.concatenate((v0[9], v[9]))
    lengths = [rows[b] if good[b] and b < 9 else 0 for b in range(9)] + [192]
    want = expect(0x2A, full_k, full_v, lengths, capacity, format)
    got = buffers(cache)
    want[4][9, :, 1], want[5][9, :, 1] = got[4][9, :, 1], got[5][9, :, 1]   # block 1 was there, nobody needs it any more
    for name, g, w in zip(('kc', 'vc', 'ks', 'vs', 'kt', 'vt'), got, want):
        same(g, w)
    for b in (2, 3, 4, 5, 6, 7, 8):
        for g, f in zip(got, first):
            same(g[b], f[b])


@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_append_borders(device, format):
    """Ties, subnormals, the largest values, blocks of zeros and of one value."""
    announce('kv append borders', format)
    dim, blocks = 64, 8
    rng = np.random.default_rng(9)
    k = np.zeros((1, 64 * blocks, 1, dim), np.float16)
    v = np.zeros_like(k)
    def block(x, i, values):
        x[0, 64 * i:64 * i + 64, 0] = values.reshape(64, dim).astype(np.float16)
    halves = np.arange(64 * dim) % 255 - 127
    block(k, 0, (halves + 0.5 * (np.arange(64 * dim) % 2)).clip(-127, 127))              # half steps of a top of 127
    block(v, 0, np.ldexp(1.0, -24) * rng.integers(-5, 6, 64 * dim))                        # subnormals, top 5 steps
    block(k, 1, np.where(rng.random(64 * dim) < .5, 65504.0, -65504.0))
    block(v, 1, np.full(64 * dim, np.ldexp(1.0, -24)))
    block(k, 3, rng.choice([1.0, 0.5, -0.5, 0.25, 63.5 / 127, 0.0, -0.0], 64 * dim))       # exact ties at top / 2
    block(v, 3, rng.standard_normal(64 * dim) * np.exp2(rng.integers(-20, 12, 64 * dim)))
    for i in range(4, blocks):                                                             # every fp16 mantissa by every top
        top = float(np.float16(1 + rng.integers(0, 1024) / 1024))
        x = rng.choice([-1, 1], 64 * dim) * (rng.integers(0, 2048, 64 * dim) / 1024 * np.exp2(rng.integers(-11, 1, 64 * dim)))
        x = np.clip(x, -top, top)
        x[0] = top
        block(k, i, x)
        block(v, i, x[::-1].copy())
    cache = fresh(device, 1, 1, 64 * blocks, dim, format)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0], device))
    want = expect(0x35, k, v, [64 * blocks], 64 * blocks, format)
    got = buffers(cache)
    for i in range(4):   # -0.0 and 0.0 are different e4m3 bytes of one value
        if format == 'fp8' and i < 2:
            g, w = (np.where(x == 0x80, 0, x) for x in (got[i], want[i]))
        else:
            g, w = got[i], want[i]
        same(g, w)
    keys, values = lb.kv_read(cache, ints([64 * blocks], device))
    assert bool(torch.isfinite(keys).all() and torch.isfinite(values).all())


@pytest.mark.parametrize('dim', [64, 128])
def test_append_rotates_and_takes_strides(device, dim):
    """RoPE as in the fp16 cache's kernels; k and v as slices of one projection, transposed, or at odd addresses."""
    announce('kv append rotate', dim)
    batch, heads, seq, capacity, start = 2, 2, 75, 256, 30
    g = np.random.default_rng(5)
    angle = g.uniform(-7, 7, (capacity, dim)).astype(np.float32)
    cos, sin = np.cos(angle).astype(np.float16), np.sin(angle).astype(np.float16)
    both = rows_of(6, batch, seq, 2 * heads, dim)
    early = rows_of(7, batch, start, 2 * heads, dim)
    k, v = both[:, :, :heads], both[:, :, heads:]
    d = dev(both, device)
    kinds = {'slices': (d[:, :, :heads], d[:, :, heads:]),
             'transposed': tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (d[:, :, :heads], d[:, :, heads:])),
             'odd': tuple(torch.cat((t.new_zeros(3), t.reshape(-1)))[3:].view(t.shape) for t in (d[:, :, :heads], d[:, :, heads:])),
             'by dim': tuple(t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for t in (d[:, :, :heads], d[:, :, heads:]))}
    turn = lambda x, at: ko.rotate(x, cos[at:at + x.shape[1], None], sin[at:at + x.shape[1], None])
    full_k = np.concatenate((turn(early[:, :, :heads], 0), turn(k, start)), 1)
    full_v = np.concatenate((early[:, :, heads:], v), 1)
    want = expect(0x35, full_k, full_v, [start + seq] * batch, capacity, 'int8')
    for kind, (kd, vd) in kinds.items():
        cache = fresh(device, batch, heads, capacity, dim, 'int8')
        tables = dict(cos=dev(cos, device), sin=dev(sin, device))
        e = dev(early, device)
        lb.kv_append(cache, e[:, :, :heads], e[:, :, heads:], ints([0] * batch, device), **tables)
        lb.kv_append(cache, kd, vd, ints([start] * batch, device), **tables)
        for g_, w in zip(buffers(cache), want):
            same(g_, w)


def test_positions_can_be_taken_back(device):
    """Rows behind a position that is taken back are overwritten as if they had never been, into the block before the
    open one as well."""
    announce('kv taken back')
    dim, heads, capacity = 64, 1, 256
    k, v = rows_of(8, 1, 200, heads, dim), rows_of(9, 1, 200, heads, dim)
    other = rows_of(10, 1, 70, heads, dim)
    cache = fresh(device, 1, heads, capacity, dim, 'int8')
    add = lambda a, b, at: lb.kv_append(cache, dev(a, device), dev(b, device), ints([at], device))
    add(k[:, :130], v[:, :130], 0)
    add(other, other, 130)              # drafted up to slot 200, then rejected back to 135 (block 2 was closed meanwhile)
    add(k[:, 135:150], v[:, 135:150], 135)
    full_k, full_v = k.copy(), v.copy()
    full_k[:, 130:135], full_v[:, 130:135] = other[:, :5], other[:, :5]
    keys, values = lb.kv_read(cache, ints([150], device), count=150)
    for got, rows in ((keys, full_k), (values, full_v)):
        want = ko.read(rows[0, :150, 0], 'int8')
        same(got.cpu().numpy()[0, 0], want)


# ---------------------------------------------------------------- read
@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('dim', [64, 128])
def test_read_gives_the_held_values(device, format, dim):
    announce('kv read', format, dim)
    lengths, heads, capacity = [0, 1, 64, 100, 129, 320], 2, 320
    batch = len(lengths)
    k, v = rows_of(11, batch, capacity, heads, dim), rows_of(12, batch, capacity, heads, dim, spread=.1)
    cache = fresh(device, batch, heads, capacity, dim, format)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints(lengths, device))
    for start, count in ((0, None), (0, 1), (63, 2), (70, 100), (319, 1)):
        n = capacity - start if count is None else count
        # outputs inside a larger buffer: every other head, rows apart
        wide = [torch.full((batch, heads * 2, n, dim + 8), 7.0, dtype=torch.float16, device=device) for _ in range(2)]
        outs = [w[:, ::2, :, :dim] for w in wide]
        got = lb.kv_read(cache, ints(lengths, device), start=start, count=count, keys=outs[0], values=outs[1])
        assert got[0] is outs[0] and got[1] is outs[1]
        for w, rows in zip(wide, (k, v)):
            exp = np.full(w.shape, 7.0, np.float16)
            for b in range(batch):
                for h in range(heads):
                    part = ko.read(rows[b, :lengths[b], h], format)[start:start + n]
                    exp[b, 2 * h, :len(part), :dim] = part
            same(w.cpu().numpy(), exp)
    bad = ints([-1, 400, 64, 100, 129, 320], device)
    keys, values = lb.kv_read(cache, bad)
    assert bool(keys[:2].isnan().all() and values[:2].isnan().all()) and not bool(keys[2:].isnan().any())


# ---------------------------------------------------------------- attention
def bound(out, weight, reach, n, dim, top):
    """The header's sum: out, weight [s, D], reach [s], n slots, top the largest |v|."""
    half = 2.0 ** -11
    a = np.maximum(weight, np.abs(out))
    return (a * (2 * half + 2 * (dim + 8) * 2.0 ** -24 * reach[:, None] + n * 2.0 ** -24) + 2 * n * 2.0 ** -25 * top
            + half * np.abs(out) + 2.0 ** -25)


def check_attention(got, q, k, v, starts, rows, format, scale, kv_heads, rotated=None):
    """got, q [b, s, heads, D]; k, v [b, slots, kv_heads, D]: every row against the oracle; returns the worst share of the
    bound that was used."""
    got, worst = got.float().cpu().numpy().astype(np.float64), 0.0
    group = q.shape[2] // kv_heads
    for b in range(q.shape[0]):
        n = starts[b] + rows[b]
        for h in range(kv_heads):
            kr, vr = ko.poison(k[b, :n, h], v[b, :n, h])
            kh, vh = ko.held(kr, format), ko.held(vr, format)
            for e in range(group):
                head = h * group + e
                out, weight, reach = ko.attend(q[b, :rows[b], head], kh, vh, starts[b], scale)
                limit = bound(out, weight, reach, n, q.shape[3], np.abs(vh[np.isfinite(vh)]).max(initial=0.0))
                off = np.abs(got[b, :rows[b], head] - out)
                assert np.array_equal(np.isnan(out), np.isnan(got[b, :rows[b], head])), (b, head)
                fine = np.isfinite(out)
                if fine.any():
                    worst = max(worst, float((off[fine] / limit[fine]).max()))
                assert (off[fine] <= limit[fine]).all(), (b, head, float((off[fine] / limit[fine]).max()))
    return worst


# heads, kv_heads, dim, seq, starts
SHAPES = [
    (9, 3, 64, 1, (0, 1, 62, 63, 64, 65, 127, 128, 200, 511)),
    (32, 8, 128, 1, (0, 63, 64, 333)),
    (8, 8, 64, 1, (5, 700)),
    (16, 1, 128, 1, (129,)),
    (20, 1, 64, 1, (64, 90)),
    (33, 1, 64, 1, (100, 63)),
    (15, 5, 64, 5, (0, 60, 62, 64, 190)),
    (4, 2, 128, 3, (0, 61, 126)),
    (6, 2, 64, 17, (0, 50, 111)),
    (9, 3, 64, 75, (0, 10, 64, 130)),
    (4, 1, 128, 70, (0, 3)),
    (2, 1, 64, 200, (0, 77)),
]


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('shape', SHAPES, ids=['h%d-kv%d-d%d-s%d' % s[:4] for s in SHAPES])
def test_attention_matches_the_definition(device, format, shape):
    heads, kv_heads, dim, seq, starts = shape
    announce('kv attention', format, shape)
    batch, total = len(starts), max(starts) + seq
    capacity = (total + 63) // 64 * 64 + 128
    k, v = rows_of(20, batch, total, kv_heads, dim), rows_of(21, batch, total, kv_heads, dim, spread=.3)
    q = rows_of(22, batch, seq, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)   # NaN wherever nothing is held
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints([s + seq for s in starts], device))
    scale = dim ** -0.5
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device))
    worst = check_attention(got, q, k, v, starts, [seq] * batch, format, scale, kv_heads)
    print(f'[kv attention] {format} {shape[:4]}: {worst:.2f} of the bound', flush=True)


@pytest.mark.parametrize('format,dim', [('int8', 64), ('fp8', 128)])
def test_attention_long(device, format, dim):
    """Thousands of slots in many parts."""
    announce('kv attention long', format, dim)
    starts, heads, kv_heads, seq = [5000, 0, 2111, 4095], 4, 2, 2
    batch, capacity = len(starts), 5120
    k, v = rows_of(30, batch, 5002, kv_heads, dim), rows_of(31, batch, 5002, kv_heads, dim)
    q = rows_of(32, batch, seq, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints([s + seq for s in starts], device))
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device))
    worst = check_attention(got, q, k, v, starts, [seq] * batch, format, dim ** -0.5, kv_heads)
    print(f'[kv attention] long {format}: {worst:.2f} of the bound', flush=True)


@pytest.mark.parametrize('seq,heads', [(3, 6), (90, 6), (1, 2)])
def test_attention_ragged_rows(device, seq, heads):
    """Padded batches: out rows behind a sequence's own are left as they were, a sequence that lies outside the capacity
    is NaN, and one of no rows is untouched."""
    announce('kv attention ragged', seq, heads)
    kv_heads, dim, capacity = 2, 64, 256
    starts, rows = [0, 100, 64, -5, 255, 7], [seq, 1, 0, 1, 2, seq]
    if seq == 1:
        rows[4] = 2          # more than seq: refused on the device
    batch = len(starts)
    good = [0 <= s and r <= seq and s + r <= capacity for s, r in zip(starts, rows)]
    k, v = rows_of(40, batch, capacity, kv_heads, dim), rows_of(41, batch, capacity, kv_heads, dim)
    q = rows_of(42, batch, seq, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, 'int8', fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device),
                 rows=ints([s + r if g else 0 for s, r, g in zip(starts, rows, good)], device))
    wide = torch.full((batch, seq, 2 * heads, dim), 3.0, dtype=torch.float16, device=device)
    out = wide[:, :, :heads]
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device), rows=ints(rows, device), out=out)
    assert got is out and bool((wide[:, :, heads:] == 3).all())
    for b in range(batch):
        if not good[b]:
            assert bool(out[b].isnan().all()), b
        else:
            assert bool((out[b, rows[b]:] == 3).all()), b
            check_attention(out[b:b + 1, :max(1, rows[b])], q[b:b + 1], k[b:b + 1], v[b:b + 1], [starts[b]], [rows[b]], 'int8',
                            dim ** -0.5, kv_heads)


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('seq', [1, 6, 80])
def test_attention_appends_and_rotates(device, format, seq):
    """k and v in the same call, RoPE of q and k, strided q and out: the same as the calls one after the other."""
    announce('kv attention append', format, seq)
    batch, heads, kv_heads, dim, capacity, starts = 3, 6, 2, 64, 320, [63, 0, 130]
    g = np.random.default_rng(50)
    angle = g.uniform(-7, 7, (capacity + 5, dim)).astype(np.float32)
    cos, sin = np.cos(angle).astype(np.float16), np.sin(angle).astype(np.float16)
    both = rows_of(51, batch, seq, heads + 2 * kv_heads, dim)
    d = dev(both, device)
    q, k, v = d[:, :, :heads], d[:, :, heads:heads + kv_heads], d[:, :, heads + kv_heads:]
    old_k, old_v = rows_of(52, batch, 130, kv_heads, dim), rows_of(53, batch, 130, kv_heads, dim)
    tables = dict(cos=dev(cos, device), sin=dev(sin, device))
    cache = fresh(device, batch, kv_heads, capacity, dim, format)
    lb.kv_append(cache, dev(old_k, device), dev(old_v, device), ints([0] * batch, device), rows=ints(starts, device), **tables)
    twin = cache.clone()
    out = torch.empty((batch, heads, seq, dim), dtype=torch.float16, device=device).transpose(1, 2)
    lb.kv_attention(q, cache, ints(starts, device), k=k, v=v, out=out, scale=0.2, **tables)
    lb.kv_append(twin, k, v, ints(starts, device), **tables)
    apart = lb.kv_attention(q, twin, ints(starts, device), scale=0.2, **tables)
    assert torch.equal(out, apart)
    for a, b in zip(cache.tensors(), twin.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    full_k, full_v, rq = [], [], []
    for b, s in enumerate(starts):
        rows = np.concatenate((old_k[b, :s], both[b, :, heads:heads + kv_heads]))
        full_k.append(np.concatenate((ko.rotate(rows, cos[:s + seq, None], sin[:s + seq, None]), np.zeros((130 - s, kv_heads, dim), np.float16))))
        full_v.append(np.concatenate((old_v[b, :s], both[b, :, heads + kv_heads:], np.zeros((130 - s, kv_heads, dim), np.float16))))
        rq.append(ko.rotate(both[b, :, :heads], cos[s:s + seq, None], sin[s:s + seq, None]))
    check_attention(out, np.stack(rq), np.stack(full_k), np.stack(full_v), starts, [seq] * batch, format, float(np.float32(0.2)), kv_heads)


@pytest.mark.parametrize('seq', [4, 100])
def test_attention_keeps_what_is_not_finite_to_the_rows_that_see_it(device, seq):
    """Rows before a NaN or an infinity (in the open block, by slot) do not notice it, rows behind it are NaN; a block with
    one is NaN to every row that sees some of it."""
    announce('kv attention not finite', seq)
    heads, kv_heads, dim, capacity = 4, 2, 64, 256
    cases = [('k', np.inf), ('v', np.nan), ('v', -np.inf), ('k', np.nan)]
    starts = [128 if seq == 4 else 100] * len(cases)
    bad = starts[0] + (2 if seq == 4 else 95)        # in the open block: slots 192 .. 199, or 128 .. 131
    batch, total = len(cases), starts[0] + seq
    k, v, q = rows_of(60, batch, total, kv_heads, dim), rows_of(61, batch, total, kv_heads, dim), rows_of(62, batch, seq, heads, dim)
    for b, (side, value) in enumerate(cases):
        (k if side == 'k' else v)[b, bad, 1, 7] = value
    cache = fresh(device, batch, kv_heads, capacity, dim, 'int8', fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device))
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device))
    at = bad - starts[0]
    assert not bool(got[:, :, :2].isnan().any()) and not bool(got[:, :at, 2:].isnan().any()) and bool(got[:, at:, 2:].isnan().all())
    check_attention(got, q, k, v, starts, [seq] * batch, 'int8', dim ** -0.5, kv_heads)
    # the block is closed: every row that sees a slot of it
    more = 64 - total % 64
    lb.kv_append(cache, dev(k[:, :more], device), dev(v[:, :more], device), ints([total] * batch, device))
    first = bad // 64 * 64
    q2 = dev(rows_of(63, batch, total + more - first + 3, heads, dim), device)
    got = lb.kv_attention(q2, cache, ints([first - 3] * batch, device))
    assert not bool(got[:, :3].isnan().any()) and bool(got[:, 3:, 2:].isnan().all()) and not bool(got[:, :, :2].isnan().any())


def test_attention_extremes(device):
    """One score far above the others late or early, equal scores, scale 0, all-zero values, scores of +-1e4."""
    announce('kv attention extremes')
    heads, kv_heads, dim, capacity, n = 3, 1, 64, 512, 500
    rng = np.random.default_rng(70)
    k, v = rows_of(71, 4, n, kv_heads, dim), rows_of(72, 4, n, kv_heads, dim)
    k[0, 490], k[0, 3] = 40.0, -40.0
    k[1] = k[1, :1]
    v[2] = 0
    k[3] *= 60
    q = rows_of(73, 4, 1, heads, dim)
    q[0] = np.abs(q[0])
    cache = fresh(device, 4, kv_heads, capacity, dim, 'int8', fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * 4, device))
    starts = [n - 1] * 4
    for scale in (dim ** -0.5, 0.0, 1.0):
        got = lb.kv_attention(dev(q, device), cache, ints(starts, device), scale=scale)
        check_attention(got, q, k, v, starts, [1] * 4, 'int8', scale, kv_heads)


def test_a_run_as_it_is_used(device):
    """Prompt, decode steps in a captured graph whose positions advance on the device, drafts taken back, a read: at each
    stage against the oracle, the captured steps (replayed, with eager work between) against eager ones."""
    announce('kv run')
    batch, heads, kv_heads, dim, capacity, prompt, steps = 2, 6, 2, 64, 256, [50, 61], 20
    k, v = rows_of(80, batch, 200, kv_heads, dim), rows_of(81, batch, 200, kv_heads, dim)
    q = rows_of(82, batch, 200, heads, dim)
    kd, vd, qd = (dev(t, device) for t in (k, v, q))
    cache = lb.QuantizedKVCache.empty(batch, kv_heads, capacity, format='fp8', device=device)
    position = ints([0, 0], device)
    rows = ints(prompt, device)
    got = lb.kv_attention(qd[:, :64], cache, position, k=kd[:, :64], v=vd[:, :64], rows=rows)
    check_attention(got, q, k, v, [0, 0], prompt, 'fp8', dim ** -0.5, kv_heads)
    position += rows
    start = position.clone()
    # a step: the token rows at each sequence's position, the call, position + 1
    qs, ks, vs = (torch.zeros((batch, 1, t.shape[2], dim), dtype=torch.float16, device=device) for t in (qd, kd, vd))
    out = torch.zeros_like(qs)
    call = lb.PreparedKVAttention(qs, cache, position, out, k=ks, v=vs)
    lane = torch.arange(batch, device=device)

    def step():
        qs.copy_(qd[lane, position][:, None])
        ks.copy_(kd[lane, position][:, None])
        vs.copy_(vd[lane, position][:, None])
        call.run()
        position.add_(1)
    twin = cache.clone()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    for t, s in zip(cache.tensors(), twin.tensors()):
        t.view(torch.uint8).copy_(s.view(torch.uint8))
    position.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(steps):
        graph.replay()
        at = start + i
        eager = lb.kv_attention(qd[lane, at][:, None], twin, at, k=kd[lane, at][:, None], v=vd[lane, at][:, None])
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
        now = [p + i for p in prompt]
        check_attention(out, np.stack([q[b, now[b]:now[b] + 1] for b in range(batch)]), k, v, now, [1] * batch, 'fp8', dim ** -0.5, kv_heads)
    for a, b in zip(cache.tensors(), twin.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # five drafts, of which two and none are kept; then the sequences go on from there
    junk = rows_of(83, batch, 5, kv_heads, dim)
    lb.kv_attention(qd[:, :5], cache, position, k=dev(junk, device), v=dev(junk, device))
    position += ints([2, 0], device)
    held = [p + steps for p in prompt]
    k[0, held[0]:held[0] + 2], v[0, held[0]:held[0] + 2] = junk[0, :2], junk[0, :2]
    starts = [held[0] + 2, held[1]]
    nk, nv = (np.stack([t[b, starts[b]:starts[b] + 30] for b in range(batch)]) for t in (k, v))
    nq = rows_of(84, batch, 30, heads, dim)
    got = lb.kv_attention(dev(nq, device), cache, position, k=dev(nk, device), v=dev(nv, device))
    check_attention(got, nq, k, v, starts, [30] * batch, 'fp8', dim ** -0.5, kv_heads)
    lengths = [s + 30 for s in starts]
    keys, values = lb.kv_read(cache, ints(lengths, device))
    for b in range(batch):
        for h in range(kv_heads):
            for g, rows_ in ((keys, k), (values, v)):
                same(g[b, h, :lengths[b]].cpu().numpy(), ko.read(rows_[b, :lengths[b], h], 'fp8'))
                assert not bool(g[b, h, lengths[b]:].any())


def test_two_calls_at_once(device):
    """Calls on two streams, each with its own cache and (eager) workspace."""
    announce('kv two streams')
    heads, kv_heads, dim, n = 4, 2, 128, 3000
    made = []
    for i in range(2):
        k, v = rows_of(90 + i, 1, n, kv_heads, dim), rows_of(92 + i, 1, n, kv_heads, dim)
        cache = lb.QuantizedKVCache.empty(1, kv_heads, n, head_dim=dim, device=device)
        lb.kv_append(cache, dev(k, device), dev(v, device), ints([0], device))
        q = dev(rows_of(94 + i, 1, 1, heads, dim), device)
        made.append((cache, q, ints([n - 1], device)))
    want = [lb.kv_attention(q, cache, at) for cache, q, at in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lb.kv_attention(made[i][1], made[i][0], made[i][2]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_caches_past_32_bit_offsets(device):
    """Codes of more than 4 GiB: the last sequence is the same as in a cache of its own."""
    announce('kv past 32 bits')
    batch, kv_heads, dim, capacity, n = 3, 8, 128, 3 << 19, 200
    cache = lb.QuantizedKVCache.empty(batch, kv_heads, capacity, head_dim=dim, format='fp8', device=device)
    assert cache.key_codes.numel() > 2 ** 32
    alone = lb.QuantizedKVCache.empty(1, kv_heads, 256, head_dim=dim, format='fp8', device=device)
    k, v, q = (dev(rows_of(s, 1, n, h, dim), device) for s, h in ((95, kv_heads), (96, kv_heads), (97, 2 * kv_heads)))
    many = lambda t: t.expand(batch, *t.shape[1:])
    lb.kv_append(cache, many(k), many(v), ints([0] * batch, device), rows=ints([0, 0, n], device))
    lb.kv_append(alone, k, v, ints([0], device))
    at = ints([0, 0, n - 1], device)
    got = lb.kv_attention(many(q[:, -1:]), cache, at, rows=ints([0, 0, 1], device))
    want = lb.kv_attention(q[:, -1:], alone, at[2:])
    check_attention(got[2:], *(t.cpu().numpy() for t in (q[:, -1:], k, v)), [n - 1], [1], 'fp8', dim ** -0.5, kv_heads)
    check_attention(want, *(t.cpu().numpy() for t in (q[:, -1:], k, v)), [n - 1], [1], 'fp8', dim ** -0.5, kv_heads)
    # far slots of the last sequence: its last block
    far = capacity - 64
    lb.kv_append(cache, many(k[:, :64]), many(v[:, :64]), ints([far] * batch, device), rows=ints([0, 0, 64], device))
    a, b = lb.kv_read(cache, ints([0, 0, capacity], device), start=far, count=64)
    for t, rows in ((a, k), (b, v)):
        for h in (0, kv_heads - 1):
            same(t[2, h].cpu().numpy(), ko.read(rows[0, :64, h].cpu().numpy(), 'fp8'))


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('dim,seq', [(64, 1), (64, 60), (128, 45)])
def test_attention_over_blocks_of_very_different_scales(device, format, dim, seq):
    """Values from block to block 1e-6 to 2e3 in size, blocks of zeros first and in between, keys of zeros."""
    announce('kv attention scales', format, dim, seq)
    heads, kv_heads, capacity, total = 4, 1, 1024, 1000
    sizes = [0, 1e-6, 1, 1e-3, 0, 6e2, 50, 1e-5, 2, 9, 0.3, 2e3, 1, 1e-6, 7, 1]
    k, v = rows_of(100, 3, total, kv_heads, dim), rows_of(101, 3, total, kv_heads, dim).astype(np.float64)
    for i, size in enumerate(sizes):
        v[:, 64 * i:64 * i + 64] *= size
    v[1] = np.abs(v[1, ::-1])
    k[2, 128:320] = 0
    v = v.astype(np.float16)
    assert np.isfinite(v).all()
    starts = [total - seq, 500, 290]
    q = rows_of(102, 3, seq, heads, dim)
    cache = fresh(device, 3, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * 3, device), rows=ints([s + seq for s in starts], device))
    got = lb.kv_attention(dev(q, device), cache, ints(starts, device))
    worst = check_attention(got, q, k, v, starts, [seq] * 3, format, dim ** -0.5, kv_heads)
    print(f'[kv attention] scales {format} {dim} {seq}: {worst:.2f} of the bound', flush=True)


def test_attention_of_many_sequences(device):
    """More sequences than a workgroup has threads: short ones, some of no rows, some outside the capacity, then long."""
    announce('kv attention many')
    batch, heads, kv_heads, dim, capacity = 700, 2, 1, 64, 192
    rng = np.random.default_rng(110)
    starts = [int(x) for x in rng.integers(0, capacity, batch)]
    rows = [int(x) for x in rng.integers(0, 3, batch) > 0]
    starts[5], starts[300], starts[699], rows[699] = -1, capacity, capacity - 1, 1
    rows[300] = 1
    good = [0 <= s and s + r <= capacity for s, r in zip(starts, rows)]
    k, v = rows_of(111, batch, capacity, kv_heads, dim), rows_of(112, batch, capacity, kv_heads, dim)
    q = rows_of(113, batch, 1, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, 'int8', fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device),
                 rows=ints([s + r if g else 0 for s, r, g in zip(starts, rows, good)], device))
    out = torch.full((batch, 1, heads, dim), 3.0, dtype=torch.float16, device=device)
    lb.kv_attention(dev(q, device), cache, ints(starts, device), rows=ints(rows, device), out=out)
    for b in range(batch):
        if not good[b]:
            assert bool(out[b].isnan().all()), b
        elif rows[b] == 0:
            assert bool((out[b] == 3).all()), b
        else:
            check_attention(out[b:b + 1], q[b:b + 1], k[b:b + 1], v[b:b + 1], [starts[b]], [1], 'int8', dim ** -0.5, kv_heads)


@pytest.mark.parametrize('batch', [2, 33, 64, 65])
def test_attention_of_unequal_lengths(device, batch):
    """Batches on both sides of what one wave ranks, from one slot to thousands, some without rows: every sequence is
    found once, whole, whichever workgroups share it."""
    announce('kv attention unequal', batch)
    heads, kv_heads, dim, capacity = 3, 1, 64, 2560
    rng = np.random.default_rng(120 + batch)
    starts = [int(x) for x in rng.choice([0, 63, 64, 200, 700, 1500, 2500], batch)]
    rows = [int(x) for x in rng.integers(0, 5, batch) > 0]
    starts[-1], rows[-1], starts[0], rows[0] = 2559, 1, 0, 1
    k, v = rows_of(121, batch, capacity, kv_heads, dim), rows_of(122, batch, capacity, kv_heads, dim, spread=.3)
    q = rows_of(123, batch, 1, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, 'fp8', fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device),
                 rows=ints([s + r for s, r in zip(starts, rows)], device))
    out = torch.full((batch, 1, heads, dim), 3.0, dtype=torch.float16, device=device)
    lb.kv_attention(dev(q, device), cache, ints(starts, device), rows=ints(rows, device), out=out)
    some = [b for b in range(batch) if rows[b]]
    assert bool((out[[b for b in range(batch) if not rows[b]]] == 3).all())
    worst = check_attention(out[some], q[some], k[some], v[some], [starts[b] for b in some], [1] * len(some), 'fp8',
                            dim ** -0.5, kv_heads)
    print(f'[kv attention] unequal {batch}: {worst:.2f} of the bound', flush=True)


def test_two_graphs_of_plain_calls(device):
    """kv_attention and kv_append captured as they are, twice; replays of both graphs at once and eager calls between
    them give what the eager calls gave."""
    announce('kv two graphs')
    heads, kv_heads, dim, n = 4, 2, 64, 4000
    made, graphs = [], []
    for i in range(2):
        k, v = rows_of(130 + i, 2, n, kv_heads, dim), rows_of(132 + i, 2, n, kv_heads, dim)
        cache = lb.QuantizedKVCache.empty(2, kv_heads, n + 64, head_dim=dim, device=device)
        at = ints([n - 65, 100], device)
        lb.kv_append(cache, dev(k[:, :n - 65], device), dev(v[:, :n - 65], device), ints([0, 0], device), rows=at)
        q = dev(rows_of(134 + i, 2, 1, heads, dim), device).expand(2, 3, heads, dim)[:, :1]
        made.append((cache, q, at, dev(k[:, n - 65:n - 64], device), dev(v[:, n - 65:n - 64], device)))
    call = lambda c, q, at, k, v: (lb.kv_append(c, k, v, at), lb.kv_attention(q, c, at, k=k, v=v))[1]
    want = [call(*m) for m in made]
    torch.cuda.synchronize()
    for m in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*m)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    for _ in range(4):
        for (graph, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, out), m, w in zip(graphs, made, want):
            assert torch.equal(out, w) and torch.equal(call(*m), w)
        torch.cuda.synchronize()


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('heads,kv_heads,dim,seq', [(8, 2, 128, 1), (20, 1, 128, 1), (20, 1, 64, 1), (32, 1, 128, 1), (4, 1, 128, 5),
                                                    (8, 1, 128, 4), (10, 2, 128, 6), (16, 2, 64, 4)])
def test_attention_of_wide_groups_appends(device, format, heads, kv_heads, dim, seq):
    """Up to 32 rows of a KV head, either head size, rows that fill a block in the same call, short and split sequences."""
    announce('kv attention wide groups', format, heads, kv_heads, dim, seq)
    starts, capacity = [63, 0, 130, 2879, 255, 64 - seq], 2944
    batch, total = len(starts), capacity
    k, v = rows_of(140, batch, total, kv_heads, dim), rows_of(141, batch, total, kv_heads, dim, spread=.3)
    q = rows_of(142, batch, seq, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device), rows=ints(starts, device))
    new = [dev(np.stack([x[b, s:s + seq] for b, s in enumerate(starts)]), device) for x in (k, v)]
    twin = cache.clone()
    out = lb.kv_attention(dev(q, device), cache, ints(starts, device), k=new[0], v=new[1])
    lb.kv_append(twin, new[0], new[1], ints(starts, device))
    assert torch.equal(out, lb.kv_attention(dev(q, device), twin, ints(starts, device)))
    for a, b in zip(cache.tensors(), twin.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    worst = check_attention(out, q, k, v, starts, [seq] * batch, format, dim ** -0.5, kv_heads)
    print(f'[kv attention] wide groups {format} {heads}/{kv_heads} {dim} {seq}: {worst:.2f} of the bound', flush=True)


@pytest.mark.parametrize('format', ['int8', 'fp8'])
@pytest.mark.parametrize('heads,kv_heads,dim,seq', [(3, 1, 64, 70), (2, 1, 128, 133), (33, 1, 128, 1), (8, 2, 64, 40),
                                                    (1, 1, 64, 129), (1, 1, 128, 131)])
def test_attention_of_chunks_in_parts(device, format, heads, kv_heads, dim, seq):
    """Chunks of a prompt behind thousands of slots beside short ones and a padded one: a tile's slots in many parts."""
    announce('kv attention chunks', format, heads, kv_heads, dim, seq)
    starts, capacity = [2500, 0, 1090], 2688
    rows = [seq, seq, max(1, seq // 2)]
    batch = len(starts)
    k, v = rows_of(150, batch, capacity, kv_heads, dim), rows_of(151, batch, capacity, kv_heads, dim, spread=.3)
    q = rows_of(152, batch, seq, heads, dim)
    cache = fresh(device, batch, kv_heads, capacity, dim, format, fill=0x7F)
    lb.kv_append(cache, dev(k, device), dev(v, device), ints([0] * batch, device),
                 rows=ints([s + r for s, r in zip(starts, rows)], device))
    out = torch.full((batch, seq, heads, dim), 3.0, dtype=torch.float16, device=device)
    lb.kv_attention(dev(q, device), cache, ints(starts, device), rows=ints(rows, device), out=out)
    assert bool((out[2, rows[2]:] == 3).all())
    worst = check_attention(out, q, k, v, starts, rows, format, dim ** -0.5, kv_heads)
    print(f'[kv attention] chunks {format} {heads}/{kv_heads} {dim} {seq}: {worst:.2f} of the bound', flush=True)


@pytest.mark.parametrize('format,dim,seed', [('int8', 64, 0), ('fp8', 64, 1), ('int8', 128, 2)])
def test_positions_taken_back_again_and_again(device, format, dim, seed):
    """Appends of one to 150 rows and positions taken back, as far as the header allows, over and over: to the start of any
    block, and into a block whose rows the ring has yet.  What is held is at every stage what the rows say, bit for bit."""
    announce('kv taken back again', format, dim, seed)
    batch, heads, capacity, steps = 3, 1, 640, 60
    rng = np.random.default_rng(160 + seed)
    cache = fresh(device, batch, heads, capacity, dim, format, fill=0x7F)
    k, v = (np.zeros((batch, capacity, heads, dim), np.float16) for _ in range(2))
    length, most = [0] * batch, [{} for _ in range(batch)]   # most[b][i]: slots held at the most since slot 64 i was appended
    inside = 0
    for step in range(steps):
        rows, seq = [], 150
        for b in range(batch):
            if length[b] and rng.random() < 0.6:             # taken back
                may = [p for p in range(length[b] + 1) if p % 64 == 0 or most[b][p // 64] < 64 * (p // 64 + 2)]
                to = int(rng.choice(may[-100:])) if rng.random() < 0.8 else int(rng.choice(may))
                inside += to % 64 != 0 and to // 64 < length[b] // 64
                length[b] = to
            rows.append(min(capacity - length[b], int(rng.choice([0, 1, 2, rng.integers(1, 20), rng.integers(1, seq + 1)]))))
        new = [rows_of(1000 * seed + 2 * step + i, batch, seq, heads, dim) for i in range(2)]
        lb.kv_append(cache, dev(new[0], device), dev(new[1], device), ints(length, device), rows=ints(rows, device))
        for b in range(batch):
            start, end = length[b], length[b] + rows[b]
            for t, x in zip((k, v), new):
                t[b, start:end] = x[b, :rows[b]]
            for i in range((start + 63) // 64, (end + 63) // 64):
                most[b][i] = 0                               # its first slot is among these rows
            most[b] = {i: max(n, end) for i, n in most[b].items()}
            length[b] = end
        got = lb.kv_read(cache, ints(length, device))
        for g, t in zip(got, (k, v)):
            g = g.cpu().numpy()
            for b in range(batch):
                same(g[b, 0, :length[b]], ko.read(t[b, :length[b], 0], format))
    assert inside >= 5, inside
