"""lb_rotary against its definition in 64 bits.

Tolerance, in parts of |a| + |b| of a value's pair times |scale|: the part of a turn, at most 1/2, is rounded to 32 bits
(pi 2^-24 of the angle), the sine and cosine are right to 2 ulp (2^-23 each), their product with the scale, the two products
and their sum are rounded (4 times 2^-24 at the most): below 2^-20 in all.  The angle in 64 bits is off by three roundings of
itself, 2^-51 |position frequency|.  Then the output's own half step, and half the type's smallest one.
"""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import serve_oracle as so

pytestmark = pytest.mark.gpu
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
SMALLEST = {'fp16': 2.0 ** -24, 'bf16': 2.0 ** -133, 'fp32': 2.0 ** -149}


def make(device, type, batch, seq, heads, dim, seed=0, gap=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((batch, seq, heads + gap, dim), generator=g).to(TYPES[type]).to(device)[:, :, :heads]


def check(got, x, position, rotary, type, back=False):
    f = rotary.frequencies.cpu().numpy()
    x64 = x.double().cpu().numpy()
    want = so.turned(x64, position, f, rotary.pairs, rotary.scale, back)
    far = 2.0 ** -51 * np.abs(np.asarray(position, np.float64)).max() * np.abs(f).max()
    part = so.partner_sizes(x64, len(f), rotary.pairs) * abs(rotary.scale) * (2.0 ** -20 + far)
    bound = part + torch.finfo(TYPES[type]).eps / 2 * (np.abs(want) + part) + SMALLEST[type] / 2
    worst = float(np.max(np.abs(got.double().cpu().numpy() - want) / bound))
    assert worst <= 1, worst               # (a NaN fails too)


def rows_at(first, seq):
    return np.asarray(first)[:, None] + np.arange(seq)


CASES = [
    # type, batch, seq, heads, k_heads, dim, part, pairs
    ('fp16', 1, 1, 9, 3, 64, 64, 'half'),
    ('fp16', 3, 5, 9, 3, 64, 32, 'neighbours'),
    ('bf16', 2, 33, 32, 8, 128, 128, 'half'),
    ('bf16', 2, 7, 4, 1, 128, 40, 'half'),
    ('bf16', 2, 7, 4, 1, 128, 40, 'neighbours'),
    ('fp32', 1, 11, 5, 5, 128, 128, 'neighbours'),
    ('fp32', 2, 3, 8, 8, 64, 2, 'half'),
    ('fp16', 2, 3, 3, 0, 6, 6, 'half'),
    ('fp16', 1, 4, 2, 1, 7, 6, 'neighbours'),
    ('fp16', 1, 2, 1, 1, 1024, 1024, 'half'),
    ('bf16', 1, 700, 15, 5, 64, 64, 'half'),
    ('fp16', 64, 1, 24, 1, 64, 64, 'half'),
    ('fp16', 3, 4001, 1, 0, 64, 64, 'half'),
    ('bf16', 3, 4001, 2, 1, 64, 24, 'neighbours'),
    ('bf16', 1, 3, 70, 10, 128, 128, 'half'),
    ('fp32', 2, 2, 3, 2, 1024, 1024, 'half'),
    ('fp32', 1, 3, 2, 1, 1023, 1022, 'neighbours'),
    ('fp16', 1, 2, 5, 2, 1020, 1016, 'half'),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c)))
@pytest.mark.parametrize('back', [False, True], ids=['on', 'back'])
def test_definition(device, case, back):
    type, batch, seq, heads, k_heads, dim, part, pairs = case
    announce('rotary', case, back)
    q, k = make(device, type, batch, seq, heads, dim, 1), make(device, type, batch, seq, max(1, k_heads), dim, 2)
    rotary = lb.Rotary(lb.rotary_frequencies(part, 5000.0, device=device), pairs=pairs, scale=1.25)
    first = [17 * b + 3 for b in range(batch)]
    position = torch.tensor(first, device=device)
    got = lb.rotary(q, position, rotary, k=k if k_heads else None, back=back)
    outs = got if k_heads else (got,)
    for out, x in zip(outs, (q, k)):
        check(out, x, rows_at(first, seq), rotary, type, back)
        assert torch.equal(out[..., part:], x[..., part:])


@pytest.mark.parametrize('type', ['fp16', 'bf16', 'fp32'])
def test_far_and_negative_positions(device, type):
    """Each row at a place of its own: beyond 32 bits, below zero, the same one twice."""
    position = np.array([[0, -1, 2 ** 20 + 1, 2 ** 31 - 1], [2 ** 33 + 5, -(2 ** 35), 131071, 131071]])
    q = make(device, type, 2, 4, 3, 64, 3)
    rotary = lb.Rotary(lb.rotary_frequencies(64, 10000.0, device=device))
    announce('rotary far', type)
    check(lb.rotary(q, torch.tensor(position, device=device), rotary), q, position, rotary, type)


@pytest.mark.parametrize('type,dim,part,shift', [('fp16', 64, 64, 0), ('bf16', 64, 32, 0), ('fp16', 64, 64, 3), ('fp32', 64, 20, 1)])
def test_slices_in_place(device, type, dim, part, shift):
    """q and k as slices of one projection's rows, at any alignment, turned where they lie; what lies beside them stays."""
    announce('rotary in place', type, part, shift)
    g = torch.Generator().manual_seed(4)
    flat = torch.randn(shift + 2 * 5 * 15 * dim, generator=g).to(TYPES[type]).to(device)
    rows = flat[shift:].view(2, 5, 15, dim)
    before = rows.clone()
    q, k = rows[:, :, :9], rows[:, :, 9:12]
    rotary = lb.Rotary(lb.rotary_frequencies(part, device=device), pairs='neighbours')
    position = torch.tensor([100, 7], device=device)
    out, out_k = lb.rotary(q, position, rotary, k=k, out=q, out_k=k)
    assert out is q and out_k is k
    check(q, before[:, :, :9], rows_at([100, 7], 5), rotary, type)
    check(k, before[:, :, 9:12], rows_at([100, 7], 5), rotary, type)
    assert torch.equal(rows[:, :, 12:], before[:, :, 12:]) and torch.equal(flat[:shift], flat[:shift])
    apart, apart_k = lb.rotary(before[:, :, :9], position, rotary, k=before[:, :, 9:12])
    assert torch.equal(apart, q) and torch.equal(apart_k, k)


def test_strided_out_and_broadcast_in(device):
    announce('rotary strides')
    q = make(device, 'fp16', 1, 1, 4, 64, 5).expand(3, 6, 4, 64)
    out = torch.full((6, 4, 3, 72), 7.0, dtype=torch.float16, device=device)[..., :64].permute(2, 0, 1, 3)
    rotary = lb.Rotary(lb.rotary_frequencies(64, device=device))
    assert lb.rotary(q, torch.tensor([0, 50, 99], device=device), rotary, out=out) is out
    check(out, q, rows_at([0, 50, 99], 6), rotary, 'fp16')


def test_back_is_the_gradient(device):
    """Against the transpose of the definition's matrix, and against differences of the forward direction."""
    announce('rotary gradient')
    x = make(device, 'fp32', 1, 2, 1, 16, 6)
    rotary = lb.Rotary(lb.rotary_frequencies(12, device=device), pairs='half', scale=1.3)
    position = torch.tensor([41], device=device)
    grad = make(device, 'fp32', 1, 2, 1, 16, 7)
    got = lb.rotary(grad, position, rotary, back=True).double()
    step = 2.0 ** -6                     # the map is linear: a difference has no error of its own but the outputs' roundings
    for i in range(32):
        e = torch.zeros(32, device=device)
        e[i] = step
        e = e.view_as(x)
        up, low = lb.rotary(x + e, position, rotary).double(), lb.rotary(x - e, position, rotary).double()
        moved = ((x + e).double() - (x - e).double()).abs().max()
        want = ((up - low) / moved * grad.double()).sum()
        # 16 outputs of a row at most change: each of the two is off by 2^-19 of what it is (below 2 * 1.3 * 4)
        assert abs(float(got.view(-1)[i] - want)) <= 4 * 2.0 ** -19 * 10.4 / float(moved) * float(grad.abs().max())
    eye = torch.eye(16, device=device).view(16, 1, 1, 16)
    at = torch.full((16,), 41, device=device)
    on, off = lb.rotary(eye, at, rotary).view(16, 16), lb.rotary(eye, at, rotary, back=True).view(16, 16)
    assert torch.equal(on.T, off)


@pytest.mark.parametrize('out', ['apart', 'in place'])
def test_many_rows(device, out):
    """Rows of more bytes than the caches keep have the values of the same rows in smaller calls."""
    announce('rotary many rows', out)
    x = make(device, 'fp16', 2, 2300, 64, 128, 10)
    before = x.clone()
    rotary = lb.Rotary(lb.rotary_frequencies(128, device=device))
    got = lb.rotary(x, torch.tensor([5, 70000], device=device), rotary, out=x if out == 'in place' else None)
    for b, first in enumerate((5, 70000)):
        for at in (0, 1000, 2000):
            part = before[b:b + 1, at:at + 1000]
            assert torch.equal(got[b:b + 1, at:at + 1000], lb.rotary(part, torch.tensor([first + at], device=device), rotary))
    if out == 'apart':
        assert torch.equal(x, before)


def test_capture_and_streams(device):
    """A captured call reads its positions at each replay; calls on other streams give the same."""
    announce('rotary capture')
    q, k = make(device, 'bf16', 4, 1, 9, 64, 8), make(device, 'bf16', 4, 1, 3, 64, 9)
    rotary = lb.Rotary(lb.rotary_frequencies(64, device=device))
    position = torch.zeros(4, dtype=torch.int64, device=device)
    out, out_k = torch.zeros_like(q), torch.zeros_like(k)
    call = lb.PreparedRotary(q, position, rotary, out, k=k, out_k=out_k)
    call.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.run()
    for first in ([0, 1, 2, 3], [9, 100, 1000, 10000]):
        position.copy_(torch.tensor(first, device=device))
        graph.replay()
        torch.cuda.synchronize()
        want = lb.rotary(q, position, rotary, k=k)
        assert torch.equal(out, want[0]) and torch.equal(out_k, want[1])
        check(out, q, rows_at(first, 1), rotary, 'bf16')
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = lb.rotary(q, position, rotary)
    side.synchronize()
    assert torch.equal(other, out)
