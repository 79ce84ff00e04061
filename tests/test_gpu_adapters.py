"""lb_adapters against its definition in 64 bits.

Tolerance: z = x A^T is a sum of K fp32 products, off by K 2^-24 of the sum of their magnitudes at the most (products of 16-bit
numbers are exact, each addition rounds; additions of parts and of slices among them).  It enters the second product as two
16-bit numbers: what is left of bf16 is 2^-17 of each z (half a step, 2^-8 of it, and what lies
below that has half a step of 2^-9 of it), of fp16 2^-22 and the subnormals' 2^-25 of the row's largest;
2^-17 of the row's largest |z| bounds both.  The second sum has 2 rank products, off by 2 rank 2^-24 of their magnitudes, and the
scale's product and the sum with y are rounded to 32 bits.  Then the output's own half step.
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


def make(device, type, M, N, K, rank, count, seed=0, scales=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=g).to(TYPES[type]).to(device)
    x, y = r(M, K), r(M, N)
    down, up = (r(count, rank, K).float() * K ** -0.5).to(TYPES[type]), (r(count, N, rank).float() * rank ** -0.5).to(TYPES[type])
    s = (torch.rand(count, generator=g) * 3 - 1.5).to(device) if scales else None
    return x, y, lb.Adapters(down, up, scales=s)


def bound(want, products, tops, y, type, K, rank):
    z = K * 2.0 ** -24 * products + (2.0 ** -17 + 2 * rank * 2.0 ** -24) * tops
    near = z + 2.0 ** -23 * (np.abs(want) + np.abs(y))
    return near + torch.finfo(TYPES[type]).eps / 2 * (np.abs(want) + near) + (2.0 ** -25 if type == 'fp16' else 2.0 ** -134)


def check(out, x, y, adapters, index, type):
    host = lambda t: t.double().cpu().numpy()
    want, products, tops = so.adapters(host(y), host(x), host(adapters.down), host(adapters.up), list(index),
                                       None if adapters.scales is None else host(adapters.scales))
    lone = np.isnan(want)
    got = host(out)
    assert np.array_equal(np.isnan(got), lone)
    limit = bound(want, products, tops, host(y), type, adapters.K, adapters.rank)
    worst = float(np.max((np.abs(got - want) / limit)[~lone], initial=0.0))
    assert worst <= 1, worst               # (a NaN fails too)
    none = np.asarray(index) == -1
    assert torch.equal(out[torch.from_numpy(none)], y[torch.from_numpy(none)])


CASES = [
    # type, M, N, K, rank, count
    ('fp16', 1, 576, 576, 8, 1),
    ('fp16', 5, 192, 576, 16, 4),
    ('bf16', 17, 1536, 576, 32, 3),
    ('fp16', 33, 1000, 264, 24, 7),
    ('bf16', 64, 576, 1536, 64, 64),
    ('fp16', 100, 130, 8, 128, 5),
    ('bf16', 16, 7, 72, 40, 2),
    ('fp16', 3, 1, 64, 8, 2),
    ('bf16', 65, 4104, 136, 56, 9),
    ('fp16', 2100, 264, 72, 16, 3),
    ('bf16', 2049, 96, 40, 32, 2),
    ('fp16', 2300, 72, 264, 64, 70),
    ('bf16', 2048, 40, 264, 128, 4),
    ('fp16', 9, 64, 4168, 104, 3),
    ('fp16', 94, 1544, 2056, 128, 21),
    ('bf16', 64, 4104, 1032, 8, 64),
    ('fp16', 200, 264, 1032, 32, 3),
    ('bf16', 130, 520, 2048, 24, 1),
    ('fp16', 128, 40, 72, 8, 2),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '-'.join(map(str, c)))
@pytest.mark.parametrize('order', ['mixed', 'runs'])
def test_definition(device, case, order):
    type, M, N, K, rank, count = case
    announce('adapters', case, order)
    x, y, adapters = make(device, type, M, N, K, rank, count, scales=count % 2 == 1)
    if order == 'mixed':
        index = [-1 if m % 5 == 4 else (m * 7 + 3) % count for m in range(M)]
    else:
        index = [min(count - 1, m * (count + 1) // M) if m * 3 < 2 * M else -1 for m in range(M)]
    at = torch.tensor(index, device=device)
    out = lb.adapters_add(y, x, adapters, at, out=torch.full_like(y, 9.0))
    check(out, x, y, adapters, index, type)
    place = y.clone()
    assert lb.adapters_add(place, x, adapters, at) is place
    assert torch.equal(place, out)


def test_numbers_that_are_no_adapter(device):
    """They give NaN in their rows, and nothing else."""
    announce('adapters bad numbers')
    x, y, adapters = make(device, 'fp16', 20, 72, 64, 8, 3)
    index = [0, 3, -1, -2, 2 ** 40, -(2 ** 40), 1, 2 ** 32 + 1] + [2, -1] * 6
    out = lb.adapters_add(y, x, adapters, torch.tensor(index, device=device), out=torch.zeros_like(y))
    check(out, x, y, adapters, index, 'fp16')


def test_rows_do_not_reach_each_other(device):
    """A row with NaN and infinities among others of its tile and adapter."""
    announce('adapters rows apart')
    for M in (16, 2048):
        x, y, adapters = make(device, 'fp16', M, 96, 264, 16, 2, seed=2)
        index = torch.arange(M, device=device) % 2
        clean = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
        x[3], x[8, 0] = float('nan'), float('inf')
        got = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
        rest = torch.ones(M, dtype=torch.bool, device=device)
        rest[3] = rest[8] = False
        assert torch.equal(got[rest], clean[rest]) and bool(got[3].isnan().all()) and not bool(got[8].isfinite().any())


@pytest.mark.parametrize('type', ['fp16', 'bf16'])
def test_large_and_small_intermediates(device, type):
    """z past fp16's range and below it: neither is lost."""
    for size in (2.0 ** 9, 2.0 ** -20):
        announce('adapters z', type, size)
        x, _, plain = make(device, type, 7, 64, 576, 16, 2, seed=3, scales=False)
        x = (x.float() * size).to(x.dtype)
        down = (plain.down.float() * min(size, 2.0 ** 9)).to(x.dtype)
        y = torch.zeros((7, 64), dtype=x.dtype, device=device)
        adapters = lb.Adapters(down, plain.up, scales=torch.full((2,), 1 / size ** 2, device=device))
        index = [0, 1, 1, 0, 0, 1, -1]
        check(lb.adapters_add(y, x, adapters, torch.tensor(index, device=device)).clone(), x, torch.zeros_like(y), adapters, index, type)


def test_strides(device):
    """Rows of x, y and out as slices of larger tensors, at any alignment; what lies beside them stays."""
    announce('adapters strides')
    x, y, adapters = make(device, 'fp16', 18, 80, 64, 8, 3, seed=4)
    index = torch.arange(18, device=device) % 4 - 1
    want = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
    wide_x = torch.zeros((18, 77), dtype=x.dtype, device=device)
    wide_y = torch.full((18, 95), 5.0, dtype=x.dtype, device=device)
    wide_x[:, 3:67], wide_y[:, 5:85] = x, y
    got = lb.adapters_add(wide_y[:, 5:85], wide_x[:, 3:67], adapters, index)
    assert torch.equal(got, want)
    assert bool((wide_y[:, :5] == 5).all()) and bool((wide_y[:, 85:] == 5).all())
    assert torch.equal(lb.adapters_add(y, x.T.contiguous().T, adapters, index, out=torch.zeros_like(y)), want)


def test_stack_of_ranks(device):
    """Adapters of several ranks, filled to the largest: each adds what it adds alone."""
    announce('adapters stack')
    g = torch.Generator().manual_seed(5)
    factors = [(torch.randn(r, 72, generator=g), torch.randn(48, r, generator=g)) for r in (1, 4, 20, 8)]
    adapters = lb.Adapters.stack(factors, scales=[1.0, 0.5, 2.0, -1.0], device=device)
    assert adapters.rank == 24 and adapters.count == 4
    x, y, _ = make(device, 'fp16', 9, 48, 72, 8, 1, seed=6)
    index = [0, 1, 2, 3, -1, 3, 2, 1, 0]
    check(lb.adapters_add(y, x, adapters, torch.tensor(index, device=device), out=torch.zeros_like(y)), x, y, adapters, index, 'fp16')


def test_capture_and_streams(device):
    """Adapter numbers are read at each replay; two captured calls have workspaces of their own."""
    announce('adapters capture')
    x, y, adapters = make(device, 'bf16', 24, 576, 576, 16, 6, seed=7)
    index = torch.zeros(24, dtype=torch.int64, device=device)
    outs = [torch.zeros_like(y), torch.zeros_like(y)]
    calls = [lb.PreparedAdapters(y, x, adapters, index, out) for out in outs]
    for call in calls:
        call.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            call.run()
        free = lb.adapters_add(y, x, adapters, index, out=torch.empty_like(y))
    for turn in range(3):
        index.copy_((torch.arange(24, device=device) * (turn + 1)) % 7 - 1)
        graph.replay()
        torch.cuda.synchronize()
        want = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(free, want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
    side.synchronize()
    assert torch.equal(other, want)


def test_copies_and_pickles(device):
    """They have factors of their own, and calls over them read those."""
    announce('adapters copies')
    x, y, adapters = make(device, 'fp16', 3, 64, 64, 8, 2, seed=8)
    index = torch.tensor([1, -1, 0], device=device)
    want = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
    for again in (copy.deepcopy, lambda a: pickle.loads(pickle.dumps(a))):
        twin = again(adapters)
        assert twin.down.data_ptr() != adapters.down.data_ptr()
        assert torch.equal(lb.adapters_add(y, x, twin, index, out=torch.zeros_like(y)), want)
        twin.up.zero_()
        assert torch.equal(lb.adapters_add(y, x, twin, index, out=torch.zeros_like(y)), y)
    assert torch.equal(lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y)), want)
    with pytest.raises(AttributeError):
        adapters.up = adapters.up.clone()
