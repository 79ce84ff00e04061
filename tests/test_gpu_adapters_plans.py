"""lb_adapters by each of its plans: one launch, or z by 16 rows of one adapter or 64 of any in 1 to 12 parts of K, then outputs by wave or
by tiles of 64 rows.  Bounds as test_gpu_adapters derives them.

The parts of K are asked of the library with each case, so that a case that a changed rule moves to another plan is noticed."""
import ctypes

import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from lowbit_hip import serve
from test_gpu_adapters import check, make

pytestmark = pytest.mark.gpu


def takes_parts(parts, M, N, K, rank, count):
    """Whether a call takes K in so many parts (0: in one launch): z has M rank 4 bytes of each in the workspace, in whole 256 bytes."""
    a, size = serve.AdaptersArgs(), ctypes.c_size_t(0)
    a.struct_size, a.M, a.N, a.K, a.rank, a.count = ctypes.sizeof(a), M, N, K, rank, count
    assert lb.library().lb_adapters_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == 0
    return size.value == -(-parts * M * rank * 4 // 256) * 256


PLANS = [
    # M, N, K, rank, count, parts of K: z, then outputs
    (20, 264, 576, 16, 3, 0),              # one launch
    (1, 64, 14336, 8, 1, 12),              # 16 rows; waves, parts past the first four
    (40, 72, 8200, 64, 5, 8),              # 16 rows, 16 ranks of four groups; waves
    (300, 136, 4104, 128, 9, 2),           # 16 rows, 32 ranks of four groups; tiles
    (1100, 130, 72, 16, 3, 1),             # 16 rows; waves, rows that are no 16-byte pieces, every adapter of 64 rows in one
    (2048, 4104, 3592, 16, 3, 4),          # 64 rows, 16 ranks; tiles, two steps of outputs and a rest
    (600, 1032, 12296, 32, 5, 12),         # 64 rows, 32 ranks; tiles
    (500, 264, 12296, 64, 3, 12),          # 64 rows, 64 ranks; tiles
    (300, 1032, 12296, 128, 5, 12),        # 64 rows, 64 ranks of two groups; tiles
    (500, 131, 12296, 64, 70, 12),         # the same with a share of 70 adapters each; waves
]


def numbers(order, M, count):
    if order == 'mixed':
        return [-1 if m % 5 == 4 else (m * 7 + 3) % count for m in range(M)]
    return [min(count - 1, m * (count + 1) // M) if m * 3 < 2 * M else -1 for m in range(M)]


@pytest.mark.parametrize('case', PLANS, ids=lambda c: '-'.join(map(str, c)))
@pytest.mark.parametrize('order', ['mixed', 'runs'])
@pytest.mark.parametrize('type', ['fp16', 'bf16'])
def test_plans(device, case, order, type):
    """Apart and in place, the same calls again, and rows whose number is no adapter among them."""
    M, N, K, rank, count, parts = case
    announce('adapters plans', case, order, type)
    assert takes_parts(parts, M, N, K, rank, count)
    x, y, adapters = make(device, type, M, N, K, rank, count, scales=count % 2 == 1)
    index = numbers(order, M, count)
    if M > 10:
        index[M // 2], index[M - 1] = count, -2
    at = torch.tensor(index, device=device)
    out = lb.adapters_add(y, x, adapters, at, out=torch.full_like(y, 9.0))
    check(out, x, y, adapters, index, type)
    place = y.clone()
    for again in (lb.adapters_add(place, x, adapters, at), lb.adapters_add(y, x, adapters, at, out=torch.zeros_like(y))):
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize('M,N,K,rank,parts', [(2100, 264, 3528, 16, 4), (600, 264, 12296, 32, 12), (500, 130, 12296, 64, 12),
                                              (300, 264, 12296, 128, 12)])
def test_rows_of_large_tiles_do_not_reach_each_other(device, M, N, K, rank, parts):
    """A row with NaN, one with an infinity and one without an adapter, among others of their tiles of 64."""
    announce('adapters tiles apart', M, N, K, rank)
    assert takes_parts(parts, M, N, K, rank, 2)     # (16 rows at a time would be in fewer)
    x, y, adapters = make(device, 'fp16', M, N, K, rank, 2, seed=2)
    index = torch.arange(M, device=device) % 2
    index[5] = -1
    clean = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
    x[3], x[8, 0], x[5], y[7, 3] = float('nan'), float('inf'), float('nan'), float('inf')
    got = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
    rest = torch.ones(M, dtype=torch.bool, device=device)
    rest[[3, 7, 8]] = False
    assert torch.equal(got[rest], clean[rest]) and torch.equal(got[5], y[5])
    assert bool(got[3].isnan().all()) and not bool(got[8].isfinite().any())
    assert bool(got[7, 3] == float('inf')) and torch.equal(got[7, 4:], clean[7, 4:])


@pytest.mark.parametrize('M,N,K,rank,shift', [(600, 264, 1032, 32, 8), (600, 264, 1032, 32, 3), (2100, 136, 3528, 16, 16), (64, 264, 4104, 64, 1)])
def test_slices(device, M, N, K, rank, shift):
    """x, y and out as slices of larger rows; what lies beside them stays."""
    announce('adapters slices', M, N, K, rank, shift)
    x, y, adapters = make(device, 'bf16', M, N, K, rank, 4, seed=3)
    index = torch.arange(M, device=device) % 5 - 1
    wide_x = torch.full((M, K + 40), float('nan'), dtype=x.dtype, device=device)
    wide_x[:, shift:shift + K] = x
    wides = [torch.full((M, N + 40), 5.0, dtype=x.dtype, device=device) for _ in range(2)]
    wides[0][:, shift:shift + N] = y
    cut = [w[:, shift:shift + N] for w in wides]
    lb.adapters_add(cut[0], wide_x[:, shift:shift + K], adapters, index, out=cut[1])
    check(cut[1].clone(), x, y, adapters, index.tolist(), 'bf16')
    assert torch.equal(cut[0], y)
    lb.adapters_add(cut[0], wide_x[:, shift:shift + K], adapters, index)
    assert torch.equal(cut[0], cut[1])
    for w in wides:
        assert bool((w[:, :shift] == 5).all()) and bool((w[:, shift + N:] == 5).all())


def test_two_launches_captured(device):
    """Calls of two launches with workspaces of their own, captured together and replayed with other numbers."""
    announce('adapters two launches captured')
    x, y, adapters = make(device, 'fp16', 300, 264, 4104, 64, 6, seed=4)
    index = torch.zeros(300, dtype=torch.int64, device=device)
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
        index.copy_((torch.arange(300, device=device) * (turn + 1)) % 7 - 1)
        graph.replay()
        torch.cuda.synchronize()
        want = lb.adapters_add(y, x, adapters, index, out=torch.zeros_like(y))
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(free, want)
        check(want, x, y, adapters, index.tolist(), 'fp16')
