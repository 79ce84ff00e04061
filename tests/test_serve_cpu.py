"""Host-only checks of rotary positions, the KV cache in pages and adapters: argument errors before any launch, workspace sizes,
the Python wrappers' refusals, frequencies, and the oracle against itself."""
import ctypes
import math

import numpy as np
import pytest
import torch

import lowbit_hip as lb
from lowbit_hip import serve
from oracle import serve_oracle as so


def fill(a, over):
    for name, value in over.items():
        target, _, field = name.partition('__')
        if field:
            setattr(getattr(a, target), field, value)
        else:
            setattr(a, target, value)
    return a


def rows(data, *strides):
    return serve.RowsStruct(data, *strides)


def rotation(**over):
    r = serve.RotationStruct(0x900000, 64, 0, 1.0, 0)
    return fill(r, over)


def rotary(**over):
    a = serve.RotaryArgs()
    a.struct_size, a.type, a.batch, a.seq, a.head_dim, a.heads, a.k_heads = ctypes.sizeof(a), 0, 2, 5, 64, 9, 3
    a.q, a.out = rows(0x100000, 5 * 960, 960, 64), rows(0x200000, 5 * 576, 576, 64)
    a.k, a.out_k = rows(0x100000 + 1152, 5 * 960, 960, 64), rows(0x300000, 5 * 192, 192, 64)
    a.position, a.rotation = 0x800000, rotation()
    return fill(a, over)


def cache():
    return serve.PagedCacheStruct(0, 64, 10, 3, 32, 0x1000000, 0x2000000)


def append(**over):
    a = serve.PagedAppendArgs()
    a.struct_size, a.cache, a.table, a.batch, a.seq = ctypes.sizeof(a), cache(), serve.PageTableStruct(0x700000, 6, 6), 2, 5
    a.k, a.v = rows(0x600000, 5 * 192, 192, 64), rows(0x610000, 5 * 192, 192, 64)
    a.position, a.rows, a.rotation = 0x800000, 0x800100, rotation()
    return fill(a, over)


def attention(**over):
    a = serve.PagedAttentionArgs()
    a.struct_size, a.cache, a.table, a.batch, a.heads = ctypes.sizeof(a), cache(), serve.PageTableStruct(0x700000, 60, 60), 2, 9
    a.q, a.out, a.position, a.scale = rows(0xA00000, 576, 0, 64), rows(0xB00000, 576, 0, 64), 0x800000, 0.125
    a.rotation, a.workspace, a.workspace_bytes = rotation(), 0x4000000, 64 << 20
    return fill(a, over)


def adapters(**over):
    a = serve.AdaptersArgs()
    a.struct_size, a.type, a.M, a.N, a.K, a.rank, a.count = ctypes.sizeof(a), 0, 20, 576, 576, 16, 4
    a.down, a.up, a.scales, a.index = 0x100000, 0x200000, 0x300000, 0x310000
    a.x, a.ldx, a.y, a.ldy, a.out, a.ldo = 0x400000, 576, 0x500000, 576, 0x600000, 576
    a.workspace, a.workspace_bytes = 0x700000, 1 << 20
    return fill(a, over)


BAD_ROTATION = [
    (dict(rotation__dims=3), 'dims'), (dict(rotation__dims=0), 'dims'), (dict(rotation__dims=66), 'dims'),
    (dict(rotation__pairs=2), 'pairs'), (dict(rotation__scale=float('nan')), 'scale'),
    (dict(rotation__frequencies=0x900004), 'frequencies'),
]
BAD_ROTARY = BAD_ROTATION + [
    (dict(struct_size=8), 'struct_size'), (dict(type=3), 'type'), (dict(batch=0), 'rows'), (dict(seq=2 ** 28), 'rows'), (dict(batch=8, seq=2 ** 22 + 1), 'rows'),
    (dict(head_dim=1), 'head_dim'), (dict(head_dim=1025), 'head_dim'), (dict(heads=0), 'heads'), (dict(k_heads=-1), 'heads'),
    (dict(rotation__frequencies=0), 'frequencies'), (dict(position=0), 'position'), (dict(position=0x800004), 'position'),
    (dict(q__data=0), 'q must'), (dict(q__data=0x100001), 'q must'), (dict(k__data=0), 'k must'),
    (dict(q__row_stride=-64), 'strides of q'), (dict(q__batch_stride=2 ** 41), 'strides of q'),
    (dict(out__head_stride=32), 'rows of out overlap'), (dict(out_k__batch_stride=0), 'rows of out_k overlap'),
    (dict(out__data=0x100002), 'overlaps'), (dict(out__data=0x300000), 'overlaps'), (dict(out__data=0x800000), 'overlaps'),
    (dict(out_k__data=0x900000), 'overlaps'),
    (dict(out__data=0x100000, out__row_stride=960, out__batch_stride=4800), 'both or neither'),
    (dict(out__data=0x100000, out__row_stride=960, out__batch_stride=4800, k__data=0x100000 + 1100, out_k__data=0x100000 + 1100,
          out_k__row_stride=960, out_k__batch_stride=4800), 'rows of q and k overlap'),
]
BAD_CACHE = [
    (dict(struct_size=8), 'struct_size', 1), (dict(cache__type=2), 'type', 1), (dict(cache__head_dim=96), 'head_dim', 5),
    (dict(cache__pages=0), 'pages', 1), (dict(cache__pages=2 ** 31), 'pages', 1), (dict(cache__kv_heads=0), 'kv_heads', 1),
    (dict(cache__page=8), 'page', 1), (dict(cache__page=48), 'page', 1), (dict(cache__page=2048), 'page', 1),
    (dict(cache__keys=0), 'keys must', 1), (dict(cache__values=0x2000008), 'values must', 1),
    (dict(cache__values=0x1000010), 'keys overlaps values', 1),
    (dict(batch=0), 'batch', 1), (dict(batch=65536), 'batch', 1), (dict(table__data=0), 'table must', 1),
    (dict(table__data=0x700002), 'table must', 1), (dict(table__longest=0), 'entries', 1),
    (dict(table__longest=2 ** 25 + 1), 'entries', 1), (dict(table__stride=-1), 'stride', 1), (dict(position=0), 'position', 1),
]
BAD_APPEND = BAD_CACHE + [(over, needle, 1) for over, needle in BAD_ROTATION] + [
    (dict(seq=0), 'seq', 1), (dict(seq=2 ** 62), 'seq', 1), (dict(k__data=0), 'k must', 1), (dict(v__data=0x610008), 'v must', 1),
    (dict(k__row_stride=100), 'strides of k', 1), (dict(v__head_stride=-64), 'strides of v', 1), (dict(rows=0x800104), 'rows', 1),
    (dict(k__data=0x1000000), 'keys overlaps k', 1), (dict(table__data=0x2000000), 'values overlaps table', 1),
]
BAD_ATTENTION = BAD_CACHE + [(over, needle, 1) for over, needle in BAD_ROTATION] + [
    (dict(heads=10), 'heads', 1), (dict(heads=0), 'heads', 1), (dict(scale=float('inf')), 'scale', 1),
    (dict(scale=float('nan')), 'scale', 1), (dict(q__data=0xA00004), 'q must', 1), (dict(out__head_stride=0), 'rows of out overlap', 1),
    (dict(out__data=0xA00040), 'out overlaps q', 1), (dict(out__data=0x2000000), 'out overlaps values', 1),
    (dict(k__data=0x600000), 'v must', 1), (dict(v__data=0x600000), 'k must', 1),
    (dict(k__data=0x1000000, v__data=0x600000), 'keys overlaps k', 1), (dict(workspace=0), 'workspace', 1),
    (dict(workspace=0x4000080), 'workspace', 1), (dict(workspace_bytes=4096), 'workspace', 1),
    (dict(workspace=0xB00000), 'overlaps', 1), (dict(workspace=0x1000000), 'overlaps', 1),
    (dict(batch=65535, heads=9 * 30, cache__kv_heads=90), '2^22', 5),
]
BAD_ADAPTERS = [
    (dict(struct_size=8), 'struct_size'), (dict(type=2), 'type'), (dict(M=0), 'M, N and K'), (dict(N=0), 'M, N and K'),
    (dict(K=4), 'M, N and K'), (dict(K=580), 'M, N and K'), (dict(M=2 ** 29), 'M, N and K'), (dict(rank=0), 'rank'), (dict(rank=12), 'rank'),
    (dict(rank=136), 'rank'), (dict(count=0), 'adapters'), (dict(count=2 ** 25), 'adapters'), (dict(down=0), 'down'),
    (dict(up=0x200008), 'up must'), (dict(scales=0x300002), 'scales'), (dict(index=0), 'index'), (dict(x=0x400002), 'x must'),
    (dict(ldx=580), 'strides of x'), (dict(y=0), 'y must'), (dict(out=0x600001), 'out must'), (dict(ldo=575), 'rows of out overlap'),
    (dict(out=0x500002), 'out overlaps y'), (dict(out=0x500000, ldo=640), 'out overlaps y'), (dict(out=0x400000), 'out overlaps x'),
    (dict(out=0x310000), 'out overlaps'), (dict(M=200, workspace=0), 'workspace'), (dict(M=200, workspace=0x700010), 'workspace'),
    (dict(M=200, workspace_bytes=12799), 'workspace'), (dict(M=200, workspace=0x500000), 'workspace overlaps y'),
    (dict(M=200, workspace=0x600000), 'out overlaps workspace'),
]


def refused(fn, a, needle, status=1):
    got = getattr(lb.library(), fn)(ctypes.byref(a), None)
    message = lb.library().lb_last_error().decode()
    assert got == status and needle in message, (got, message)


@pytest.mark.parametrize('over,needle', BAD_ROTARY, ids=lambda v: str(v)[:60])
def test_rotary_refusals(over, needle):
    refused('lb_rotary', rotary(**over), needle)


@pytest.mark.parametrize('over,needle,status', BAD_APPEND, ids=lambda v: str(v)[:60])
def test_append_refusals(over, needle, status):
    refused('lb_paged_append', append(**over), needle, status)


@pytest.mark.parametrize('over,needle,status', BAD_ATTENTION, ids=lambda v: str(v)[:60])
def test_attention_refusals(over, needle, status):
    refused('lb_paged_attention', attention(**over), needle, status)


@pytest.mark.parametrize('over,needle', BAD_ADAPTERS, ids=lambda v: str(v)[:60])
def test_adapters_refusals(over, needle):
    refused('lb_adapters', adapters(**over), needle)


def test_null_arguments():
    for fn in ('lb_rotary', 'lb_paged_append', 'lb_paged_attention', 'lb_adapters'):
        assert getattr(lb.library(), fn)(None, None) == 1
    for fn, a in (('lb_paged_attention_workspace_bytes', attention()), ('lb_adapters_workspace_bytes', adapters())):
        assert getattr(lb.library(), fn)(ctypes.byref(a), None) == 1


def test_workspaces():
    size = ctypes.c_size_t(1)
    ask = lambda fn, a: getattr(lb.library(), fn)(ctypes.byref(a), ctypes.byref(size))
    assert ask('lb_paged_attention_workspace_bytes', attention(table__longest=4)) == 0 and size.value == 0   # too short to be split
    assert ask('lb_paged_attention_workspace_bytes', attention(table__longest=10 ** 5)) == 0
    assert lb.ZEROED_WORKSPACE_BYTES < size.value < 64 << 20
    assert ask('lb_paged_attention_workspace_bytes', attention(heads=10)) == 1 and size.value == 0
    assert ask('lb_adapters_workspace_bytes', adapters()) == 0 and size.value == 0      # both products in one launch
    assert ask('lb_adapters_workspace_bytes', adapters(K=4096)) == 0 and size.value >= 20 * 16 * 4
    assert ask('lb_adapters_workspace_bytes', adapters(rank=9)) == 1 and size.value == 0


def test_struct_sizes():
    """The packed structs are as long as their mirrors, and the mirrors as the library's own (a shorter one is refused)."""
    r = serve._ROTATION.size
    assert serve._ROTARY.size + r == ctypes.sizeof(serve.RotaryArgs)
    head = serve._PAGED_HEAD.size + serve._PAGED_CACHE.size
    assert head + serve._APPEND.size + r == ctypes.sizeof(serve.PagedAppendArgs)
    assert serve._ADAPTERS.size == ctypes.sizeof(serve.AdaptersArgs)
    assert head + serve._ATTENTION.size + r + serve._ATTENTION_TAIL.size == ctypes.sizeof(serve.PagedAttentionArgs)
    for fn, a in (('lb_rotary', rotary()), ('lb_paged_append', append()), ('lb_paged_attention', attention()), ('lb_adapters', adapters())):
        a.struct_size -= 1
        refused(fn, a, 'struct_size')


def test_wrappers_refuse_host_tensors_and_wrong_ones():
    q = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match='device tensor'):
        lb.Rotary(lb.rotary_frequencies(64))
    for bad in (torch.zeros(32), torch.zeros(2, 2, dtype=torch.float64), torch.zeros(0, dtype=torch.float64), None):
        with pytest.raises(ValueError, match='float64'):
            lb.Rotary(bad)
    with pytest.raises(ValueError, match='q must'):
        lb.rotary(q, torch.zeros(1, dtype=torch.int64), None)
    with pytest.raises(ValueError, match='PagedKVCache'):
        lb.paged_append(None, q, q, None, None)
    with pytest.raises(ValueError, match='PagedKVCache'):
        lb.paged_attention(q[:, 0], object(), None, None)
    with pytest.raises(ValueError, match='Adapters'):
        lb.adapters_add(q, q, None, None)
    with pytest.raises(ValueError, match='ROCm device'):
        lb.PagedKVCache.empty(2, 3, device='cpu')
    with pytest.raises(ValueError, match='ROCm device'):
        lb.Adapters(torch.zeros(1, 8, 16, dtype=torch.float16), torch.zeros(1, 4, 8, dtype=torch.float16))
    for shape in ((0, 3, 16, 64), (2, 3, 24, 64), (2, 3, 16, 96), (2, 3, 16)):
        with pytest.raises(ValueError, match='keys'):
            lb.PagedKVCache(torch.zeros(shape, dtype=torch.float16), None)
    for options in (dict(page=24), dict(page=8), dict(head_dim=32), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            lb.PagedKVCache.empty(2, 3, **options)
    for pages in (0, True, 1.5):
        with pytest.raises(ValueError, match='pages'):
            lb.PagedKVCache.empty(pages, 3)
    for rank in (4, 136):
        with pytest.raises(ValueError, match='rank'):
            lb.Adapters(torch.zeros(1, rank, 16, dtype=torch.float16), torch.zeros(1, 4, rank, dtype=torch.float16))
    for factors in ([], [(torch.zeros(4, 16), torch.zeros(8, 5))], [(torch.zeros(4, 16), torch.zeros(8, 4)), (torch.zeros(4, 24), torch.zeros(8, 4))]):
        with pytest.raises(ValueError):
            lb.Adapters.stack(factors, device='cpu')


def test_frequencies():
    plain = lb.rotary_frequencies(8, 10000.0)
    assert plain.dtype == torch.float64 and np.allclose(plain, [1, 0.1, 0.01, 0.001], rtol=1e-14)
    assert np.allclose(lb.rotary_frequencies(8, 10000.0, stretch='linear', factor=4), plain / 4, rtol=1e-14)
    raised = lb.rotary_frequencies(8, 10000.0, stretch='theta', factor=4)
    assert np.allclose(raised[-1], plain[-1] / 4, rtol=1e-12) and float(raised[0]) == 1.0
    assert np.allclose(lb.rotary_frequencies(2, 10000.0, stretch='theta', factor=4), [0.25])
    parts = lb.rotary_frequencies(8, 10000.0, stretch='parts', factor=4, length=2 * math.pi * 1000, low=2, high=50)
    turns = 1000 * plain.numpy()                          # 1000, 100, 10, 1
    want = plain.numpy() * np.array([1, 1, 0.25 + 0.75 * (turns[2] - 2) / 48, 0.25])
    assert np.allclose(parts, want, rtol=1e-12)
    for bad in (dict(dims=7), dict(dims=0), dict(dims=8, theta=0), dict(dims=8, stretch='other'), dict(dims=8, factor=-1),
                dict(dims=8, stretch='parts'), dict(dims=8, stretch='parts', length=9, low=3, high=3)):
        with pytest.raises(ValueError):
            lb.rotary_frequencies(**bad)


def test_oracle():
    """Rotation: a turn keeps each pair's length, positions add, back undoes it; attention of equal scores is a mean; adapters."""
    rng = np.random.default_rng(0)
    x, f = rng.standard_normal((4, 2, 8)), np.array([0.7, 0.01, 3.0])
    for pairs, first, second in (('half', [0, 1, 2], [3, 4, 5]), ('neighbours', [0, 2, 4], [1, 3, 5])):
        y = so.turned(x, np.arange(4), f, pairs)
        assert np.allclose(np.hypot(y[..., first], y[..., second]), np.hypot(x[..., first], x[..., second]))
        assert np.array_equal(y[..., 6:], x[..., 6:]) and np.allclose(y[0], x[0])
        assert np.allclose(so.turned(y, np.full(4, 5), f, pairs), so.turned(x, np.arange(4) + 5, f, pairs))
        assert np.allclose(so.turned(y, np.arange(4), f, pairs, back=True), x)
        assert np.allclose(so.partner_sizes(x, 3, pairs)[..., first], np.abs(x[..., first]) + np.abs(x[..., second]))
    values = rng.standard_normal((2, 3, 8, 16))
    by_slot = so.values_by_slot(values)
    assert by_slot.shape == (2, 48, 8) and by_slot[1, 37, 5] == values[1, 2, 5, 5]
    k, v = rng.standard_normal((1, 5, 8)), rng.standard_normal((1, 5, 8))
    out, mean, size = so.attention(np.zeros((2, 8)), k, v, 1.0)
    assert np.allclose(out, v[0].mean(0)) and np.allclose(mean, np.abs(v[0]).mean(0)) and np.all(size == 0)
    A, B, x, y = rng.standard_normal((2, 3, 4)), rng.standard_normal((2, 5, 3)), rng.standard_normal((4, 4)), rng.standard_normal((4, 5))
    out, _, _ = so.adapters(y, x, A, B, [1, -1, 2, 0], [0.5, 2.0])
    assert np.allclose(out[0], y[0] + 2 * B[1] @ A[1] @ x[0]) and np.array_equal(out[1], y[1]) and np.isnan(out[2]).all()
