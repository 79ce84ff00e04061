"""Host-only checks of the 8-bit KV cache's entry points: argument errors before any launch, workspace sizes, the Python
wrappers' refusals, and the oracle's own rounding."""
import ctypes

import numpy as np
import pytest
import torch

import lowbit_hip as lb
from oracle import kv_oracle as ko


def cache(**over):
    c = lb.KVCacheStruct()
    c.format, c.head_dim, c.batch, c.kv_heads, c.capacity = 0, 64, 2, 3, 256
    c.key_codes, c.value_codes, c.key_scales, c.value_scales = 0x100000, 0x200000, 0x300000, 0x310000
    c.key_tail, c.value_tail = 0x400000, 0x500000
    for name, value in over.items():
        setattr(c, name, value)
    return c


def fill(a, over):
    for name, value in over.items():
        target, _, field = name.partition('__')
        if field:
            setattr(getattr(a, target), field, value)
        else:
            setattr(a, target, value)
    return a


def append(**over):
    a = lb.KVAppendArgs()
    a.struct_size, a.cache, a.seq = ctypes.sizeof(a), cache(), 5
    a.k, a.v = lb.KVRows(0x600000, 5 * 192, 192, 64), lb.KVRows(0x610000, 5 * 192, 192, 64)
    a.position, a.rows = 0x700000, 0x700100
    return fill(a, over)


def read(**over):
    a = lb.KVReadArgs()
    a.struct_size, a.cache, a.length, a.start, a.count = ctypes.sizeof(a), cache(), 0x700000, 3, 100
    a.keys, a.values = lb.KVRows(0x800000, 3 * 6400, 64, 6400), lb.KVRows(0x900000, 3 * 6400, 64, 6400)
    return fill(a, over)


def attention(**over):
    a = lb.KVAttentionArgs()
    a.struct_size, a.cache, a.seq, a.heads, a.scale = ctypes.sizeof(a), cache(), 5, 9, 0.125
    a.q, a.out = lb.KVRows(0xA00000, 5 * 576, 576, 64), lb.KVRows(0xB00000, 5 * 576, 576, 64)
    a.position, a.workspace, a.workspace_bytes = 0x700000, 0xC00000, 4 << 20
    return fill(a, over)


FAR = dict(cache__capacity=1 << 20, cache__key_codes=1 << 32, cache__value_codes=2 << 32, cache__key_scales=3 << 32,
           cache__value_scales=4 << 32, cache__key_tail=5 << 32, cache__value_tail=6 << 32)   # a long cache: needs a workspace
BAD_CACHE = [
    (dict(cache__format=2), 'format', lb.INVALID_ARGUMENT),
    (dict(cache__head_dim=96), 'head_dim', lb.UNSUPPORTED),
    (dict(cache__batch=0), 'batch', lb.INVALID_ARGUMENT),
    (dict(cache__kv_heads=65536), 'kv_heads', lb.INVALID_ARGUMENT),
    (dict(cache__capacity=100), 'capacity', lb.INVALID_ARGUMENT),
    (dict(cache__capacity=2 ** 28 + 64), 'capacity', lb.INVALID_ARGUMENT),
    (dict(cache__capacity=2 ** 63 - 64), 'capacity', lb.INVALID_ARGUMENT),
    (dict(cache__key_codes=0), 'key_codes must', lb.INVALID_ARGUMENT),
    (dict(cache__value_tail=0x500008), 'value_tail must', lb.INVALID_ARGUMENT),
    (dict(cache__value_codes=0x100000 + 2 * 3 * 256 * 64 - 16), 'key_codes overlaps value_codes', lb.INVALID_ARGUMENT),
    (dict(cache__value_scales=0x300000), 'key_scales overlaps value_scales', lb.INVALID_ARGUMENT),
    (dict(struct_size=8), 'struct_size', lb.INVALID_ARGUMENT),
]
BAD_APPEND = [
    (dict(seq=0), 'seq', lb.INVALID_ARGUMENT),
    (dict(seq=2 ** 62), 'seq', lb.INVALID_ARGUMENT),
    (dict(k__data=0), 'k must', lb.INVALID_ARGUMENT),
    (dict(v__data=0x610008), 'v must', lb.INVALID_ARGUMENT),
    (dict(k__row_stride=100), 'strides of k', lb.INVALID_ARGUMENT),
    (dict(v__head_stride=-64), 'strides of v', lb.INVALID_ARGUMENT),
    (dict(v__batch_stride=2 ** 62), 'strides of v', lb.INVALID_ARGUMENT),
    (dict(position=0), 'position', lb.INVALID_ARGUMENT),
    (dict(rows=0x700104), 'rows', lb.INVALID_ARGUMENT),
    (dict(cos=0x780000), 'cos and sin', lb.INVALID_ARGUMENT),
    (dict(k__data=0x400000 + 64), 'key_tail overlaps k', lb.INVALID_ARGUMENT),
    (dict(position=0x310000), 'value_scales overlaps position', lb.INVALID_ARGUMENT),
]
BAD_READ = [
    (dict(start=-1), 'start', lb.INVALID_ARGUMENT),
    (dict(count=0), 'count', lb.INVALID_ARGUMENT),
    (dict(start=157), 'start', lb.INVALID_ARGUMENT),
    (dict(start=2 ** 63 - 1), 'start', lb.INVALID_ARGUMENT),
    (dict(length=0), 'length', lb.INVALID_ARGUMENT),
    (dict(keys__data=0), 'keys must', lb.INVALID_ARGUMENT),
    (dict(keys__row_stride=56), 'rows of keys overlap', lb.INVALID_ARGUMENT),
    (dict(values__batch_stride=6400), 'rows of values overlap', lb.INVALID_ARGUMENT),
    (dict(values__data=0x800000), 'keys overlaps values', lb.INVALID_ARGUMENT),
    (dict(values__data=0x100000), 'values overlaps key_codes', lb.INVALID_ARGUMENT),
]
BAD_ATTENTION = [
    (dict(heads=10), 'kv_heads', lb.INVALID_ARGUMENT),
    (dict(heads=0), 'heads', lb.INVALID_ARGUMENT),
    (dict(seq=2 ** 27), '2^28 rows', lb.INVALID_ARGUMENT),
    (dict(cache__batch=65535, cache__kv_heads=300, heads=300), 'overlaps', lb.INVALID_ARGUMENT),
    (dict(scale=float('nan')), 'scale', lb.INVALID_ARGUMENT),
    (dict(scale=float('inf')), 'scale', lb.INVALID_ARGUMENT),
    (dict(scale=-1.0), 'scale', lb.INVALID_ARGUMENT),
    (dict(scale=65537.0), 'scale', lb.INVALID_ARGUMENT),
    (dict(q__data=0xA00004), 'q must', lb.INVALID_ARGUMENT),
    (dict(out__head_stride=0), 'rows of out overlap', lb.INVALID_ARGUMENT),
    (dict(out__data=0xA00040), 'out overlaps q', lb.INVALID_ARGUMENT),
    (dict(out__data=0x200000), 'out overlaps value_codes', lb.INVALID_ARGUMENT),
    (dict(FAR, workspace=0xC00080), 'workspace', lb.INVALID_ARGUMENT),
    (dict(FAR, workspace_bytes=50000), 'workspace', lb.INVALID_ARGUMENT),
    (dict(FAR, workspace=0xB00000), 'out overlaps workspace', lb.INVALID_ARGUMENT),
    (dict(FAR, workspace=0xA00000), 'workspace overlaps q', lb.INVALID_ARGUMENT),
    (dict(sin=0x780000), 'cos and sin', lb.INVALID_ARGUMENT),
    (dict(k__data=0x600000), 'v must', lb.INVALID_ARGUMENT),
    (dict(v__data=0x600000), 'k must', lb.INVALID_ARGUMENT),
    (dict(FAR, workspace=0), 'workspace', lb.INVALID_ARGUMENT),
]


@pytest.mark.parametrize('entry,make,over,needle,status',
                         [(e, m, *bad) for e, m in (('lb_kv_append', append), ('lb_kv_read', read), ('lb_kv_attention', attention))
                          for bad in BAD_CACHE]
                         + [('lb_kv_append', append, *bad) for bad in BAD_APPEND]
                         + [('lb_kv_read', read, *bad) for bad in BAD_READ]
                         + [('lb_kv_attention', attention, *bad) for bad in BAD_ATTENTION])
def test_argument_errors_come_before_any_launch(entry, make, over, needle, status):
    lib = lb.library()
    assert getattr(lib, entry)(ctypes.byref(make(**over)), None) == status, lib.lb_last_error().decode()
    assert needle in lib.lb_last_error().decode()


def test_null_args_and_workspace_query():
    lib = lb.library()
    for entry in ('lb_kv_append', 'lb_kv_read', 'lb_kv_attention'):
        assert getattr(lib, entry)(None, None) == lb.INVALID_ARGUMENT and 'NULL' in lib.lb_last_error().decode()
    size = ctypes.c_size_t(7)
    assert lib.lb_kv_attention_workspace_bytes(None, ctypes.byref(size)) == lb.INVALID_ARGUMENT
    a = attention()
    assert lib.lb_kv_attention_workspace_bytes(ctypes.byref(a), None) == lb.INVALID_ARGUMENT
    assert lib.lb_kv_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == lb.OK and size.value == 0
    a = attention(heads=10)
    assert lib.lb_kv_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == lb.INVALID_ARGUMENT
    a = attention(seq=1, **FAR)     # a long cache: parts with 16 rows of 64 sums and two statistics, behind the zeroed bytes
    assert lib.lb_kv_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == lb.OK
    assert size.value == 4096 + 514 * 16 * 66 * 4
    a = attention(seq=11, cache__capacity=64, cache__batch=200, **{k: v for k, v in FAR.items() if k != 'cache__capacity'})
    assert lib.lb_kv_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == lb.OK and size.value == 0   # 600 tiles


def test_failed_state_refuses_the_cache_entries():
    import subprocess
    import sys
    from pathlib import Path
    code = r'''
import ctypes, sys
sys.path[:0] = sys.argv[1:]
import lowbit_hip as lb
lib = lb.library()
lb.mark_failed('forced by the test')
for name, args in (('lb_kv_append', lb.KVAppendArgs), ('lb_kv_read', lb.KVReadArgs), ('lb_kv_attention', lb.KVAttentionArgs)):
    assert getattr(lib, name)(ctypes.byref(args()), None) == lb.DEVICE_FAILED, name
    assert 'forced by the test' in lib.lb_last_error().decode()
print('ok')
'''
    root = Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, '-c', code, str(root), str(root / 'torch-intel-npu_amd')], capture_output=True,
                         text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip().endswith('ok'), out.stdout + out.stderr


def buffers(batch=2, heads=3, blocks=2, dim=64, dtype=torch.int8):
    z = lambda dt, *s: torch.zeros((batch, heads, *s), dtype=torch.uint8 if dt == torch.float8_e4m3fn else dt).view(dt)
    return dict(key_codes=z(dtype, blocks, 64, dim), value_codes=z(dtype, blocks, dim, 64), key_scales=z(torch.float32, blocks),
                value_scales=z(torch.float32, blocks), key_tail=z(torch.float16, 2, 64, dim), value_tail=z(torch.float16, 2, dim, 64))


@pytest.mark.parametrize('over,needle', [
    (dict(key_codes=torch.zeros(2, 3, 2, 64, 64)), 'key_codes must be int8'),
    (dict(key_codes=torch.zeros(2, 3, 2, 32, 64, dtype=torch.int8)), 'key_codes must be'),
    (dict(value_codes=torch.zeros(2, 3, 2, 64, 64, dtype=torch.uint8)), 'value_codes must be'),
    (dict(key_scales=torch.zeros(2, 3, 2, dtype=torch.float16)), 'key_scales must be'),
    (dict(value_scales=torch.zeros(2, 2, 3).transpose(1, 2)), 'value_scales must be contiguous'),
    (dict(key_tail=torch.zeros(2, 3, 64, 64, dtype=torch.float16)), 'key_tail must be'),
    (dict(value_tail=torch.zeros(2, 3, 2, 64, 64, dtype=torch.float16, device='meta')), 'value_tail must be on'),
    (dict(), 'ROCm device tensor'),
])
def test_cache_buffers_are_checked(over, needle):
    with pytest.raises(ValueError, match=needle):
        lb.QuantizedKVCache(**{**buffers(), **over})


@pytest.mark.parametrize('args,options,needle', [
    ((1, 1, 64), dict(format='int4'), 'format'),
    ((0, 1, 64), {}, 'batch'),
    ((1, True, 64), {}, 'kv_heads'),
    ((1, 1, 64.0), {}, 'capacity'),
    ((1, 1, 64), dict(head_dim=80), 'head_dim'),
])
def test_empty_cache_arguments(args, options, needle):
    with pytest.raises(ValueError, match=needle):
        lb.QuantizedKVCache.empty(*args, device='cpu', **options)


class HostCache(lb.QuantizedKVCache):
    """A cache on the host, past the constructor's device check, for the wrappers' own checks."""

    def __init__(self, dtype=torch.int8):
        for name, t in buffers(dtype=dtype).items():
            setattr(self, name, t)
        self.format, self.device = 'int8', torch.device('cpu')
        self.batch, self.kv_heads, self.head_dim, self.capacity = 2, 3, 64, 128
        self._bound()


def half(*shape, **options):
    return torch.zeros(shape, dtype=torch.float16, **options)


AT = torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize('call,needle', [
    (lambda c: lb.kv_append('cache', half(2, 1, 3, 64), half(2, 1, 3, 64), AT), 'QuantizedKVCache'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64).float(), half(2, 1, 3, 64), AT), 'k must be fp16'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64), half(2, 2, 3, 64), AT), 'v must be fp16'),
    (lambda c: lb.kv_append(c, half(1, 1, 3, 64), half(1, 1, 3, 64), AT), 'k must be fp16'),
    (lambda c: lb.kv_append(c, half(2, 0, 3, 64), half(2, 0, 3, 64), AT), 'k must be fp16'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64, device='meta'), half(2, 1, 3, 64), AT), 'k must be on'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64), half(2, 1, 3, 64), AT.int()), 'position must be'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64), half(2, 1, 3, 64), AT, rows=AT[:1]), 'rows must be'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64), half(2, 1, 3, 64), AT, cos=half(128, 64)), 'sin must be'),
    (lambda c: lb.kv_append(c, half(2, 1, 3, 64), half(2, 1, 3, 64), AT, cos=half(127, 64), sin=half(128, 64)), 'cos must be'),
    (lambda c: lb.kv_read(c, AT, start=128), 'capacity'),
    (lambda c: lb.kv_read(c, AT, start=100, count=29), 'capacity'),
    (lambda c: lb.kv_read(c, AT, count=5, keys=half(2, 3, 6, 64)), 'keys must be'),
    (lambda c: lb.kv_read(c, AT, count=5, values=half(2, 3, 64, 5).transpose(2, 3)), '16-byte'),
    (lambda c: lb.kv_attention(half(2, 1, 4, 64), c, AT), 'multiple of the kv_heads'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 32), c, AT), 'q must be'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, k=half(2, 1, 3, 64)), 'go together'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, scale=1e300), 'scale'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, scale=float('nan')), 'scale'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, scale=-0.1), 'scale'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, scale=1e6), 'scale'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, k=half(2, 2, 3, 64), v=half(2, 2, 3, 64)), 'k must be'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, out=half(2, 1, 64, 9).transpose(2, 3)), '16-byte'),
    (lambda c: lb.kv_attention(half(2, 1, 9, 64), c, AT, out=half(2, 2, 9, 64)), 'out must be'),
    (lambda c: lb.PreparedKVAppend(c, half(2, 1, 64, 3).transpose(2, 3), half(2, 1, 3, 64), AT), '16-byte'),
    (lambda c: lb.PreparedKVAttention(half(2, 1, 9, 64), c, AT, None), 'out must be'),
])
def test_wrappers_refuse(call, needle):
    with pytest.raises(ValueError, match=needle):
        call(HostCache())


def test_packed_structs_match_their_mirrors():
    for packed, mirror in ((lb._KV_APPEND, lb.KVAppendArgs), (lb._KV_READ, lb.KVReadArgs), (lb._KV_ATTENTION, lb.KVAttentionArgs)):
        assert lb._KV_HEAD.size + ctypes.sizeof(lb.KVCacheStruct) + packed.size == ctypes.sizeof(mirror)
    c = HostCache()
    a, need = lb._kv_attention_args(half(2, 1, 9, 64), c, AT, half(2, 1, 9, 64), None, None, None, 0.5, None, None, [], True)
    assert (a.struct_size, a.seq, a.heads, a.scale) == (ctypes.sizeof(a), 1, 9, 0.5)
    assert a.cache.capacity == 128 and a.cache.value_tail == c.value_tail.data_ptr() and a.q.head_stride == 64
    assert a.position == AT.data_ptr() and not a.rows and not a.k.data and need == 0


def test_struct_sizes_match_the_library():
    # A struct that is smaller than the library's is refused; these are the C layouts' sizes.
    assert ctypes.sizeof(lb.KVCacheStruct) == 8 + 3 * 8 + 6 * 8
    assert ctypes.sizeof(lb.KVRows) == 32
    assert ctypes.sizeof(lb.KVAppendArgs) == 8 + 80 + 8 + 64 + 32
    assert ctypes.sizeof(lb.KVReadArgs) == 8 + 80 + 24 + 64
    assert ctypes.sizeof(lb.KVAttentionArgs) == 8 + 80 + 16 + 64 + 32 + 64 + 8 + 16


def test_oracle_e4m3_is_the_format():
    """Every e4m3fn byte decodes to a value that rounds to itself, and midpoints go to the even byte."""
    bits = np.array([b for b in range(256) if b & 0x7F != 0x7F], np.uint8)
    values = torch.from_numpy(bits).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ko.e4m3(values), values) and np.array_equal(ko.e4m3_bits(values), bits)
    up = values[:126]
    mid = (up[:-1] + up[1:]) / 2
    even = np.where(bits[:125] % 2 == 0, up[:-1], up[1:])
    assert np.array_equal(ko.e4m3(mid), even)
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).integers(-12, 7, 20000))
    assert np.array_equal(ko.e4m3(x.astype(np.float32)), torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy())


def test_layer_cache_formats():
    import smollm_random
    from torch_npu_smollm import FrozenSmolLayer, FrozenSmolStack, _SHAPES
    config = smollm_random.config(theta=10000.0, layers=1)
    weights = {n: torch.zeros(s) if len(s) == 1 else torch.eye(*s) for n, s in _SHAPES.items()}
    with pytest.raises(ValueError, match='cache must be'):
        FrozenSmolLayer(config, weights, cache='int4')
    layers = [FrozenSmolLayer(config, weights, mode='fp16', cache=c) for c in ('fp16', 'fp8')]
    assert [layer.cache for layer in layers] == ['fp16', 'fp8'] and layers[1]._kv_capacity() == 64
    with pytest.raises(ValueError, match='cache format'):
        FrozenSmolStack.from_layers(layers)
    state = layers[0].__dict__
    del state['_cache_format']               # as a layer pickled before there was a choice
    assert layers[0].cache == 'fp16'


def test_the_buffers_are_fixed():
    """What calls are given was packed once: another tensor in place of a buffer is refused, copies have their own."""
    import copy
    import pickle
    cache = HostCache()
    with pytest.raises(AttributeError, match='fixed'):
        cache.key_codes = torch.zeros_like(cache.key_codes)
    for twin in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert twin.key_codes.data_ptr() != cache.key_codes.data_ptr()
        packed = bytes(twin._heads[lb.KVReadArgs])
        assert twin.key_codes.data_ptr().to_bytes(8, 'little') in packed
        assert cache.key_codes.data_ptr().to_bytes(8, 'little') not in packed


# Sizes whose products pass 64 bits: a cache of 2^64 bytes, rows of 2^24 + 1 strides of 2^40 elements (2^65 bytes and a row).
APART = {name: (1 + i) << 56 for i, name in enumerate((
    'cache__key_codes', 'cache__value_codes', 'cache__key_scales', 'cache__value_scales', 'cache__key_tail', 'cache__value_tail',
    'position'))}
VAST = dict(APART, cache__head_dim=128, cache__batch=1 << 14, cache__kv_heads=1 << 15, cache__capacity=1 << 28)
BEYOND = [
    ('lb_kv_append', append, dict(VAST, k__data=8 << 56, v__data=9 << 56)),
    ('lb_kv_read', read, {**{k: v for k, v in VAST.items() if k != 'position'}, 'keys__data': 8 << 56, 'values__data': 9 << 56,
                          'keys__batch_stride': 1 << 40, 'keys__head_stride': 1 << 20, 'values__batch_stride': 1 << 40,
                          'values__head_stride': 1 << 20}),
    ('lb_kv_append', append, dict(seq=(1 << 24) + 1, k__row_stride=1 << 40, k__data=1 << 56, v__data=2 << 56)),
    ('lb_kv_append', append, dict(seq=(1 << 24) + 1, v__row_stride=1 << 40, v__data=1 << 56, k__data=2 << 56)),
    ('lb_kv_read', read, dict(APART, cache__batch=1, cache__capacity=1 << 28, start=0, count=(1 << 24) + 1, keys__row_stride=1 << 40,
                              values__head_stride=1 << 40, keys__data=8 << 56, values__data=9 << 56)),
    ('lb_kv_attention', attention, dict(cache__batch=1, seq=(1 << 24) + 1, q__row_stride=1 << 40, q__data=1 << 56, out__data=2 << 56)),
    ('lb_kv_attention', attention, dict(cache__batch=1, seq=(1 << 24) + 1, out__row_stride=1 << 40, out__data=1 << 56,
                                        q__data=2 << 56)),
]
BEYOND[4][2].pop('position')


@pytest.mark.parametrize('entry,make,over', BEYOND, ids=[f'{entry}-{i}' for i, (entry, _, _) in enumerate(BEYOND)])
def test_sizes_past_the_address_space_are_refused(entry, make, over):
    """Every range is computed without overflow: what no memory can hold is refused, not taken for a short range."""
    lib = lb.library()
    assert getattr(lib, entry)(ctypes.byref(make(**over)), None) == lb.INVALID_ARGUMENT, lib.lb_last_error().decode()
    assert 'address space' in lib.lb_last_error().decode()


class Cleared(torch.utils._python_dispatch.TorchDispatchMode):
    """Bytes that operations under it fill with zeros."""
    bytes = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if any(word in func.__name__ for word in ('zero', 'fill')):
            self.bytes += out.numel() * out.element_size()
        return out


@pytest.mark.parametrize('captured', [True, False])
def test_a_workspace_is_cleared_no_further_than_its_counters(monkeypatch, captured):
    """The sums of parts behind LB_ZEROED_WORKSPACE_BYTES are written before they are read; a captured call's fill is
    repeated by every replay."""
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: captured)
    monkeypatch.setattr(lb, '_raw_stream', lambda device: 0)
    monkeypatch.setattr(lb, '_kv_workspaces', {})
    with Cleared() as cleared:
        workspace = lb._kv_workspace(5 << 20, torch.device('cpu'))
    assert workspace.numel() >= 5 << 20 and not bool(workspace[:4096].any())
    assert cleared.bytes == 4096
    again = lb._kv_workspace(1 << 20, torch.device('cpu'))
    assert (again is workspace) is not captured


def test_whether_a_call_is_captured_is_asked_of_its_own_device(monkeypatch):
    """The cache's device need not be the current one: its current stream is the one that may be capturing."""
    current = [0]

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.was, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.was
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: current[0])
    monkeypatch.setattr(torch.cuda, 'device', device)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: current[0] == 1)   # a capture on device 1
    monkeypatch.setattr(lb, '_raw_stream', lambda device: 0)
    monkeypatch.setattr(lb, '_kv_workspaces', {})
    monkeypatch.setattr(lb, '_kv_new_workspace', lambda need, device: torch.zeros(need, dtype=torch.uint8))
    for index, shared in ((1, False), (0, True)):
        first, second = (lb._kv_workspace(8192, torch.device('cuda', index)) for _ in range(2))
        assert (first is second) is shared, index
    assert [key[0].index for key in lb._kv_workspaces] == [0]
