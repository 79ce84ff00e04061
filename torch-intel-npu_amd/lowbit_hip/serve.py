"""Serving many requests at once (include/lowbit_decode_hip.h): rotary positions, a KV cache in pages with the attention that
reads it, and the low-rank adapters of many requests beside a shared projection.  Everything here is reached as
lowbit_hip.<name>; there is no CPU or PyTorch fallback."""
import ctypes
import math
import operator
import struct

import torch

from . import (OK, _aligned, _check, _kv_new_workspace, _kv_run, _kv_workspace, _PreparedKV, library)

PAGE_CHUNK = 16                                       # LB_PAGE_CHUNK: slots of a value dim that lie side by side
MAX_RANK = 128                                        # LB_ADAPTERS_MAX_RANK
ROTARY_MAX_DIMS = 1024                                # LB_ROTARY_MAX_DIMS
TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}   # lb_type
PAIRS = {'half': 0, 'neighbours': 1}                  # LB_PAIRS_*


class RowsStruct(ctypes.Structure):
    """Mirror of lb_rows."""
    _fields_ = [('data', ctypes.c_void_p), ('batch_stride', ctypes.c_int64), ('row_stride', ctypes.c_int64),
                ('head_stride', ctypes.c_int64)]


class RotationStruct(ctypes.Structure):
    """Mirror of lb_rotation."""
    _fields_ = [('frequencies', ctypes.c_void_p), ('dims', ctypes.c_uint32), ('pairs', ctypes.c_uint32),
                ('scale', ctypes.c_float), ('reserved', ctypes.c_uint32)]


class RotaryArgs(ctypes.Structure):
    """Mirror of lb_rotary_args."""
    _fields_ = [('struct_size', ctypes.c_uint32), ('type', ctypes.c_uint32), ('batch', ctypes.c_int64),
                ('seq', ctypes.c_int64), ('head_dim', ctypes.c_int64), ('heads', ctypes.c_int64),
                ('k_heads', ctypes.c_int64), ('q', RowsStruct), ('out', RowsStruct), ('k', RowsStruct),
                ('out_k', RowsStruct), ('position', ctypes.c_void_p), ('per_row', ctypes.c_uint32),
                ('back', ctypes.c_uint32), ('rotation', RotationStruct)]


class PagedCacheStruct(ctypes.Structure):
    """Mirror of lb_paged_cache."""
    _fields_ = [('type', ctypes.c_uint32), ('head_dim', ctypes.c_uint32), ('pages', ctypes.c_int64),
                ('kv_heads', ctypes.c_int64), ('page', ctypes.c_int64), ('keys', ctypes.c_void_p),
                ('values', ctypes.c_void_p)]


class PageTableStruct(ctypes.Structure):
    """Mirror of lb_page_table."""
    _fields_ = [('data', ctypes.c_void_p), ('stride', ctypes.c_int64), ('longest', ctypes.c_int64)]


class PagedAppendArgs(ctypes.Structure):
    """Mirror of lb_paged_append_args."""
    _fields_ = [('struct_size', ctypes.c_uint32), ('reserved', ctypes.c_uint32), ('cache', PagedCacheStruct),
                ('table', PageTableStruct), ('batch', ctypes.c_int64), ('seq', ctypes.c_int64), ('k', RowsStruct),
                ('v', RowsStruct), ('position', ctypes.c_void_p), ('rows', ctypes.c_void_p), ('rotation', RotationStruct)]


class PagedAttentionArgs(ctypes.Structure):
    """Mirror of lb_paged_attention_args."""
    _fields_ = [('struct_size', ctypes.c_uint32), ('reserved', ctypes.c_uint32), ('cache', PagedCacheStruct),
                ('table', PageTableStruct), ('batch', ctypes.c_int64), ('heads', ctypes.c_int64), ('q', RowsStruct),
                ('out', RowsStruct), ('position', ctypes.c_void_p), ('k', RowsStruct), ('v', RowsStruct),
                ('rotation', RotationStruct), ('scale', ctypes.c_float), ('reserved2', ctypes.c_uint32),
                ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_size_t)]


class AdaptersArgs(ctypes.Structure):
    """Mirror of lb_adapters_args."""
    _fields_ = [('struct_size', ctypes.c_uint32), ('type', ctypes.c_uint32), ('M', ctypes.c_int64), ('N', ctypes.c_int64),
                ('K', ctypes.c_int64), ('rank', ctypes.c_int64), ('count', ctypes.c_int64), ('down', ctypes.c_void_p),
                ('up', ctypes.c_void_p), ('scales', ctypes.c_void_p), ('index', ctypes.c_void_p), ('x', ctypes.c_void_p),
                ('ldx', ctypes.c_int64), ('y', ctypes.c_void_p), ('ldy', ctypes.c_int64), ('out', ctypes.c_void_p),
                ('ldo', ctypes.c_int64), ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_size_t)]


def declare(lib):
    """The signatures of the entry points, on the loaded library."""
    size = ctypes.POINTER(ctypes.c_size_t)
    for name, args in (('lb_rotary', RotaryArgs), ('lb_paged_append', PagedAppendArgs),
                       ('lb_paged_attention', PagedAttentionArgs), ('lb_adapters', AdaptersArgs)):
        getattr(lib, name).restype = ctypes.c_int
        getattr(lib, name).argtypes = [ctypes.POINTER(args), ctypes.c_void_p]
        if name in ('lb_paged_attention', 'lb_adapters'):
            getattr(lib, name + '_workspace_bytes').restype = ctypes.c_int
            getattr(lib, name + '_workspace_bytes').argtypes = [ctypes.POINTER(args), size]


# The argument structs packed in one go (nested ctypes fields cost a call several microseconds).
_ROTATION = struct.Struct('=QIIfI')                   # frequencies, dims, pairs, scale, 0
_ROTARY = struct.Struct('=IIqqqqq16qQII')             # size, type, batch, seq, head_dim, heads, k_heads; q, out, k, out_k; position, per_row, back
_PAGED_HEAD = struct.Struct('=II')
_PAGED_CACHE = struct.Struct('=IIqqqQQ')
_APPEND = struct.Struct('=Qqqqq8qQQ')                 # table, stride, longest; batch, seq; k, v; position, rows
_ATTENTION = struct.Struct('=Qqqqq8qQ8q')             # table, stride, longest; batch, heads; q, out; position; k, v
_ATTENTION_TAIL = struct.Struct('=fIQQ')              # scale, 0, workspace, bytes
_NO_ROWS = (0, 0, 0, 0)
_NO_ROTATION = _ROTATION.pack(0, 0, 0, 0.0, 0)


def _whole(value, name, low=1, high=None):
    if isinstance(value, bool) or not hasattr(value, '__index__') or value < low or (high is not None and value > high):
        raise ValueError(f'{name} must be an integer, {low} or more' + (f' up to {high}' if high is not None else ''))
    return operator.index(value)


def _rows(t, name, shape, dtype, device, keep, copy):
    """(address, batch, row and head strides) of a tensor of `shape` ([batch, seq, heads, dim]); where its rows are not whole
    16-byte pieces, of a copy (added to `keep`) if `copy`."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape:
        raise ValueError(f'{name} must be {dtype} {list(shape)}')
    if t.device != device:
        raise ValueError(f'{name} must be on {device} with the rest (found {t.device})')
    b, i, h, d = t.stride()
    at = t.data_ptr()
    if d != 1 or at % 16 or (b | i | h) % 8:
        if d != 1 or at % 16 or any(s % 8 and n > 1 for s, n in zip((b, i, h), shape)):
            if not copy:
                raise ValueError(f'the rows of {name} must be 16-byte pieces')
            t = _aligned(t)
            keep.append(t)
            b, i, h, _ = t.stride()
            at = t.data_ptr()
    return at, b, i, h


def _inference(what, *tensors):
    """No gradient is recorded, so none may be asked for."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f'{what} is inference-only; use no_grad/inference_mode')


def _counts(t, name, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f'{name} must be a contiguous int64 tensor {list(shape)}')
    if t.device != device:
        raise ValueError(f'{name} must be on {device} with the rest (found {t.device})')
    return t.data_ptr()


# ---------------------------------------------------------------- rotary positions
def rotary_frequencies(dims, theta=10000.0, *, factor=1.0, stretch=None, length=None, low=1.0, high=32.0, device=None):
    """The frequencies theta ** (-2 i / dims) of dims / 2 pairs, in 64 bits, stretched `factor` times for contexts longer than
    the `length` that a model was trained on:

      stretch='linear'  all of them divided by the factor;
      stretch='theta'   theta raised so that the slowest pair is divided by the factor, the others by less;
      stretch='parts'   pairs that make fewer than `low` turns over `length` positions are divided by the factor, those
                        that make more than `high` are kept, and those between are mixed in proportion to their turns.
    """
    dims = _whole(dims, 'dims', 2, ROTARY_MAX_DIMS)
    if dims % 2:
        raise ValueError('dims must be even')
    if stretch not in (None, 'linear', 'theta', 'parts'):
        raise ValueError("stretch must be None, 'linear', 'theta' or 'parts'")
    if not (math.isfinite(theta) and theta > 0) or not (math.isfinite(factor) and factor > 0):
        raise ValueError('theta and factor must be positive')
    if stretch == 'theta' and dims > 2:
        theta = theta * factor ** (dims / (dims - 2))
    f = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims)
    if stretch == 'linear' or (stretch == 'theta' and dims == 2):
        f = f / factor
    if stretch == 'parts':
        if length is None or not 0 < length or not 0 <= low < high:
            raise ValueError("stretch='parts' needs the length, and 0 <= low < high")
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


class Rotary:
    """How positions turn heads (lb_rotation): pair i of a head's first 2 len(frequencies) dims by the angle
    position * frequencies[i], cosines and sines times `scale`.  frequencies: float64 on the device (rotary_frequencies);
    pairs: 'half' (i, i + dims / 2) or 'neighbours' (2 i, 2 i + 1)."""

    def __init__(self, frequencies, *, pairs='half', scale=1.0):
        if (not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.float64 or frequencies.ndim != 1
                or not 1 <= frequencies.numel() <= ROTARY_MAX_DIMS // 2 or not frequencies.is_contiguous()):
            raise ValueError('frequencies must be a contiguous float64 vector')
        if frequencies.device.type != 'cuda':
            raise ValueError('frequencies must be a ROCm device tensor')
        if pairs not in PAIRS:
            raise ValueError("pairs must be 'half' or 'neighbours'")
        if not math.isfinite(scale):
            raise ValueError('scale must be finite')
        self.frequencies, self.pairs, self.scale = frequencies, pairs, float(scale)
        self.dims, self.device = 2 * frequencies.numel(), frequencies.device
        self._bound()

    def _bound(self):
        """What calls are given of it."""
        self.__dict__['_bytes'] = _ROTATION.pack(self.frequencies.data_ptr(), self.dims, PAIRS[self.pairs], self.scale, 0)

    def __setattr__(self, name, value):
        """Fixed: its address and values are in what calls are given."""
        if '_bytes' in self.__dict__:
            raise AttributeError(f'{name}: a Rotary is fixed; make another')
        super().__setattr__(name, value)

    def __getstate__(self):
        """Copies and pickles have frequencies of their own."""
        return {name: value for name, value in self.__dict__.items() if name != '_bytes'}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.__dict__['device'] = self.frequencies.device
        self._bound()

    def _packed(self, device, head_dim):
        if self.device != device:
            raise ValueError(f'the frequencies must be on {device} with the rest (found {self.device})')
        if self.dims > head_dim:
            raise ValueError(f'{self.dims} dims turn, but heads have {head_dim}')
        return self._bytes


def _rotation(rotary, device, head_dim):
    if rotary is None:
        return _NO_ROTATION
    if not isinstance(rotary, Rotary):
        raise ValueError('rotary must be a Rotary')
    return rotary._packed(device, head_dim)


def _head_rows(t, name, shape, dtype, device):
    """(address, strides) of rows of heads of contiguous values, at any alignment."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape:
        raise ValueError(f'{name} must be {dtype} [batch, seq, heads, head_dim] = {list(shape)}')
    if t.device != device:
        raise ValueError(f'{name} must be on {device} with q (found {t.device})')
    return _heads(t, name)


def _heads(t, name):
    b, i, h, d = t.stride()
    if d != 1 and t.shape[3] > 1:
        raise ValueError(f'the heads of {name} must be contiguous')
    return t.data_ptr(), b, i, h


def _rotary_args(q, position, rotary, out, k, out_k, back):
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype not in TYPES or q.ndim != 4 or q.numel() == 0:
        raise ValueError('q must be fp16, bf16 or fp32 [batch, seq, heads, head_dim] on a ROCm device')
    if not isinstance(rotary, Rotary):
        raise ValueError('rotary must be a Rotary')
    shape, dtype, device = q.shape, q.dtype, q.device
    batch, seq, heads, dim = shape
    if (k is None) != (out_k is None):
        raise ValueError('k and out_k go together')
    q, out = _heads(q, 'q'), _head_rows(out, 'out', shape, dtype, device)
    if k is None:
        k_heads, k, out_k = 0, _NO_ROWS, _NO_ROWS
    else:
        if not isinstance(k, torch.Tensor) or k.ndim != 4 or k.numel() == 0:
            raise ValueError(f'k must be {dtype} [batch, seq, heads, head_dim]')
        k_heads = k.shape[2]
        shape = (batch, seq, k_heads, dim)
        k, out_k = _head_rows(k, 'k', shape, dtype, device), _head_rows(out_k, 'out_k', shape, dtype, device)
    per_row = isinstance(position, torch.Tensor) and position.ndim == 2
    at = _counts(position, 'position', (batch, seq) if per_row else (batch,), device)
    return RotaryArgs.from_buffer_copy(_ROTARY.pack(
        ctypes.sizeof(RotaryArgs), TYPES[dtype], batch, seq, dim, heads, k_heads, *q, *out, *k, *out_k, at, per_row, bool(back))
        + rotary._packed(device, dim))


def rotary(q, position, rotary, *, k=None, out=None, out_k=None, back=False):
    """lb_rotary: the rows of q [batch, seq, heads, head_dim] (fp16, bf16 or fp32, any strides of contiguous heads) turned by
    their positions, and with k [batch, seq, k_heads, head_dim] its rows too, in one launch.  position: int64 [batch] (row i
    of sequence b lies at position[b] + i) or [batch, seq] (each row's own), on the device.  Into out and out_k, which may be
    q and k themselves (both or neither) or slices of one tensor; new tensors where they are not given.  back: by the negative angle, still times the
    scale, which is the transpose: of an output's gradient it makes the input's (autograd does not record
    the call).  Returns out, or (out, out_k)."""
    if out is None and isinstance(q, torch.Tensor):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out_k is None and isinstance(k, torch.Tensor):
        out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    a = _rotary_args(q, position, rotary, out, k, out_k, back)
    _kv_run(library().lb_rotary, a, q.device, 'lb_rotary')
    return out if k is None else (out, out_k)


class PreparedRotary(_PreparedKV):
    """A fixed lb_rotary call for hot loops: rotary's arguments over buffers that stay.  run() enqueues it on the current
    stream; positions are read on the device."""

    def __init__(self, q, position, rotary, out, *, k=None, out_k=None, back=False):
        a = _rotary_args(q, position, rotary, out, k, out_k, back)
        self._bind('lb_rotary', 'lb_rotary', a, q.device, [q, position, rotary, out, k, out_k])


# ---------------------------------------------------------------- a KV cache in pages
class PagedKVCache:
    """The pages of a KV cache of one layer (lb_paged_cache).  keys fp16 or bf16 [pages, kv_heads, page, D] (D 64 or 128;
    page 16, 32, .. 1024 slots), values [pages, kv_heads, page / 16, D, 16]: by chunks of 16 slots, the slots of a dim side
    by side.  Which pages a sequence has, the program says by a table, int32 [batch, pages of the longest] on the device:
    slot p of sequence b lies in page table[b, p // page].  Pages may be shared between sequences (a common prefix) as long
    as no two append into one."""

    def __init__(self, keys, values):
        if (not isinstance(keys, torch.Tensor) or keys.dtype not in (torch.float16, torch.bfloat16) or keys.ndim != 4
                or not keys.is_contiguous() or keys.data_ptr() % 16):
            raise ValueError('keys must be contiguous fp16 or bf16 [pages, kv_heads, page, head_dim]')
        pages, heads, page, dim = keys.shape
        if pages < 1 or heads < 1 or page not in (16, 32, 64, 128, 256, 512, 1024) or dim not in (64, 128):
            raise ValueError('keys must be [pages, kv_heads, page, head_dim] with page 16, 32, .. 1024 and head_dim 64 or 128')
        shape = (pages, heads, page // PAGE_CHUNK, dim, PAGE_CHUNK)
        if (not isinstance(values, torch.Tensor) or values.dtype != keys.dtype or values.shape != shape
                or not values.is_contiguous() or values.data_ptr() % 16):
            raise ValueError(f'values must be contiguous {keys.dtype} {list(shape)}')
        if keys.device.type != 'cuda' or values.device != keys.device:
            raise ValueError('keys and values must be on one ROCm device')
        self.keys, self.values, self.dtype, self.device = keys, values, keys.dtype, keys.device
        self.pages, self.kv_heads, self.page, self.head_dim = pages, heads, page, dim
        self._bound()

    def _bound(self):
        """What the calls' argument structs begin with."""
        cache = _PAGED_CACHE.pack(TYPES[self.dtype], self.head_dim, self.pages, self.kv_heads, self.page, self.keys.data_ptr(),
                                  self.values.data_ptr())
        heads = {args: _PAGED_HEAD.pack(ctypes.sizeof(args), 0) + cache for args in (PagedAppendArgs, PagedAttentionArgs)}
        self.__dict__.update(_heads=heads, _needs={})

    def __setattr__(self, name, value):
        """The buffers are fixed: their addresses are in what calls are given."""
        if '_heads' in self.__dict__:
            raise AttributeError(f'{name}: the buffers of a PagedKVCache are fixed; make another of other tensors')
        super().__setattr__(name, value)

    def __getstate__(self):
        """Copies and pickles have buffers of their own."""
        return {name: value for name, value in self.__dict__.items() if name not in ('_heads', '_needs')}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.device = self.keys.device
        self._bound()

    @classmethod
    def empty(cls, pages, kv_heads, *, page=64, head_dim=64, dtype=torch.float16, device='cuda'):
        """Pages of zeros."""
        pages, kv_heads = _whole(pages, 'pages', 1, 2 ** 31 - 1), _whole(kv_heads, 'kv_heads', 1, 65535)
        page = _whole(page, 'page', 16, 1024)
        if page & (page - 1) or head_dim not in (64, 128) or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError('page must be 16, 32, .. 1024, head_dim 64 or 128, and dtype fp16 or bf16')
        return cls(torch.zeros((pages, kv_heads, page, head_dim), dtype=dtype, device=device),
                   torch.zeros((pages, kv_heads, page // PAGE_CHUNK, head_dim, PAGE_CHUNK), dtype=dtype, device=device))

    def read(self, pages, length):
        """Keys and values [kv_heads, length, head_dim] of a sequence with these pages (int64 or int32 numbers, as a list or a
        tensor), in the order of its slots."""
        pages = torch.as_tensor(pages).reshape(-1).long()
        length = _whole(length, 'length', 0, pages.numel() * self.page)
        pages = pages[:-(-length // self.page)].to(self.device)     # (what stands behind them may be no page)
        if length and not bool(((pages >= 0) & (pages < self.pages)).all()):
            raise ValueError(f'pages must be 0 to {self.pages - 1}')
        keys = self.keys[pages].transpose(0, 1).reshape(self.kv_heads, pages.numel() * self.page, self.head_dim)
        values = self.values[pages].transpose(-1, -2).transpose(0, 1).reshape(self.kv_heads, pages.numel() * self.page, self.head_dim)
        return keys[:, :length].contiguous(), values[:, :length].contiguous()

    def nbytes(self):
        """Bytes of all pages."""
        return 2 * self.keys.numel() * self.keys.element_size()


def _paged_cache(cache):
    if not isinstance(cache, PagedKVCache):
        raise ValueError('cache must be a PagedKVCache')
    return cache


def _page_table(t, batch, device):
    if isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.ndim == 2:
        (rows, longest), (stride, step) = t.shape, t.stride()
        if rows == batch and longest >= 1 and (step == 1 or longest == 1):
            if t.device != device:
                raise ValueError(f'table must be on {device} with the cache (found {t.device})')
            return t.data_ptr(), stride, longest
    raise ValueError(f'table must be int32 [batch, pages] = [{batch}, pages] with contiguous rows')


def _append_args(cache, k, v, table, position, rows, rotary, keep, copy):
    cache = _paged_cache(cache)
    if not isinstance(k, torch.Tensor) or k.ndim != 4 or k.numel() == 0:
        raise ValueError('k must be [batch, seq, kv_heads, head_dim]')
    batch, seq, _, _ = k.shape
    device, dtype, dim = cache.device, cache.dtype, cache.head_dim
    shape, counts = (batch, seq, cache.kv_heads, dim), (batch,)
    a = PagedAppendArgs.from_buffer_copy(cache._heads[PagedAppendArgs] + _APPEND.pack(
        *_page_table(table, batch, device), batch, seq, *_rows(k, 'k', shape, dtype, device, keep, copy),
        *_rows(v, 'v', shape, dtype, device, keep, copy), _counts(position, 'position', counts, device),
        0 if rows is None else _counts(rows, 'rows', counts, device)) + _rotation(rotary, device, dim))
    _inference('paged_append', k, v)
    return a


def paged_append(cache, k, v, table, position, *, rows=None, rotary=None):
    """lb_paged_append: the first rows[b] (default: all) rows of k and v [batch, seq, kv_heads, head_dim] go to slots
    position[b] .. of each sequence, in the pages that the table gives them.  table: int32 [batch, pages], position and rows:
    int64 [batch], on the device.  With a Rotary the keys are turned by their slots first.  A sequence whose rows do not lie in
    the table's slots is left alone, as are rows whose entry is not a page.  k and v may have any strides (a copy is made where
    rows are not 16-byte pieces).  Inference only: rows that ask for a gradient are refused."""
    keep = []
    a = _append_args(cache, k, v, table, position, rows, rotary, keep, True)
    _kv_run(library().lb_paged_append, a, cache.device, 'lb_paged_append')


class PreparedPagedAppend(_PreparedKV):
    """A fixed lb_paged_append call for hot loops: paged_append's arguments over buffers that stay (no copies are made, so k
    and v need rows of 16-byte pieces).  run() enqueues it on the current stream; table and positions are read on the device."""

    def __init__(self, cache, k, v, table, position, *, rows=None, rotary=None):
        a = _append_args(cache, k, v, table, position, rows, rotary, None, False)
        self._bind('lb_paged_append', 'lb_paged_append', a, cache.device, [cache, k, v, table, position, rows, rotary])


def _needed(fn, what, args):
    size = ctypes.c_size_t(0)
    _check(fn(ctypes.byref(args), ctypes.byref(size)), what)
    return size.value


def _attention_args(q, cache, table, position, out, k, v, rotary, scale, keep, copy):
    """The argument struct without its workspace, and the bytes that it needs of one."""
    cache = _paged_cache(cache)
    if not isinstance(q, torch.Tensor) or q.ndim != 3 or q.numel() == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError(f'q must be [batch, heads, {cache.head_dim}], its heads a multiple of the kv_heads ({cache.kv_heads})')
    if (k is None) != (v is None):
        raise ValueError('k and v go together')
    batch, heads = q.shape[:2]
    device, dim = cache.device, cache.head_dim

    def rows(t, name, heads, copy):
        if not isinstance(t, torch.Tensor) or t.ndim != 3:
            raise ValueError(f'{name} must be {cache.dtype} {[batch, heads, dim]}')
        return _rows(t.unsqueeze(1), name, (batch, 1, heads, dim), cache.dtype, device, keep, copy)

    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError('scale must be finite')
    table, stride, longest = _page_table(table, batch, device)
    a = PagedAttentionArgs.from_buffer_copy(cache._heads[PagedAttentionArgs] + _ATTENTION.pack(
        table, stride, longest, batch, heads, *rows(q, 'q', heads, copy), *rows(out, 'out', heads, False),
        _counts(position, 'position', (batch,), device),
        *(_NO_ROWS if k is None else rows(k, 'k', cache.kv_heads, copy)),
        *(_NO_ROWS if v is None else rows(v, 'v', cache.kv_heads, copy)))
        + _rotation(rotary, device, dim) + _ATTENTION_TAIL.pack(scale, 0, 0, 0))
    _inference('paged_attention', q, k, v, out)
    need = cache._needs.get((batch, heads, longest))
    if need is None:
        need = _needed(library().lb_paged_attention_workspace_bytes, 'lb_paged_attention_workspace_bytes', a)
        if len(cache._needs) >= 256:
            cache._needs.clear()
        cache._needs[batch, heads, longest] = need
    return a, need


def paged_attention(q, cache, table, position, *, k=None, v=None, rotary=None, scale=None, out=None):
    """lb_paged_attention: one new token a sequence, q [batch, heads, head_dim], over the pages that the table gives its
    sequence.  The token of sequence b lies at slot position[b] and attends over slots 0 .. position[b], which the pages hold
    already, or get here where k and v [batch, kv_heads, head_dim] are given.  position -1: no token, its out is 0; a position
    that does not lie in the table, or a page that there is not, gives NaN.  With a Rotary q (and k) are turned by the position
    first.  table: int32 [batch, pages], position: int64 [batch], on the device; scale: default head_dim ** -0.5.  Any strides of
    q, k and v (a copy is made where rows are not 16-byte pieces).  Inference only: tensors that ask for a gradient are
    refused."""
    if out is None and isinstance(q, torch.Tensor):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    keep = []
    a, need = _attention_args(q, cache, table, position, out, k, v, rotary, scale, keep, True)
    if need:
        workspace = _kv_workspace(need, cache.device)   # (held until the call is enqueued, whoever replaces it)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    _kv_run(library().lb_paged_attention, a, cache.device, 'lb_paged_attention')
    return out


class PreparedPagedAttention(_PreparedKV):
    """A fixed lb_paged_attention call for hot loops: paged_attention's arguments over buffers that stay (with rows of 16-byte
    pieces).  Owns its workspace unless it is given one (zeros, that calls in order on one stream share), so calls of one
    instance must be ordered too."""

    def __init__(self, q, cache, table, position, out, *, k=None, v=None, rotary=None, scale=None, workspace=None):
        a, need = _attention_args(q, cache, table, position, out, k, v, rotary, scale, None, False)
        keep = [q, cache, table, position, out, k, v, rotary]
        if need:
            if workspace is None:
                workspace = _kv_new_workspace(need, cache.device)
            elif (not isinstance(workspace, torch.Tensor) or workspace.device != cache.device or workspace.dtype != torch.uint8
                  or workspace.numel() < need or not workspace.is_contiguous() or workspace.data_ptr() % 256):
                raise ValueError(f'the workspace must be {need} contiguous bytes (uint8) at a 256-byte address on {cache.device}')
            keep.append(workspace)
            a.workspace, a.workspace_bytes = workspace.data_ptr(), need
        self._bind('lb_paged_attention', 'lb_paged_attention', a, cache.device, keep)
        self.out, self.scratch = out, workspace


# ---------------------------------------------------------------- low-rank adapters
class Adapters:
    """Low-rank adapters of one projection (lb_adapters): adapter a adds scales[a] (x . down[a]^T) . up[a]^T to the rows that
    are its.  down [count, rank, K] and up [count, N, rank] fp16 or bf16, contiguous on the device, rank a multiple of 8 up to
    128, K a multiple of 8; scales: float32 [count], or None for 1."""

    def __init__(self, down, up, *, scales=None):
        if (not isinstance(down, torch.Tensor) or down.dtype not in (torch.float16, torch.bfloat16) or down.ndim != 3
                or not down.is_contiguous() or down.data_ptr() % 16 or down.numel() == 0 or down.shape[2] % 8):
            raise ValueError('down must be contiguous fp16 or bf16 [count, rank, K] with K a multiple of 8')
        count, rank, k = down.shape
        if rank % 8 or rank > MAX_RANK:
            raise ValueError(f'rank must be a multiple of 8 up to {MAX_RANK}')
        if (not isinstance(up, torch.Tensor) or up.dtype != down.dtype or up.ndim != 3 or up.shape[0] != count
                or up.shape[2] != rank or up.shape[1] < 1 or not up.is_contiguous() or up.data_ptr() % 16):
            raise ValueError(f'up must be contiguous {down.dtype} [count, N, rank] = [{count}, N, {rank}]')
        if down.device.type != 'cuda' or up.device != down.device:
            raise ValueError('down and up must be on one ROCm device')
        if scales is not None and (not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or scales.shape != (count,)
                                   or not scales.is_contiguous() or scales.device != down.device):
            raise ValueError(f'scales must be contiguous float32 [{count}] with the factors')
        self.down, self.up, self.scales = down, up, scales
        self.count, self.rank, self.N, self.K = count, rank, up.shape[1], k
        self.dtype, self.device = down.dtype, down.device
        self._bound()

    def _bound(self):
        """What calls are given of them, and the workspaces that calls need by their rows."""
        at = self.down.data_ptr(), self.up.data_ptr(), 0 if self.scales is None else self.scales.data_ptr()
        self.__dict__.update(_at=at, _needs={})

    def __setattr__(self, name, value):
        """The factors are fixed: their addresses are in what calls are given."""
        if '_at' in self.__dict__:
            raise AttributeError(f'{name}: the factors of Adapters are fixed (their contents are not); make others of other tensors')
        super().__setattr__(name, value)

    def __getstate__(self):
        """Copies and pickles have factors of their own."""
        return {name: value for name, value in self.__dict__.items() if name not in ('_at', '_needs')}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.__dict__['device'] = self.down.device
        self._bound()

    @classmethod
    def stack(cls, factors, *, scales=None, dtype=torch.float16, device='cuda'):
        """Adapters of (down [rank, K], up [N, rank]) pairs of any ranks up to 128, filled with zeros to the largest."""
        factors = list(factors)
        if not factors:
            raise ValueError('at least one adapter is required')
        for down, up in factors:
            if (down.ndim != 2 or up.ndim != 2 or down.shape[0] != up.shape[1] or not 1 <= down.shape[0] <= MAX_RANK
                    or down.shape[1] != factors[0][0].shape[1] or up.shape[0] != factors[0][1].shape[0]):
                raise ValueError(f'factors must be (down [rank, K], up [N, rank]) of one projection, rank up to {MAX_RANK}')
        rank = -(-max(down.shape[0] for down, _ in factors) // 8) * 8
        k, n = factors[0][0].shape[1], factors[0][1].shape[0]
        downs = torch.zeros((len(factors), rank, k), dtype=dtype, device=device)
        ups = torch.zeros((len(factors), n, rank), dtype=dtype, device=device)
        for i, (down, up) in enumerate(factors):
            downs[i, :down.shape[0]] = down
            ups[i, :, :up.shape[1]] = up
        if scales is not None:
            scales = torch.as_tensor(scales, dtype=torch.float32).to(downs.device).contiguous()
        return cls(downs, ups, scales=scales)


_ADAPTERS = struct.Struct('=IIqqqqqQQQQQqQqQqQQ')    # size, type, M, N, K, rank, count; down, up, scales, index; x, ldx, y, ldy, out, ldo; workspace, bytes


def _adapters_args(y, x, adapters, index, out, keep, copy):
    """The argument struct without its workspace, and the bytes that it needs of one."""
    if not isinstance(adapters, Adapters):
        raise ValueError('adapters must be Adapters')
    N, K, dtype, device = adapters.N, adapters.K, adapters.dtype, adapters.device
    if not isinstance(x, torch.Tensor) or x.dtype != dtype or x.ndim != 2 or x.shape[1] != K or x.shape[0] < 1:
        raise ValueError(f'x must be {dtype} [M, {K}]')
    M = x.shape[0]
    places = []
    for t, name in ((y, 'y'),) if out is y else ((y, 'y'), (out, 'out')):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != (M, N):
            raise ValueError(f'{name} must be {dtype} [{M}, {N}]')
        if t.device != device:
            raise ValueError(f'{name} must be on {device} with the adapters (found {t.device})')
        ld, step = t.stride()
        if step != 1 and N > 1:
            raise ValueError(f'the rows of {name} must be contiguous')
        places += (t.data_ptr(), ld)
    if x.device != device:
        raise ValueError(f'x must be on {device} with the adapters (found {x.device})')
    at = _counts(index, 'index', (M,), device)
    ldx, step = x.stride()
    if step != 1 or x.data_ptr() % 16 or (M > 1 and ldx % 8):
        if not copy:
            raise ValueError('the rows of x must be 16-byte pieces')
        x = _aligned(x)
        keep.append(x)
        ldx = x.stride(0)
    a = AdaptersArgs.from_buffer_copy(_ADAPTERS.pack(_ADAPTERS.size, TYPES[dtype], M, N, K, adapters.rank, adapters.count, *adapters._at, at,
                                                     x.data_ptr(), ldx, *places[:2], *places[-2:], 0, 0))
    _inference('adapters_add', x, y, out, adapters.down, adapters.up, adapters.scales)
    need = adapters._needs.get(M)
    if need is None:
        need = _needed(library().lb_adapters_workspace_bytes, 'lb_adapters_workspace_bytes', a)
        if len(adapters._needs) >= 256:
            adapters._needs.clear()
        adapters._needs[M] = need
    return a, need


def adapters_add(y, x, adapters, index, *, out=None):
    """lb_adapters: adds to the rows of y [M, N], a projection of x [M, K], what the adapter of each adds to it:
    y[m] + scales[a] (x[m] . down[a]^T) . up[a]^T with a = index[m] (int64 on the device; -1: none, the row stays; any other
    number that is no adapter: NaN).  In place, or into out.  Inference only: tensors and factors that ask for a gradient are
    refused."""
    out = y if out is None else out
    keep = []
    a, need = _adapters_args(y, x, adapters, index, out, keep, True)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=adapters.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    _kv_run(library().lb_adapters, a, adapters.device, 'lb_adapters')
    return out


class PreparedAdapters(_PreparedKV):
    """A fixed lb_adapters call for hot loops: adapters_add's arguments over buffers that stay (x with rows of 16-byte pieces).
    run() enqueues it on the current stream; adapter numbers are read on the device.  Owns its workspace, so calls of one
    instance must be ordered."""

    def __init__(self, y, x, adapters, index, out=None):
        out = y if out is None else out
        a, need = _adapters_args(y, x, adapters, index, out, None, False)
        keep = [y, x, adapters, index, out]
        if need:
            keep.append(torch.empty(need, dtype=torch.uint8, device=adapters.device))
            a.workspace, a.workspace_bytes = keep[-1].data_ptr(), need
        self._bind('lb_adapters', 'lb_adapters', a, adapters.device, keep)
        self.out = out
