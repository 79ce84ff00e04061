"""What a call's workspace says of how it will be run, by the library's own host code."""
import ctypes

import pytest

import lowbit_hip as lb
from test_serve_cpu import attention


def workspace(fn, a):
    size = ctypes.c_size_t(1)
    assert getattr(lb.library(), fn)(ctypes.byref(a), ctypes.byref(size)) == 0
    return size.value


@pytest.mark.parametrize('dim,whole', [(64, 1024), (128, 512)])
@pytest.mark.parametrize('batch,page', [(1, 16), (2, 32), (40, 16), (300, 64)])
def test_attention_over_short_tables(dim, whole, batch, page):
    """Sequences that are never split need no workspace; a page more, and they do."""
    of = lambda slots: workspace('lb_paged_attention_workspace_bytes', attention(
        cache__head_dim=dim, cache__page=page, batch=batch, table__longest=slots // page, table__stride=slots // page))
    assert of(page) == of(whole - page) == of(whole) == 0
    assert of(whole + page) == of(8 * whole) > lb.ZEROED_WORKSPACE_BYTES
