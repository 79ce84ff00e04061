"""Serving calls record no gradient: where one is asked for they refuse instead of dropping it, and leave their operands as they are."""
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from torch_npu_lowbit import QuantizedLinear, quantize_weight

pytestmark = pytest.mark.gpu


def rand(device, *shape, seed=1):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).half().to(device)


def refused(call):
    with pytest.raises(ValueError, match='inference-only'):
        call()


@pytest.mark.parametrize('which', ['x', 'y', 'down', 'up', 'scales', 'out'])
def test_adapters(device, which):
    announce('grad adapters', which)
    t = dict(x=rand(device, 5, 64), y=rand(device, 5, 72, seed=2), down=rand(device, 2, 8, 64, seed=3), up=rand(device, 2, 72, 8, seed=4),
             scales=torch.ones(2, device=device), out=torch.zeros((5, 72), dtype=torch.float16, device=device))
    index = torch.tensor([0, 1, -1, 0, 1], device=device)
    before = {name: v.clone() for name, v in t.items()}
    t[which].requires_grad_()
    adapters = lb.Adapters(t['down'], t['up'], scales=t['scales'])
    refused(lambda: lb.adapters_add(t['y'], t['x'], adapters, index, out=t['out']))
    refused(lambda: lb.PreparedAdapters(t['y'], t['x'], adapters, index, t['out']))
    if which in ('down', 'up', 'scales'):
        linear = QuantizedLinear(quantize_weight(torch.randn(72, 64), format='int8', group_size=64))
        refused(lambda: linear(t['x'], adapters, index))
    torch.cuda.synchronize()
    assert all(torch.equal(t[name], before[name]) for name in t)
    for context in (torch.no_grad, torch.inference_mode):
        with context():
            out = lb.adapters_add(t['y'], t['x'], adapters, index, out=torch.zeros_like(before['out']))
            want = lb.adapters_add(before['y'], before['x'], lb.Adapters(before['down'], before['up'], scales=before['scales']), index,
                                   out=torch.zeros_like(before['out']))
            assert torch.equal(out, want)


@pytest.mark.parametrize('which', ['q', 'k', 'v'])
def test_pages(device, which):
    announce('grad pages', which)
    cache = lb.PagedKVCache.empty(3, 2, page=16, device=device)
    t = dict(q=rand(device, 1, 4, 64), k=rand(device, 1, 2, 64, seed=2), v=rand(device, 1, 2, 64, seed=3))
    t[which].requires_grad_()
    table, position = torch.tensor([[0, 2]], dtype=torch.int32, device=device), torch.tensor([0], device=device)
    refused(lambda: lb.paged_attention(t['q'], cache, table, position, k=t['k'], v=t['v']))
    refused(lambda: lb.PreparedPagedAttention(t['q'], cache, table, position, torch.empty_like(t['q']).detach(), k=t['k'], v=t['v']))
    if which != 'q':
        refused(lambda: lb.paged_append(cache, t['k'][:, None], t['v'][:, None], table, position))
        refused(lambda: lb.PreparedPagedAppend(cache, t['k'][:, None], t['v'][:, None], table, position))
    torch.cuda.synchronize()
    assert not bool(cache.keys.any()) and not bool(cache.values.any())
    with torch.no_grad():
        out = lb.paged_attention(t['q'], cache, table, position, k=t['k'], v=t['v'])
    assert torch.equal(out, t['v'].detach().repeat_interleave(2, 1))
