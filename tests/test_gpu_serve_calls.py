"""Serving calls as servers make them: batches of hundreds of sequences, other signs of the scale, pages listed twice, host threads, and
captured calls replayed beside eager ones (bounds as test_gpu_paged derives them)."""
import threading

import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce
from oracle import serve_oracle as so
from test_gpu_adapters import make
from test_gpu_paged import check, filled, forget, host, ints, rand, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('type,heads,kv,dim,batch,long', [
    ('fp16', 3, 1, 64, 300, 3000), ('bf16', 6, 2, 128, 257, 1500), ('fp16', 9, 3, 64, 1100, 40), ('bf16', 20, 1, 64, 129, 5000),
    ('fp16', 2, 2, 128, 65, 9000)])
def test_hundreds_of_sequences(device, type, heads, kv, dim, batch, long):
    """Lengths of all kinds, a long one at each end and places without a token between; nothing that is not held is looked at."""
    announce('serve hundreds', type, heads, kv, dim, batch, long)
    page = 16
    lengths = [1 + (b * 7919) % 50 for b in range(batch)]
    lengths[0] = lengths[-1] = lengths[batch // 2] = long
    pages = sum(-(-n // page) for n in lengths) + 1
    cache, table = filled(device, type, pages, kv, page, dim, seed=61), table_of(device, lengths, page, pages, wide=2)
    forget(cache, table, lengths)
    position = [n - 1 for n in lengths]
    none = list(range(5, batch, 9))
    q, at = rand(device, type, batch, heads, dim, seed=62), ints(position, device)
    at[none] = -1
    out = lb.paged_attention(q, cache, table, at)
    there = [b for b in range(batch) if b not in set(none)]
    assert not bool(out[none].any())
    check(out[there], q[there], cache, table[there].cpu(), [position[b] for b in there], dim ** -0.5, type)
    assert torch.equal(out, lb.paged_attention(q, cache, table, at))


@pytest.mark.parametrize('type', ['fp16', 'bf16'])
@pytest.mark.parametrize('scale,turn', [(-0.2, 1.0), (0.3, -0.5), (-0.1, -1.5)])
def test_negative_scales(device, type, scale, turn):
    """Of the scores and of the rotation."""
    announce('serve negative scales', type, scale, turn)
    lengths, page, dim = [70, 700], 32, 64
    cache, table = filled(device, type, 30, 2, page, dim, seed=63), table_of(device, lengths, page, 30)
    rotary = lb.Rotary(lb.rotary_frequencies(dim, device=device), scale=turn)
    q, k, v = rand(device, type, 2, 6, dim, seed=64), rand(device, type, 2, 2, dim, seed=65), rand(device, type, 2, 2, dim, seed=66)
    out = lb.paged_attention(q, cache, table, ints([69, 699], device), k=k, v=v, rotary=rotary, scale=scale)
    q64 = so.turned(host(q)[:, None], np.array([[69], [699]]), rotary.frequencies.cpu().numpy(), 'half', turn)[:, 0]
    check(out, q64, cache, table.cpu(), [69, 699], scale, type, True)


def test_a_page_listed_twice(device):
    """It holds both ranges of the sequence's slots."""
    announce('serve page twice')
    cache, table = filled(device, 'fp16', 4, 2, 16, 64, seed=67), ints([[3, 1, 3, 3, 0]], device).int()
    q = rand(device, 'fp16', 1, 4, 64)
    check(lb.paged_attention(q, cache, table, ints([75], device)), q, cache, table.cpu(), [75], 0.125, 'fp16')


def test_host_threads(device):
    """Threads with streams of their own, and two on one stream, over the same cache, adapters and rotation."""
    announce('serve threads')
    lengths = [3000, 900, 20]
    cache, table = filled(device, 'fp16', 300, 2, 16, 64, seed=68), table_of(device, lengths, 16, 300)
    position, q = ints([n - 1 for n in lengths], device), rand(device, 'fp16', 3, 6, 64)
    x, y, adapters = make(device, 'fp16', 40, 264, 4104, 32, 4)
    index, rotary = torch.arange(40, device=device) % 5 - 1, lb.Rotary(lb.rotary_frequencies(64, device=device))

    def calls():
        return (lb.paged_attention(q, cache, table, position), lb.adapters_add(y, x, adapters, index, out=torch.empty_like(y)),
                lb.rotary(q[:, None], position, rotary))

    want = calls()
    torch.cuda.synchronize()
    shared, results, errors = torch.cuda.Stream(), {}, []

    def work(name, stream):
        try:
            with torch.cuda.stream(stream):
                results[name] = [calls() for _ in range(20)]
            stream.synchronize()
        except Exception as e:             # (said by the test, not by the thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i, shared if i < 2 else torch.cuda.Stream())) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and len(results) == 4
    for got in results.values():
        for turn in got:
            assert all(torch.equal(a, b) for a, b in zip(turn, want))


def test_replays_beside_eager_calls(device):
    """A captured call with parts, replayed on a stream of its own while eager ones go on over the same cache on another."""
    announce('serve replays')
    cache, table = filled(device, 'bf16', 300, 2, 16, 128, seed=69), table_of(device, [4000, 600], 16, 300)
    q, position = rand(device, 'bf16', 2, 8, 128), ints([3999, 599], device)
    want = lb.paged_attention(q, cache, table, position)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lb.paged_attention(q, cache, table, position)
    side = torch.cuda.Stream()
    for _ in range(4):
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        eager = []
        with torch.cuda.stream(side):
            for _ in range(5):
                graph.replay()
        for _ in range(5):
            eager.append(lb.paged_attention(q, cache, table, position))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(e, want) for e in eager)


def test_workspaces_that_are_none(device):
    """Too short, of another type, of bytes that do not lie side by side (an expanded byte is one), or at any address: refused when the call
    is prepared."""
    announce('serve workspaces')
    cache, table = filled(device, 'fp16', 70, 2, 16, 128, seed=70), table_of(device, [1000], 16, 70)
    q, position = rand(device, 'fp16', 1, 4, 128), ints([999], device)
    prepare = lambda workspace: lb.PreparedPagedAttention(q, cache, table, position, torch.zeros_like(q), workspace=workspace)
    need = prepare(None).scratch.numel()
    zeros = lambda n, dtype=torch.uint8: torch.zeros(n, dtype=dtype, device=device)
    for bad in (zeros(need - 1), zeros(need, torch.int8), zeros(1).expand(need), zeros(2 * need)[::2], zeros(need + 16)[16:], torch.zeros(need, dtype=torch.uint8),
                need):
        with pytest.raises(ValueError, match='workspace must'):
            prepare(bad)
    call = prepare(zeros(need + 256)[256:])
    call.run()
    check(call.out, q, cache, table.cpu(), [999], 128 ** -0.5, 'fp16')
