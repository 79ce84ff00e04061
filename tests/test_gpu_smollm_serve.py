"""SmolBatchDecoder: requests of their own lengths and adapters in one batch, against the CPU oracle's decoder of each request by
itself (fed the same tokens), with low-rank adapters as the definition adds them.

Bar: logits rel-L2 1e-2, the decoder bar (the batch's attention has fp32 scores and 64-bit angles where the oracle has the
reference's fp16 ones; the operators' own errors are tested in test_gpu_paged, test_gpu_rotary and test_gpu_adapters).
"""
import math

import pytest
import torch

import lowbit_hip as lb
import smollm_random
from conftest import announce
from oracle import smollm_oracle as so
from torch_npu_lowbit import QuantizedLinear, quantize_weight
from torch_npu_smollm import FrozenSmolLayer, FrozenSmolStack, _SHAPES
from torch_npu_smollm_io import FrozenSmolIO
from torch_npu_smollm_serve import SmolBatchDecoder

pytestmark = pytest.mark.gpu
CONFIG = {**smollm_random.config(theta=10000.0, layers=2), 'vocab_size': 1000}


class AdaptedLayer(so.OracleLayer):
    """The oracle's layer with one request's factors beside its projections: name -> (down, up, scale)."""
    factors = {}

    def linear(self, v, name):
        y = super().linear(v, name)
        if name in self.factors:
            down, up, scale = self.factors[name]
            y = (y.double() + scale * (v.double() @ down.double().T @ up.double().T)).half()
        return y


def make(device, mode, corrections=False, seed=11, capacity=96):
    g = torch.Generator().manual_seed(seed)
    layers, oracles = [], []
    for _ in range(2):
        w = {n: (torch.randn(s, generator=g) * .04).half() if len(s) == 2 else (1 + torch.randn(s, generator=g) * .1).half()
             for n, s in _SHAPES.items()}
        layer = FrozenSmolLayer(CONFIG, w, mode=mode, capacity=capacity)
        layers.append(layer)
        oracles.append(AdaptedLayer(w, {n: (q.format, q.shape, q.group_size, q.data, q.scales) for n, q in layer._packed.items()},
                                    theta=10000.0, capacity=capacity))
    embedding, norm = torch.randn(1000, 576, generator=g) * .5, 1 + torch.randn(576, generator=g) * .1
    stack, io = FrozenSmolStack.from_layers(layers), FrozenSmolIO(CONFIG, embedding, norm).to(device)
    return stack, io, so.OracleModel(oracles, embedding, norm), g


def make_adapters(device, g, count=3):
    """Per layer, by projection (the second layer has them beside three alone): on the device, and each adapter's own factors."""
    held, factors = [], [[{} for _ in range(2)] for _ in range(count)]
    for i in range(2):
        layer = {}
        for name in (so.PROJECTIONS if i == 0 else so.PROJECTIONS[1:4]):
            n, k = _SHAPES[name]
            pairs = [((torch.randn(r, k, generator=g) * .05).half(), (torch.randn(n, r, generator=g) * .1).half()) for r in (8, 3, 16)[:count]]
            scales = [1.0, 0.5, 2.0][:count]
            layer[name] = lb.Adapters.stack(pairs, scales=scales, device=device)
            for a, (down, up) in enumerate(pairs):
                factors[a][i][name] = (down, up, scales[a])
        held.append(layer)
    return held, factors


def logits_of(model, factors, adapter, ids, tokens):
    """The oracle's logits after the prompt and after each of the tokens but the last."""
    for i, layer in enumerate(model.layers):
        layer.factors = {} if adapter < 0 else factors[adapter][i]
    return model.generate(torch.tensor([ids]), len(tokens), forced=tokens)[1]


def rel_l2(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize('mode,graph', [('w8a16', True), ('w4a16', False), ('fp16', True)])
def test_requests_of_their_own_lengths_and_adapters(device, mode, graph):
    """Four requests, admitted at different times; one ends and another takes its place and pages."""
    announce('smollm serve', mode, graph)
    stack, io, model, g = make(device, mode)
    held, factors = make_adapters(device, g)
    decoder = SmolBatchDecoder(stack, io, batch=3, slots=90, page=16, pages=11, adapters=held, graph=graph)
    prompt = lambda n: torch.randint(0, 1000, (n,), generator=g).tolist()
    plan = {0: [(prompt(5), -1, 12), (prompt(33), 0, 9)], 4: [(prompt(17), 2, 15)], 9: [(prompt(31), 1, 8)]}   # by step
    live, done = {}, []
    for step in range(17):
        for ids, adapter, steps in plan.get(step, ()):
            place = decoder.admit(ids, steps=steps, adapter=adapter)
            live[place] = dict(ids=ids, adapter=adapter, steps=steps, tokens=[int(decoder.tokens[place])], logits=[])
        before = decoder.tokens.clone()
        tokens = decoder.step()
        assert tokens is decoder.tokens
        for place in range(3):
            if place not in live:
                assert int(tokens[place]) == -1 == int(before[place]) == int(decoder.position[place])
                continue
            r = live[place]
            r['tokens'].append(int(tokens[place]))
            r['logits'].append(decoder.logits[place].cpu())
            assert r['tokens'][-1] == int(decoder.logits[place].argmax())
            if len(r['logits']) == r['steps']:
                decoder.release(place)
                done.append(live.pop(place))
    assert len(done) == 3 and len(live) == 1 and len(decoder._free) == 11 - 2
    for r in done + list(live.values()):
        want = logits_of(model, factors, r['adapter'], r['ids'], r['tokens'])
        assert rel_l2(torch.stack(r['logits']), want[1:]) <= 1e-2, (len(r['ids']), r['adapter'])
        top = want[0].float().topk(2).values
        assert r['tokens'][0] == int(want[0].float().argmax()) or float(top[0] - top[1]) < 0.05 * float(want[0].float().std())
    # The adapters matter: without them the logits are others.
    r = next(r for r in done if r['adapter'] == 0)
    assert rel_l2(logits_of(model, factors, 0, r['ids'], r['tokens']), logits_of(model, factors, -1, r['ids'], r['tokens'])) > 0.1


def test_a_batch_is_its_requests(device):
    """The same request alone and among others, replayed and eager: the same tokens, and logits to a rounding of a few steps (other
    row counts take other kernels of the projections)."""
    announce('smollm serve batch')
    stack, io, _, g = make(device, 'w8a16', seed=12)
    ids = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (40, 7, 23)]
    runs = []
    for batch, graph in ((1, True), (8, True), (8, False)):
        decoder = SmolBatchDecoder(stack, io, batch=batch, slots=64, page=32, graph=graph)
        place = decoder.admit(ids[0], steps=10)
        for other in ids[1:] if batch > 1 else ():
            decoder.admit(other, steps=10)
        logits = []
        for _ in range(10):
            decoder.step()
            logits.append(decoder.logits[place].clone())
        runs.append(torch.stack(logits))
    assert torch.equal(runs[1], runs[2])
    assert rel_l2(runs[0], runs[1]) <= 1e-2


def test_refusals(device):
    announce('smollm serve refusals')
    stack, io, _, g = make(device, 'w8a16', capacity=32)
    held, _ = make_adapters(device, g)
    for options in (dict(batch=0), dict(slots=0), dict(page=24), dict(pages=0), dict(adapters=[{}]), dict(adapters=[{}, {}]),
                    dict(adapters=[held[0], {'x': held[0][so.PROJECTIONS[0]]}]),
                    dict(adapters=[{so.PROJECTIONS[1]: held[0][so.PROJECTIONS[0]]}, {}])):
        with pytest.raises(ValueError):
            SmolBatchDecoder(stack, io, graph=False, **options)
    eight = FrozenSmolStack.from_layers([FrozenSmolLayer(CONFIG, stack.layers[0]._weights, mode='fp16', cache='int8')])
    with pytest.raises(ValueError, match='fp16'):
        SmolBatchDecoder(eight, io, graph=False)
    decoder = SmolBatchDecoder(stack, io, batch=2, slots=40, page=16, pages=4, graph=False)
    with pytest.raises(ValueError, match='no request'):
        decoder.step()
    for ids, options in (([], {}), (list(range(33)), {}), ([1, 2], dict(steps=39)), ([1], dict(steps=-1)), ([1], dict(adapter=0))):
        with pytest.raises(ValueError):
            decoder.admit(ids, **{'steps': 1, **options})
    a = decoder.admit([1, 2, 3], steps=30)               # 3 pages
    with pytest.raises(ValueError, match='pages'):
        decoder.admit([4], steps=16)                     # 2 pages
    b = decoder.admit([4], steps=1)
    with pytest.raises(ValueError, match='no place'):
        decoder.admit([4], steps=1)
    decoder.step()
    with pytest.raises(ValueError, match=f'\\[{b}\\]'):
        decoder.step()
    decoder.release(b)
    for place in (b, 5, -1, 'x'):
        with pytest.raises(ValueError, match='holds no request'):
            decoder.release(place)
    decoder.step()
    decoder.release(a)
    assert sorted(decoder._free) == [0, 1, 2, 3]


def test_prompts_that_are_none(device):
    """Tokens outside the vocabulary, two rows and numbers that are not whole are refused before anything is enqueued."""
    announce('smollm serve prompts')
    stack, io, _, _ = make(device, 'w8a16', capacity=32)
    decoder = SmolBatchDecoder(stack, io, batch=1, slots=32, page=16, graph=False)
    for ids in ([-1], [io.vocab_size], [[1], [2]], [1.5], torch.tensor([1], dtype=torch.int32), torch.tensor([[[1]]])):
        with pytest.raises(ValueError, match='tokens'):
            decoder.admit(ids, steps=1)
    assert sorted(decoder._free) == [0, 1]
    place = decoder.admit(torch.tensor([[1, io.vocab_size - 1]], device=device), steps=1)
    decoder.step()
    decoder.release(place)


def test_operators_together(device):
    """Rotary, append, attention and adapters in the order in which a layer uses them, against each other's definitions: a prompt
    appended, then tokens one at a time, equal a token's attention over all of its rows turned by lb_rotary."""
    announce('serving operators together')
    g = torch.Generator().manual_seed(13)
    rows, heads, kv, dim = 70, 6, 2, 64
    r = lambda *shape: torch.randn(shape, generator=g).half().to(device)
    q, k, v = r(1, rows, heads, dim), r(1, rows, kv, dim), r(1, rows, kv, dim)
    rotary = lb.Rotary(lb.rotary_frequencies(dim, device=device))
    table, start = torch.tensor([[3, 0, 4, 1, 2]], dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int64, device=device)
    cache = lb.PagedKVCache.empty(5, kv, page=16, device=device)
    lb.paged_append(cache, k[:, :60], v[:, :60], table, start, rotary=rotary)
    turned_q, turned_k = lb.rotary(q, start, rotary, k=k)
    for i in range(60, rows):
        out = lb.paged_attention(q[:, i], cache, table, start + i, k=k[:, i], v=v[:, i], rotary=rotary)
        s = torch.einsum('hd,khd->hk', turned_q[0, i].cpu().double(), turned_k[0, :i + 1].cpu().double().repeat_interleave(3, 1)) * dim ** -0.5
        want = torch.einsum('hk,khd->hd', s.softmax(-1), v[0, :i + 1].cpu().double().repeat_interleave(3, 1))
        # q as lb_rotary rounds it: 2^-11 of the products of a score, at most R of them; then the probabilities' rounding to fp16, in
        # the sum and in the total, the output's, and what is left in 32 bits (a hundredth of those)
        R = float((turned_q[0, i].abs().double() @ turned_k[0, :i + 1].abs().double().flatten(0, 1).amax(0))[..., None].max()) * dim ** -0.5
        near = (2 * math.expm1(2.0 ** -11 * R) + 3.1 * 2.0 ** -11) * float(v.abs().max())
        assert float((out[0].cpu().double() - want).abs().max()) <= near
    keys, values = cache.read(table[0], rows)
    assert torch.equal(values, v[0].transpose(0, 1))
    assert float((keys - turned_k[0].transpose(0, 1)).abs().max()) <= 2.0 ** -10 * float(k.abs().max()) * 2


def test_quantized_linear_with_adapters(device):
    """The module beside its adapters: its own output where a row has none, and theirs added where it has."""
    announce('quantized linear adapters')
    g = torch.Generator().manual_seed(14)
    weight = quantize_weight(torch.randn(192, 128, generator=g) * .05, format='int4', group_size=32)
    linear = QuantizedLinear(weight)
    x = torch.randn(9, 128, generator=g).half().to(device)
    down, up = (torch.randn(2, 8, 128, generator=g) * .1).half().to(device), (torch.randn(2, 192, 8, generator=g) * .1).half().to(device)
    adapters, index = lb.Adapters(down, up), torch.tensor([0, -1, 1, 1, 0, -1, -1, 0, 1], device=device)
    plain, got = linear(x), linear(x, adapters, index)
    none = index < 0
    assert torch.equal(got[none], plain[none])
    want = plain.double()
    for m in range(9):
        if int(index[m]) >= 0:
            want[m] += up[index[m]].double() @ (down[index[m]].double() @ x[m].double())
    # half a step of the output and of the sums in 32 bits (128 + 16 products)
    assert bool(((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16 * 8).all())
    with pytest.raises(ValueError, match='together'):
        linear(x, adapters)
    with pytest.raises(ValueError, match='x must'):
        linear(x, lb.Adapters(down[:, :, :64].contiguous(), up), index)
