"""SmolLM layers with the KV cache in 8 bits: prefill and decode against the CPU oracle's layer with its attention over the
held values (64 bits), snapshots, and a snapshot taken over by GraphDecoder.

Bar: rel-L2 1e-2, the decoder bar (the layer's stages round to fp16 as the oracle's do; the attention's own error is
tested in test_gpu_kv.py).  What is read back is compared with the rows' own quantisation bit for bit, where the rows are
the device's.
"""
import copy
import pickle

import numpy as np
import pytest
import torch

import lowbit_hip as lb
import smollm_random
from conftest import announce
from oracle import kv_oracle as ko
from oracle import smollm_oracle as so
from torch_npu_smollm import FrozenSmolLayer, FrozenSmolStack, GraphDecoder, generate_greedy, SmolQuantizedKVCache, _SHAPES
from torch_npu_smollm_io import FrozenSmolIO

pytestmark = pytest.mark.gpu
CONFIG = smollm_random.config(theta=10000.0, layers=1)


def rel_l2(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / b.norm())


def make(mode, format, capacity, seed=5):
    g = torch.Generator().manual_seed(seed)
    w = {n: (torch.randn(s, generator=g) * .04).half() if len(s) == 2 else (1 + torch.randn(s, generator=g) * .1).half()
         for n, s in _SHAPES.items()}
    layer = FrozenSmolLayer(CONFIG, w, mode=mode, capacity=capacity, cache=format)
    oracle = so.OracleLayer(layer._weights, {n: (q.format, q.shape, q.group_size, q.data, q.scales) for n, q in layer._packed.items()},
                            theta=10000.0, capacity=capacity)
    return layer, oracle, g


class HeldLayer:
    """The oracle's layer over a cache that holds `format`."""

    def __init__(self, oracle, format):
        self.o, self.format, self.k, self.v = oracle, format, None, None

    def rows(self, x, only=None):
        """New rows x [b, s, 576]; outputs of all rows, or of the last `only`."""
        o, (b, s, d) = self.o, x.shape
        first = 0 if self.k is None else self.k.shape[2]
        n1 = o.norm(x, 'input_layernorm.weight')
        q, k, v = (o.linear(n1, f'self_attn.{n}_proj.weight').view(b, s, -1, 64).transpose(1, 2) for n in 'qkv')
        cos, sin = o.cos[first:first + s][None, None], o.sin[first:first + s][None, None]
        q, k = o._rotate(q, cos, sin), o._rotate(k, cos, sin)
        self.k = k if self.k is None else torch.cat((self.k, k), 2)
        self.v = v if self.v is None else torch.cat((self.v, v), 2)
        take = s if only is None else only
        att = np.zeros((b, take, 9, 64))
        for i in range(b):
            for h in range(9):
                held = [ko.held(t[i, h // 3].numpy(), self.format) for t in (self.k, self.v)]
                att[i, :, h] = ko.attend(q[i, h, s - take:].numpy(), *held, first + s - take, 0.125)[0]
        att = torch.from_numpy(att).half().reshape(b, take, d)
        value = (x[:, s - take:] + o.linear(att, 'self_attn.o_proj.weight')).half()
        return o._mlp(value, {})


@pytest.mark.parametrize('mode', ['w8a16', 'w4a16', 'fp16'])
@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_prefill_and_decode_match_the_held_values(device, mode, format):
    announce('smollm kv', mode, format)
    layer, oracle, g = make(mode, format, 150)
    held = HeldLayer(oracle, format)
    x = (torch.randn(2, 61, 576, generator=g) * .5).half()
    out, cache = layer.prefill(x.to(device))
    assert type(cache) is SmolQuantizedKVCache and cache.length == 61 and cache.cache.format == format
    assert rel_l2(out, held.rows(x)) <= 1e-2
    for step in range(6):                     # across the end of the first block
        x = (torch.randn(2, 1, 576, generator=g) * .5).half()
        out, cache = layer.decode(x.to(device), cache)
        assert rel_l2(out, held.rows(x)) <= 1e-2, step
    keys, values = cache.read()
    assert cache.length == 67 and tuple(keys.shape) == (2, 3, 150, 64) and not bool(keys[:, :, 67:].any())
    for got, want in ((keys, held.k), (values, held.v)):
        # The decoder bar and the codes' own rounding: int8 steps of a top near 4.5 sigma / 127 are 1.0e-2 sigma rms off,
        # e4m3 values by half a step of 1/8 to 1/16 of them, 2.6e-2 rms; together below 3e-2.
        assert rel_l2(got[:, :, :67], want) <= 3e-2
    assert torch.equal(cache.keys, keys) and torch.equal(cache.values, values)


def test_prefill_past_the_fp16_path(device):
    """A prompt longer than lb_layer_rows takes: the last rows against the oracle."""
    announce('smollm kv long')
    layer, oracle, g = make('w8a16', 'int8', 2600)
    held = HeldLayer(oracle, 'int8')
    x = (torch.randn(1, 2500, 576, generator=g) * .5).half()
    out, cache = layer.prefill(x.to(device))
    assert rel_l2(out[:, -3:], held.rows(x, only=3)) <= 1e-2
    x = (torch.randn(1, 1, 576, generator=g) * .5).half()
    out, cache = layer.decode(x.to(device), cache)
    assert rel_l2(out, held.rows(x)) <= 1e-2


def test_snapshots(device):
    """A snapshot's positions survive later decodes, and it can be gone on from: exactly within the block before the open
    one, from its block's 8-bit values behind that."""
    announce('smollm kv snapshots')
    layer, _, g = make('w8a16', 'int8', 320)
    x = (torch.randn(1, 70, 576, generator=g) * .5).half().to(device)
    rows = (torch.randn(1, 200, 576, generator=g) * .5).half().to(device)
    _, early = layer.prefill(x)
    first = early.read()
    want = layer.decode(rows[:, :1], early)[0]             # (on the shared storage: slot 70)
    assert torch.equal(layer.decode(rows[:, :1], early)[0], want)   # from a copy now
    cache = early
    for i in range(120):                                   # to slot 190: the open block of `early` is closed at 128
        _, cache = layer.decode(rows[:, i:i + 1], cache)
    for got, old in zip(early.read(), first):
        assert torch.equal(got, old)                       # (190 // 64 - 1 = 70 // 64: the rows are there yet)
    assert torch.equal(layer.decode(rows[:, :1], early)[0], want)
    for i in range(120, 130):                              # to slot 200: past the block
        _, cache = layer.decode(rows[:, i:i + 1], cache)
    got = early.read()
    assert torch.equal(got[0][:, :, :64], first[0][:, :, :64]) and not bool(got[0][:, :, 70:].any())
    step = first[0][:, :, :64].abs().amax() / 127
    assert bool((got[0][:, :, 64:70] - first[0][:, :, 64:70]).abs().amax() <= step)   # half a step of a block with a top below twice this one's
    assert rel_l2(layer.decode(rows[:, :1], early)[0], want) <= 1e-2
    assert cache.length == 200 and cache._storage.high == 200


def test_stack_generation_and_graph_decoder(device):
    """generate_greedy over 8-bit caches, and GraphDecoder going on from an 8-bit snapshot with fp16 caches of its values."""
    announce('smollm kv generate')
    cfg = smollm_random.config(theta=10000.0, layers=2)
    weights, embedding, norm, _ = smollm_random.random_weights(3, 2, 0, std=0.06, embed_std=0.5)
    layers = [FrozenSmolLayer(cfg, w, mode='w8a16', capacity=128, cache='fp8') for w in weights]
    stack, io = FrozenSmolStack.from_layers(layers), FrozenSmolIO(cfg, embedding, norm).to(device)
    ids = smollm_random.prompt(1, 60)
    tokens, logits = generate_greedy(stack, io, ids, 8)
    assert len(tokens) == 8 and bool(torch.isfinite(logits).all())
    with torch.no_grad():
        h, caches = stack.prefill(io.embed_tokens(ids.to(device)))
        assert int(io.logits(h[:, -1:])[0, 0].float().argmax()) == tokens[0]
    decoder = GraphDecoder(stack, io)
    decoder.load(caches, tokens[0])
    for i, c in enumerate(caches):
        assert torch.equal(decoder.keys[i], c.keys) and torch.equal(decoder.values[i], c.values)
    assert len(decoder.generate(4)) == 4
    staged = GraphDecoder(stack, io, fused=False)
    staged.load(caches, tokens[0])
    assert torch.equal(staged.keys[1][:, :, :60], caches[1].keys[:, :, :60])


def test_refusals(device):
    layer, _, g = make('w8a16', 'int8', 64)
    other, _, _ = make('w8a16', 'fp16', 64)
    x = (torch.randn(1, 63, 576, generator=g) * .5).half().to(device)
    _, cache = layer.prefill(x)
    _, plain = other.prefill(x)
    with pytest.raises(ValueError, match="own KV cache"):
        layer.decode(x[:, :1], plain)
    with pytest.raises(ValueError, match="own KV cache"):
        other.decode(x[:, :1], cache)
    with pytest.raises(ValueError, match='batch'):
        layer.decode(x[:, :1].expand(2, -1, -1), cache)
    _, cache = layer.decode(x[:, :1], cache)
    with pytest.raises(ValueError, match='full'):
        layer.decode(x[:, :1], cache)
    twin = copy.deepcopy(cache.cache)
    again = pickle.loads(pickle.dumps(cache.cache))
    for c in (twin, again):
        for a, b in zip(c.tensors(), cache.cache.tensors()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and a.data_ptr() != b.data_ptr()
        for a, b in zip(lb.kv_read(c, cache._position), lb.kv_read(cache.cache, cache._position)):
            assert torch.equal(a, b)


@pytest.mark.parametrize('format', ['int8', 'fp8'])
def test_every_step_of_a_generation(device, format):
    """generate_greedy over 8-bit caches: each step's logits against two of the oracle's layers in sequence, fed the tokens
    that were produced, across the end of a block; each token is its step's largest logit.  Then GraphDecoder from the
    prompt's snapshot: every replayed step against the oracle's fp16 decode going on from the values read back."""
    announce('smollm kv every step', format)
    cfg = smollm_random.config(theta=10000.0, layers=2)
    weights, embedding, norm, _ = smollm_random.random_weights(3, 2, 0, std=0.06, embed_std=0.5)
    layers = [FrozenSmolLayer(cfg, w, mode='w8a16', capacity=128, cache=format) for w in weights]
    stack, io = FrozenSmolStack.from_layers(layers), FrozenSmolIO(cfg, embedding, norm).to(device)
    oracles = [so.OracleLayer(layer._weights, {n: (q.format, q.shape, q.group_size, q.data, q.scales) for n, q in layer._packed.items()},
                              theta=10000.0, capacity=128) for layer in layers]
    model = so.OracleModel(oracles, embedding, norm)
    ids, steps = smollm_random.prompt(1, 60), 10            # slots 60 .. 68: a block closes at 64
    tokens, logits = generate_greedy(stack, io, ids, steps)
    held = [HeldLayer(o, format) for o in oracles]

    def through(x):
        for layer in held:
            x = layer.rows(x)
        return model.logits(x[:, -1:])[0, 0]
    want = through(model.embed(ids))
    for step in range(steps):
        assert rel_l2(logits[step], want) <= 1e-2, step
        assert tokens[step] == int(logits[step].float().argmax()), step
        if step < steps - 1:
            want = through(model.embed(torch.tensor([[tokens[step]]])))
    assert len(set(tokens)) > 1

    with torch.no_grad():
        _, caches = stack.prefill(io.embed_tokens(ids.to(device)))
    decoder = GraphDecoder(stack, io)
    decoder.load(caches, tokens[0])
    decoder.capture()
    kv = [tuple(t.cpu()[:, :, :60] for t in c.read()) for c in caches]
    token = tokens[0]
    for step in range(6):
        x = model.embed(torch.tensor([[token]]))
        for i, o in enumerate(oracles):
            x, *kv[i] = o.decode(x, *kv[i], 60 + step)
        token = decoder.generate(1)[0]
        got = decoder.logits.view(-1).clone()
        assert rel_l2(got, model.logits(x)[0, 0]) <= 1e-2, step
        assert token == int(got.float().argmax()), step
