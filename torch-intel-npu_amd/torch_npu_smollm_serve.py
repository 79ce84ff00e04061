"""Greedy decode of many requests at once: a batch of places over one frozen SmolLM stack, each request with its own length,
its own pages of the KV caches, and (optionally) its own low-rank adapter beside every projection.

The reference decodes one sequence at a time (torch_npu_smollm.py:506-544, :628-657) and has no adapters; the weights,
corrections and rounding points of the projections are those of FrozenSmolLayer.  A decode step runs, for each layer,
RMSNorm, one lb_linear per projection with lb_adapters beside it, one lb_paged_attention (rotation, append and attention of
every request), and the MLP; positions, page tables and adapter numbers stay on the device, so a step is captured once and
replayed for whatever requests the batch holds.  Attention is in fp32 with angles in 64 bits (lb_paged_attention), where
FrozenSmolLayer has the reference's fp16 tables and scores: logits differ by those roundings.
"""
import torch
import torch.nn.functional as F

import lowbit_hip
from torch_npu_smollm import _ROWS_ORDER, _SHAPES, HEAD_DIM, HEADS, HIDDEN, KV_HEADS, FrozenSmolStack
from torch_npu_smollm_io import FrozenSmolIO

Q, K, V, O, GATE, UP, DOWN = _ROWS_ORDER


class SmolBatchDecoder:
    """`batch` places for requests of up to `slots` tokens (prompt and answer).

    pages: the pages of `page` slots that the requests share, per layer (default: enough for every place to be full).
    adapters: None, or one dict per layer of projection weight names to lowbit_hip.Adapters (fp16, all of one count): a
    request takes one of their numbers, or none.  graph=False runs every step eagerly.

    A prompt without an adapter runs through the layers as they are, keys turned by their fp16 tables; one with an adapter has its keys turned
    by lb_rotary, as every step has.

    admit() prefills a request into a free place, step() gives every request its next token, release() frees a place.
    tokens holds the last token of each place (int64 on the device, -1 where there is no request), logits the last step's.
    """

    def __init__(self, stack, io, *, batch=16, slots=2048, page=64, pages=None, adapters=None, graph=True):
        if not isinstance(stack, FrozenSmolStack) or not isinstance(io, FrozenSmolIO):
            raise ValueError('Requires a FrozenSmolStack and a FrozenSmolIO')
        if any(layer.cache != 'fp16' for layer in stack.layers):
            raise ValueError('SmolBatchDecoder keeps fp16 pages; it needs layers with cache=\'fp16\'')
        if len({layer._theta for layer in stack.layers}) != 1:
            raise ValueError('Layers must share rope_theta')
        device = io.embedding.device
        if device.type != 'cuda':
            raise ValueError('SmolBatchDecoder needs FrozenSmolIO moved to a ROCm device')
        for name, value in (('batch', batch), ('slots', slots)):
            if type(value) is not int or value < 1:
                raise ValueError(f'{name} must be a positive int')
        longest = -(-slots // page) if type(page) is int and page > 0 else 0
        pages = batch * longest if pages is None else pages
        self.stack, self.io, self.device, self.batch, self.slots, self.page = stack, io, device, batch, slots, page
        self.adapters, self.count = self._check_adapters(stack, adapters)
        self.caches = [lowbit_hip.PagedKVCache.empty(pages, KV_HEADS, page=page, head_dim=HEAD_DIM, device=device) for _ in stack.layers]
        self.rotary = lowbit_hip.Rotary(lowbit_hip.rotary_frequencies(HEAD_DIM, stack.layers[0]._theta, device=device))
        ints = lambda *shape, dtype=torch.int64: torch.full(shape, -1, dtype=dtype, device=device)
        self.table, self.position, self.tokens, self.index = ints(batch, longest, dtype=torch.int32), ints(batch), ints(batch), ints(batch)
        self.logits = torch.zeros((batch, io.vocab_size), dtype=torch.float16, device=device)
        self._free = list(range(pages))
        self._held = [None] * batch       # of each place: (pages, tokens that it may still take)
        rows = torch.zeros((batch, (HEADS + 2 * KV_HEADS) * HEAD_DIM), dtype=torch.float16, device=device)
        self._qkv = rows.split((HIDDEN, KV_HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM), 1)
        q, k, v = (t.unflatten(1, (-1, HEAD_DIM)) for t in self._qkv)
        self._att = torch.zeros((batch, HEADS, HEAD_DIM), dtype=torch.float16, device=device)
        self._attend, scratch = [], None
        for cache in self.caches:         # (in order on one stream, so they share a workspace)
            call = lowbit_hip.PreparedPagedAttention(q, cache, self.table, self.position, self._att, k=k, v=v, rotary=self.rotary,
                                                     scale=0.125, workspace=scratch)
            scratch = call.scratch
            self._attend.append(call)
        self._graph = None
        if graph:
            self._capture()

    @staticmethod
    def _check_adapters(stack, adapters):
        if adapters is None:
            return [{}] * stack.num_layers, 0
        if not isinstance(adapters, (list, tuple)) or len(adapters) != stack.num_layers:
            raise ValueError('adapters must have one dict per layer')
        counts = set()
        for layer in adapters:
            if not isinstance(layer, dict) or not set(layer) <= set(_ROWS_ORDER):
                raise ValueError('adapters must be dicts by SmolLM projection weight names')
            for name, a in layer.items():
                if not isinstance(a, lowbit_hip.Adapters) or (a.N, a.K) != _SHAPES[name] or a.dtype != torch.float16:
                    raise ValueError(f'{name} requires fp16 Adapters of shape {_SHAPES[name]}')
                counts.add(a.count)
        if len(counts) != 1:
            raise ValueError('adapters must all have the same count, and there must be some')
        return [dict(layer) for layer in adapters], counts.pop()

    # ---------------------------------------------------------------- the layers
    def _project(self, layer, state, x, name, adapters, index, out=None):
        y = layer._linear(state, x, name, out=out)
        if name in adapters:
            lowbit_hip.adapters_add(y, x, adapters[name], index)
        return y

    def _mlp(self, layer, state, value, adapters, index):
        n2 = lowbit_hip.rms_rows(value, state['norm2'])
        gate = self._project(layer, state, n2, GATE, adapters, index)
        up = self._project(layer, state, n2, UP, adapters, index)
        hidden = (F.silu(gate.float()).half() * up).half()
        return (value + self._project(layer, state, hidden, DOWN, adapters, index)).half()

    def _step(self):
        """One token of every place: tokens -> logits.  Everything it reads and writes stays where it is."""
        x = self.io.embed_tokens(self.tokens.clamp(min=0)[None])[0]
        for layer, adapters, attend in zip(self.stack.layers, self.adapters, self._attend):
            state = layer._dev(self.device)
            n1 = lowbit_hip.rms_rows(x, state['norm1'])
            for name, out in zip((Q, K, V), self._qkv):
                self._project(layer, state, n1, name, adapters, self.index, out=out)
            attend.run()
            delta = self._project(layer, state, self._att.view(self.batch, HIDDEN), O, adapters, self.index)
            x = self._mlp(layer, state, (x + delta).half(), adapters, self.index)
        self.logits.copy_(self.io.logits(x[:, None])[:, 0])

    def _capture(self):
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.device(self.device), torch.cuda.stream(side), torch.no_grad():
            self._step()                  # (no place holds a request: nothing is appended)
        torch.cuda.current_stream(self.device).wait_stream(side)
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.device(self.device), torch.no_grad(), torch.cuda.graph(self._graph):
            self._step()

    def _prompt(self, x, adapter, table):
        """The prompt's rows x [1, S, 576] through the layers, into the pages; the last row's output."""
        at = torch.zeros(1, dtype=torch.int64, device=self.device)
        if adapter < 0:
            x, caches = self.stack.prefill(x)
            for held, cache in zip(caches, self.caches):
                k, v = (t[:, :, :held.length].transpose(1, 2) for t in (held.keys, held.values))
                lowbit_hip.paged_append(cache, k, v, table, at)
            return x[:, -1:]
        s = x.shape[1]
        x = x[0]
        index = torch.full((s,), adapter, dtype=torch.int64, device=self.device)
        mask = torch.triu(torch.full((s, s), float('-inf'), device=self.device), diagonal=1)
        for layer, adapters, cache in zip(self.stack.layers, self.adapters, self.caches):
            state = layer._dev(self.device)
            n1 = lowbit_hip.rms_rows(x, state['norm1'])
            q, k, v = (self._project(layer, state, n1, name, adapters, index).view(1, s, -1, HEAD_DIM) for name in (Q, K, V))
            lowbit_hip.rotary(q, at, self.rotary, k=k, out=q, out_k=k)
            lowbit_hip.paged_append(cache, k, v, table, at)
            att = layer._attend(*(t.transpose(1, 2) for t in (q, k, v)), mask).transpose(1, 2).reshape(s, HIDDEN)
            delta = self._project(layer, state, att, O, adapters, index)
            x = self._mlp(layer, state, (x + delta).half(), adapters, index)
        return x[None, -1:]

    # ---------------------------------------------------------------- requests
    @torch.no_grad()
    def admit(self, ids, *, steps, adapter=-1):
        """Prefills a request (ids: its prompt's int64 tokens, one row) that may take up to `steps` steps, with an adapter's number
        or -1, into a free place.  Its first token is then tokens[place].  Returns the place.  ValueError where no place
        is free or the pages left are too few (a request gets all of its pages here)."""
        ids = torch.as_tensor(ids)
        if ids.numel() == 0 or ids.dtype != torch.int64 or ids.ndim > 2 or (ids.ndim == 2 and ids.shape[0] != 1):
            raise ValueError('ids must be one row of int64 tokens')
        if int(ids.min()) < 0 or int(ids.max()) >= self.io.vocab_size:
            raise ValueError(f'tokens must be 0 to {self.io.vocab_size - 1}')
        ids = ids.to(self.device).reshape(1, -1)
        s = ids.shape[1]
        if type(steps) is not int or steps < 0 or s < 1 or s + steps > self.slots or s > self.stack.layers[0].capacity:
            raise ValueError(f'a request takes 1 to {self.stack.layers[0].capacity} prompt tokens and {self.slots} slots in all')
        if type(adapter) is not int or not -1 <= adapter < max(self.count, 0):
            raise ValueError(f'adapter must be -1 or one of {self.count}')
        if None not in self._held:
            raise ValueError('no place is free')
        place, need = self._held.index(None), -(-(s + steps) // self.page)
        if need > len(self._free):
            raise ValueError(f'{need} pages are needed and {len(self._free)} are free')
        taken = self._free[:-need - 1:-1]               # (theirs only once the prompt is in them, whatever ends it)
        row = torch.tensor([taken], dtype=torch.int32, device=self.device)
        token = self.io.logits(self._prompt(self.io.embed_tokens(ids), adapter, row))[0, 0].argmax()
        del self._free[-need:]
        self._held[place] = [taken, steps]
        self.table[place, :need] = row[0]
        self.table[place, need:] = -1
        self.position[place], self.index[place], self.tokens[place] = s, adapter, token
        return place

    @torch.no_grad()
    def step(self):
        """The next token of every request (tokens, which is returned, changes in place).  ValueError where a request has taken
        all of its steps: release it first."""
        if all(held is None for held in self._held):
            raise ValueError('no request is held')
        full = [place for place, held in enumerate(self._held) if held is not None and held[1] == 0]
        if full:
            raise ValueError(f'places {full} have taken all of their steps; release them')
        if self._graph is None:
            self._step()
        else:
            self._graph.replay()
        live = self.position >= 0
        self.tokens.copy_(torch.where(live, self.logits.argmax(-1), self.tokens))
        self.position.add_(live)
        for held in self._held:
            if held is not None:
                held[1] -= 1
        return self.tokens

    def release(self, place):
        """Frees a place and its pages."""
        if type(place) is not int or not 0 <= place < self.batch or self._held[place] is None:
            raise ValueError(f'place {place!r} holds no request')
        self._free += self._held[place][0]
        self._held[place] = None
        self.table[place] = -1
        for t in (self.position, self.index, self.tokens):
            t[place] = -1
