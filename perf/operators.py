"""The KV cache in 8 bits: rows quantised as they are appended, read back, and attended over.

A cache of `capacity` slots holds, for each sequence and KV head, blocks of 64 slots.  A block that is full
is held in 8 bits with one scale for its keys and one for its values (a: the largest magnitude of the block):

  int8  scale = a / 127, code = rint(127 x / a)          fp8  scale = a / 448, code = e4m3(448 x / a)

and the rows of the open block, and of the block before it, in fp16, in a ring of two blocks (slot mod 128).
Keys of a block lie by slot [64, D], values by dim [D, 64], the slots of a value row in the order in which
the matrix instructions take them: slot 16 s + 4 g + r at place 16 g + 4 s + r.

Four kinds of case:

  attention  new query rows (one token, a few drafted ones, a chunk of a prompt, a prompt) over the cache:
             the row at slot p attends over slots 0 .. p, query heads in groups that share a KV head.
  step       one token per sequence: its key and value are appended, then it attends.
  append     rows of projections [batch, seq, kv_heads, D] into the cache.
  read       held slots back as fp16 [batch, kv_heads, slots, D].

Head layouts: SmolLM-135M (9 query heads, 3 KV heads, D 64), SmolLM-360M (15, 5, 64), Llama-3-8B (32, 8, 128)
and generic ones.  Queries, keys and values are normal, keys with a few large dims, as projections give them.
"""
import sys
from pathlib import Path

import torch

own = False
BLOCK = 64
LIMIT = {'int8': 127.0, 'fp8': 448.0}
CODES = {'int8': torch.int8, 'fp8': torch.float8_e4m3fn}
S135, S360, L8B = (9, 3, 64), (15, 5, 64), (32, 8, 128)
LAYOUTS = (S135, S360, L8B, (8, 8, 64), (16, 1, 128), (24, 3, 64), (5, 5, 128))


def _case(op, format, layout, batch, seq, context, ragged=False, name=None):
    """context: slots that the longest sequence holds before the new rows (read: in all)."""
    case = dict(op=op, format=format, heads=layout[0], kv_heads=layout[1], dim=layout[2], batch=batch, seq=seq,
                context=context, ragged=ragged)
    return dict(case, name=name) if name else case


def listed():
    return [
        # The smallest call: one token of one short chat with a 135M model; latency.
        _case('attention', 'int8', S135, 1, 1, 149, name='decode int8 135m b1 n150'),
        # One long document with an 8B model: a single token's work spread over the whole chip.
        _case('attention', 'fp8', L8B, 1, 1, 130998, name='decode fp8 8b b1 n130999'),
        # A full serving batch, sequences of every length: the cache's bandwidth.
        _case('attention', 'int8', L8B, 64, 1, 8191, ragged=True, name='decode int8 8b b64 n8192'),
        # Five drafted tokens a sequence to be verified, not all sequences with all five.
        _case('attention', 'int8', S360, 16, 5, 2001, ragged=True, name='drafts int8 360m b16 s5 n2006'),
        # A decode step of a small batch: append and attention, a block closing here and there.
        _case('step', 'int8', S135, 32, 1, 1983, ragged=True, name='step int8 135m b32 n1984'),
        # Prompts of a padded batch.
        _case('attention', 'int8', S135, 8, 500, 0, ragged=True, name='prefill int8 135m b8 s500'),
        # One long prompt with an 8B model: the matrix units.
        _case('attention', 'fp8', L8B, 1, 8192, 0, name='prefill fp8 8b b1 s8192'),
        # A chunk of a long prompt behind what is already held.
        _case('attention', 'int8', L8B, 1, 509, 32259, name='chunk int8 8b b1 s509 n32768'),
        # What a decode step of a large batch of a small model appends.
        _case('append', 'int8', S135, 64, 1, 1023, ragged=True, name='append int8 135m b64 s1'),
        # What a prefill of four prompts appends.
        _case('append', 'fp8', L8B, 4, 4100, 0, ragged=True, name='append fp8 8b b4 s4100'),
        # A short batch read back: a snapshot taken over by a decoder with fp16 caches.
        _case('read', 'fp8', S135, 8, 0, 777, ragged=True, name='read fp8 135m b8 n777'),
        # A long document read back, to be written out.
        _case('read', 'int8', L8B, 1, 0, 130999, name='read int8 8b b1 n130999'),
    ]


def _size(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, int(low * ((high + 1) / low) ** rng.random()))


def draw(rng):
    op = rng.choice(('attention', 'attention', 'attention', 'step', 'append', 'read'))
    layout, format, ragged = rng.choice(LAYOUTS), rng.choice(('int8', 'fp8')), rng.random() < 0.6
    batch = _size(rng, 1, 64)
    slots = max(64, min(131072, (1 << 29) // (batch * layout[1] * layout[2])))  # what the largest listed cache has
    if op == 'read':
        return _case(op, format, layout, batch, 0, _size(rng, 1, min(slots, (1 << 27) // (batch * layout[1] * layout[2]))), ragged)
    if op == 'step':
        return _case(op, format, layout, batch, 1, _size(rng, 1, slots) - 1, ragged)
    if op == 'append':
        rows = max(1, min(8192, (1 << 24) // (batch * layout[1] * layout[2])))
        return _case(op, format, layout, batch, _size(rng, 1, rows), 64 * (_size(rng, 1, 17) - 1), ragged)
    kind = rng.randrange(3)
    if kind == 0:                                       # a token
        return _case(op, format, layout, batch, 1, _size(rng, 1, slots) - 1, ragged)
    if kind == 1:                                       # drafts
        return _case(op, format, layout, batch, rng.randint(2, 9), _size(rng, 1, min(slots, 16384)), ragged)
    pairs = (1 << 35) // (layout[0] * layout[2])        # a prompt or a chunk: a quarter of the longest prompt's work
    batch = min(batch, 16)
    seq = _size(rng, 10, min(8192, max(10, int((pairs // batch) ** 0.5))))
    context = 0 if rng.random() < 0.5 else _size(rng, 1, max(1, min(32768, pairs // batch // seq)))
    return _case(op, format, layout, batch, seq, context, ragged)


# ---------------------------------------------------------------- inputs
def _spans(case):
    """(slots held before the call, new rows) of each sequence."""
    batch, seq, context = case['batch'], case['seq'], case['context']
    if not case['ragged']:
        return [(context, seq)] * batch
    spans = []
    for b in range(batch):
        part = (b * 40503 % 65536) / 65536              # spread over 0 .. 1; the first sequence is the longest
        held = context - int(context * part)
        if case['op'] == 'append':
            held = held // BLOCK * BLOCK if seq > 1 else held
        spans.append((held, seq if not seq else max(1, seq - int(seq * ((b * 25173) % 65536) / 65536))))
    return spans


def _held(case):
    return [held + rows for held, rows in _spans(case)]


def _capacity(case):
    return (max(1, case['context'] + case['seq']) + BLOCK - 1) // BLOCK * BLOCK


def _place(v):
    """[.., 64 slots, D] as value rows [.., D, 64 places]."""
    *lead, _, dim = v.shape
    at = len(lead)
    return v.reshape(*lead, 4, 4, 4, dim).permute(*range(at), at + 3, at + 1, at, at + 2).reshape(*lead, dim, BLOCK)


def _unplace(v):
    """[.., D, 64 places] as [.., 64 slots, D]."""
    *lead, dim, _ = v.shape
    at = len(lead)
    return v.reshape(*lead, dim, 4, 4, 4).permute(*range(at), at + 2, at + 1, at + 3, at).reshape(*lead, BLOCK, dim)


def _quantise(x, format):
    """(codes, scales) of blocks [.., 64, D], in 32 bits: 127 x is exact there, and one division is rounded once."""
    x = x.float()
    top = x.abs().amax((-1, -2), keepdim=True)
    unit = torch.where(top > 0, x * LIMIT[format] / top, torch.zeros_like(x))
    codes = torch.round(unit).to(torch.int8) if format == 'int8' else unit.to(torch.float8_e4m3fn)
    return codes, (top / LIMIT[format])[..., 0, 0]


def _rows(case, g, device, slots):
    """Keys and values [batch, slots, kv_heads, D]: normal, a few key dims of each head larger than the others."""
    shape = (case['batch'], slots, case['kv_heads'], case['dim'])
    loud = 1 + 5 * (torch.rand(case['kv_heads'], case['dim'], generator=g, device=device) < 0.06)
    k = torch.randn(shape, generator=g, device=device, dtype=torch.float16) * loud.half()
    v = torch.randn(shape, generator=g, device=device, dtype=torch.float16) * 0.7
    return k, v


def prepare(case, seed):
    device = torch.device('cuda')
    g = torch.Generator(device=device).manual_seed(int(seed))
    batch, seq, capacity = case['batch'], case['seq'], _capacity(case)
    blocks, kv, dim = capacity // BLOCK, case['kv_heads'], case['dim']
    spans = _spans(case)
    old = [h if case['op'] in ('append', 'step') else h + r for h, r in spans]     # slots the cache holds before the call
    # The cache, as appends of these rows leave it: blocks of each sequence up to its length, and the ring.
    k, v = (t.transpose(1, 2).reshape(batch, kv, blocks, BLOCK, dim) for t in _rows(case, g, device, capacity))
    length = torch.tensor(old, device=device)
    first = torch.arange(blocks, device=device) * BLOCK
    closed = (first + BLOCK <= length[:, None])[:, None, :, None, None]
    (kc, ks), (vc, vs) = _quantise(k, case['format']), _quantise(v, case['format'])
    blank = torch.zeros((), device=device)
    kc = torch.where(closed, kc.view(torch.int8), blank.to(torch.int8)).view(CODES[case['format']])
    vc = torch.where(closed, vc.view(torch.int8), blank.to(torch.int8))
    vc = _place(vc).contiguous().view(CODES[case['format']])
    ks, vs = (torch.where(closed[..., 0, 0], s, blank) for s in (ks, vs))
    ring = torch.zeros((2, batch, kv, 2, BLOCK, dim), dtype=torch.float16, device=device)
    for back in (1, 0):                                 # the block before the open one, then the open one
        at = length // BLOCK - back
        live = (at >= 0) & (at < blocks)
        block = at.clamp(0, blocks - 1)
        seen = live[:, None] & (block[:, None] * BLOCK + torch.arange(BLOCK, device=device) < length[:, None])
        for i, t in enumerate((k, v)):
            rows = t[torch.arange(batch, device=device), :, block]
            part = torch.where(seen[:, None, :, None], rows, blank.half())
            half = (at % 2)[:, None] == torch.arange(2, device=device)
            ring[i] = torch.where((half & live[:, None])[:, None, :, None, None], part[:, :, None], ring[i])
    state = dict(case=case, key_codes=kc.contiguous(), value_codes=vc, key_scales=ks.contiguous(),
                 value_scales=vs.contiguous(), key_tail=ring[0].contiguous(), value_tail=_place(ring[1]).contiguous())
    del k, v, ring, kc, vc
    if case['op'] == 'read':
        state['length'] = length
        state['out'] = [torch.zeros((batch, kv, case['context'], dim), dtype=torch.float16, device=device) for _ in range(2)]
    else:
        state['position'] = torch.tensor([h for h, _ in spans], device=device)
        state['rows'] = torch.tensor([r for _, r in spans], device=device) if case['ragged'] and seq > 1 else None
    if case['op'] in ('append', 'step'):
        state['k'], state['v'] = _rows(case, g, device, seq)
    if case['op'] in ('attention', 'step'):
        state['q'] = torch.randn((batch, seq, case['heads'], dim), generator=g, device=device, dtype=torch.float16)
        state['out'] = torch.zeros_like(state['q'])
    if own:
        package = str(Path(__file__).resolve().parents[1] / 'torch-intel-npu_amd')
        if package not in sys.path:
            sys.path.insert(0, package)
        import lowbit_hip
        state['lb'] = lowbit_hip
        state['cache'] = cache = lowbit_hip.QuantizedKVCache(
            state['key_codes'], state['value_codes'], state['key_scales'], state['value_scales'], state['key_tail'],
            state['value_tail'])
        if seq == 1:                                    # a decode loop keeps its call, over buffers that stay
            if case['op'] == 'append':
                state['call'] = lowbit_hip.PreparedKVAppend(cache, state['k'], state['v'], state['position'])
            else:
                state['call'] = lowbit_hip.PreparedKVAttention(state['q'], cache, state['position'], state['out'],
                                                               k=state.get('k'), v=state.get('v'))
    return state


# ---------------------------------------------------------------- one pass
def _outputs(state, *first):
    return [*first, *(state[n] for n in ('key_codes', 'value_codes', 'key_scales', 'value_scales', 'key_tail', 'value_tail'))]


def run(state):
    case = state['case']
    if not own:
        return _PLAIN[case['op']](state)
    lb, cache = state['lb'], state['cache']
    if case['op'] == 'read':
        lb.kv_read(cache, state['length'], count=case['context'], keys=state['out'][0], values=state['out'][1])
        return state['out']
    if 'call' in state:
        state['call'].run()
    elif case['op'] == 'append':
        lb.kv_append(cache, state['k'], state['v'], state['position'], rows=state['rows'])
    else:
        lb.kv_attention(state['q'], cache, state['position'], rows=state['rows'], out=state['out'])
    if case['op'] == 'attention':
        return state['out']
    return _outputs(state, *([state['out']] if case['op'] == 'step' else []))


def _values(state, length):
    """Keys and values [batch, kv_heads, capacity, D] in 32 bits as the cache holds them at `length` slots."""
    kc, ks = state['key_codes'].float(), state['key_scales']
    batch, kv, blocks, _, dim = kc.shape
    k = kc * ks[..., None, None]
    v = _unplace(state['value_codes'].float()) * state['value_scales'][..., None, None]
    # The open block comes out of the ring.
    at = (length // BLOCK).clamp(max=blocks - 1)
    every = torch.arange(batch, device=kc.device)
    open_ = (torch.arange(blocks, device=kc.device) == (length // BLOCK)[:, None])[:, None, :, None, None]
    k = torch.where(open_, state['key_tail'][every, :, at % 2].float()[:, :, None], k)
    v = torch.where(open_, _unplace(state['value_tail'][every, :, at % 2].float())[:, :, None], v)
    return k.view(batch, kv, blocks * BLOCK, dim), v.view(batch, kv, blocks * BLOCK, dim)


def _plain_read(state):
    length, count = state['length'], state['case']['context']
    live = (torch.arange(count, device=length.device) < length[:, None])[:, None, :, None]
    for out, t in zip(state['out'], _values(state, length)):
        out.copy_(torch.where(live, t[:, :, :count].half(), out))
    return state['out']


def _plain_attention(state):
    q, position, out = state['q'], state['position'], state['out']
    batch, seq, heads, dim = q.shape
    kv = state['case']['kv_heads']
    rows = torch.full_like(position, seq) if state['rows'] is None else state['rows']
    k, v = _values(state, position + rows)
    slots = k.shape[2]
    at = position[:, None] + torch.arange(seq, device=q.device)
    q = q.view(batch, seq, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, dim).float()
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(batch, kv, -1, seq, slots) * dim ** -0.5
    unseen = torch.arange(slots, device=q.device) > at[..., None]
    score.masked_fill_(unseen[:, None, None], float('-inf'))
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1, keepdim=True)
    # What lies past the last slot is not part of the cache.
    v = torch.where((torch.arange(slots, device=q.device) < (position + rows)[:, None])[:, None, :, None], v, torch.zeros_like(v))
    y = torch.matmul(score.view(batch, kv, -1, slots), v).view(batch, kv, -1, seq, dim) / total
    y = y.permute(0, 3, 1, 2, 4).reshape(batch, seq, heads, dim)
    live = (torch.arange(seq, device=q.device) < rows[:, None])[:, :, None, None]
    out.copy_(torch.where(live, y.half(), out))
    return out


def _plain_append(state):
    case, position = state['case'], state['position']
    batch, seq, kv, dim = state['k'].shape
    device, capacity = position.device, _capacity(case)
    blocks = capacity // BLOCK
    rows = torch.full_like(position, seq) if state['rows'] is None else state['rows']
    end, every = position + rows, torch.arange(batch, device=position.device)
    slot = torch.arange(capacity, device=device)
    row = slot - position[:, None]                      # the new row at each slot, if there is one
    new = ((row >= 0) & (row < rows[:, None])).view(batch, 1, blocks, BLOCK, 1)
    held = (position // BLOCK)[:, None] == torch.arange(blocks, device=device)   # the block that was open
    closing = ((torch.arange(blocks, device=device) >= (position // BLOCK)[:, None])
               & (torch.arange(blocks, device=device) < (end // BLOCK)[:, None]))[:, None]
    ring = ((torch.arange(blocks, device=device) - (end // BLOCK)[:, None] + 1).unsqueeze(1) // 2 == 0)  # end's block and the one before
    for side in ('key', 'value'):
        tail = state[side + '_tail'] if side == 'key' else _unplace(state['value_tail'])
        fresh = state[side[0]].transpose(1, 2)[every[:, None, None], torch.arange(kv, device=device)[:, None],
                                               row.clamp(0, seq - 1)[:, None]].view(batch, kv, blocks, BLOCK, dim)
        was = tail[every, :, (position // BLOCK) % 2][:, :, None]
        block = torch.where(new, fresh, torch.where(held[:, None, :, None, None], was, torch.zeros_like(was)))
        codes, scales = _quantise(block, case['format'])
        codes = codes if side == 'key' else _place(codes.view(torch.int8))
        name = side + '_codes'
        state[name].view(torch.int8).copy_(torch.where(closing[..., None, None], codes.view(torch.int8), state[name].view(torch.int8)))
        name = side + '_scales'
        state[name].copy_(torch.where(closing, scales, state[name]))
        for half in (0, 1):                             # at most one of the two blocks lies in each half
            mine = (ring & (torch.arange(blocks, device=device) % 2 == half)).expand(batch, kv, blocks)[..., None, None]
            written = (mine & new).any(2)
            rows_ = torch.where(mine & new, fresh, torch.zeros_like(fresh)).sum(2, dtype=torch.float32).half()
            tail[:, :, half] = torch.where(written, rows_, tail[:, :, half])
        if side == 'value':
            state['value_tail'].copy_(_place(tail))
    return _outputs(state)


def _plain_step(state):
    _plain_append(state)
    return _outputs(state, _plain_attention(state))


_PLAIN = {'read': _plain_read, 'attention': _plain_attention, 'append': _plain_append, 'step': _plain_step}


# ---------------------------------------------------------------- work, and the definition in 64 bits
def work(case):
    kv, dim, heads = case['kv_heads'], case['dim'], case['heads']
    spans = _spans(case)

    def held(n):                                        # bytes of n slots of a head's keys and values: codes and scales, fp16
        return n // BLOCK * (2 * BLOCK * dim + 8) + n % BLOCK * 4 * dim

    if case['op'] == 'read':
        n = [h for h, _ in spans]
        return {'bytes': kv * sum(held(h) + 4 * dim * h for h in n), 'flops': 2 * kv * dim * sum(n)}
    wrote = flops = 0
    if case['op'] in ('append', 'step'):
        for h, r in spans:
            end = h + r
            closed = end // BLOCK - h // BLOCK
            fp16 = min(r, end - max(0, (end // BLOCK - 1) * BLOCK))
            wrote += kv * (4 * dim * r + 4 * dim * fp16 + closed * (2 * BLOCK * dim + 8) + (4 * dim * (h % BLOCK) if closed else 0))
            flops += kv * closed * 4 * BLOCK * dim
    if case['op'] == 'append':
        return {'bytes': wrote, 'flops': flops}
    pairs = sum(r * h + r * (r + 1) // 2 for h, r in spans)
    return {'bytes': wrote + sum(kv * held(h + r) + 4 * heads * dim * r for h, r in spans), 'flops': flops + 4 * heads * dim * pairs}


def exact(case, seed):
    state = prepare(case, seed)
    kv, dim, seq = case['kv_heads'], case['dim'], case['seq']
    group = case['heads'] // kv
    spans, op = _spans(case), case['op']
    names = ('key_codes', 'value_codes', 'key_scales', 'value_scales')
    pos = torch.tensor([16 * (s % 16 // 4) + 4 * (s // 16) + s % 4 for s in range(BLOCK)], device=state['key_codes'].device)
    made = {}
    if op in ('append', 'step'):                        # the rows in place, then each new full block's scales
        scales = [state[n].double().clone() for n in names[2:]]
        for b, (h, r) in enumerate(spans):
            for side in (0, 1):
                tail = state['key_tail'][b] if side == 0 else state['value_tail'][b][..., pos].transpose(-1, -2)
                start = h // BLOCK
                x = torch.cat((tail[:, start % 2, :h % BLOCK], state['kv'[side]][b, :r].transpose(0, 1)), 1).double()
                n = (h + r) // BLOCK - start
                full = x[:, :n * BLOCK].reshape(kv, n, BLOCK * dim)
                scales[side][b, :, start:start + n] = full.abs().amax(-1) / LIMIT[case['format']]
                made[b, side] = (start, x, scales[side][b])
    if op == 'append':
        return [None, None, *scales, None, None]

    def values(b, side, n):
        """Slots 0 .. n - 1 of sequence b [kv, n, D]."""
        codes = state[names[side]][b].double()
        tail = (state['key_tail'] if side == 0 else state['value_tail'])[b].double()
        if side:
            codes, tail = codes[..., pos].transpose(-1, -2), tail[..., pos].transpose(-1, -2)
        x = codes * state[names[2 + side]][b].double()[..., None, None]
        whole = n // BLOCK
        x = torch.cat((x[:, :whole].reshape(kv, -1, dim), tail[:, whole % 2, :n % BLOCK]), 1)
        if (b, side) in made:
            start, rows, scale = made[b, side]
            full = (n // BLOCK - start) * BLOCK
            block = rows[:, :full].reshape(kv, -1, BLOCK, dim)
            top = block.abs().amax((-1, -2), keepdim=True)
            unit = torch.where(top > 0, block * LIMIT[case['format']] / top, torch.zeros_like(block))
            if case['format'] == 'int8':
                unit = torch.round(unit)
            else:                                       # e4m3: 3 bits behind the first, steps of 2^-9 at the least
                step = torch.exp2(torch.clamp(torch.frexp(unit).exponent.double() - 4, min=-9))
                unit = torch.round(unit / step) * step
            block = unit * scale[:, start:start + full // BLOCK, None, None]
            x = torch.cat((x[:, :start * BLOCK], block.reshape(kv, -1, dim), rows[:, full:]), 1)
        return x

    if op == 'read':
        outs = [torch.zeros(o.shape, dtype=torch.float64, device=o.device) for o in state['out']]
        for b, (h, _) in enumerate(spans):
            for side in (0, 1):
                outs[side][b, :, :h] = values(b, side, h)
        return outs
    out = torch.zeros(state['q'].shape, dtype=torch.float64, device=state['q'].device)
    for b, (h, r) in enumerate(spans):
        k, v = values(b, 0, h + r), values(b, 1, h + r)
        for first in range(0, r, 1024):                 # rows at a time, for the scores' memory
            last = min(r, first + 1024)
            seen = torch.arange(h + r, device=out.device) <= torch.arange(h + first, h + last, device=out.device)[:, None]
            for head in range(case['heads']):
                s = (state['q'][b, first:last, head].double() @ k[head // group].T) / dim ** 0.5
                s = torch.where(seen, s, torch.full_like(s, float('-inf')))
                out[b, first:last, head] = torch.softmax(s, -1) @ v[head // group]
    if op == 'attention':
        return out
    return [out, None, None, *scales, None, None]
