"""Serving many requests at once: rotary positions, a KV cache in pages with the attention that reads it, and the
low-rank adapters of many requests beside a shared projection.

  rotary     rows of heads turned by their positions: pairs of dims (i, i + R / 2) or (2 i, 2 i + 1) of the first R dims
             of each head, by the angle position * frequency[i], the cosines and sines times `scale`; dims from R on stay.
             `back` turns the other way (the gradient's direction).
  append     key and value rows of projections into the pages of their sequences, the keys turned first.
  attention  one new token a sequence over the pages that it holds: the token at slot p attends over slots 0 .. p.
  step       the same with its key and value appended first, query and key turned: a decode step.
  adapters   y + scale[a] (x . down[a]^T) . up[a]^T, a the adapter of each row (-1: none), beside a projection's y.

A cache of pages: keys [pages, kv_heads, page, D], values [pages, kv_heads, page / 16, D, 16] (16 slots of a dim side by
side, as the matrix instructions take them).  table [batch, pages of the longest]: slot p of sequence b lies in page
table[b, p // page].

Head layouts: SmolLM-135M (9 query heads, 3 KV heads, D 64), SmolLM-360M (15, 5, 64), Llama-3-8B (32, 8, 128) and generic
ones.  Queries, keys and values are normal, keys with a few large dims, as projections give them.
"""
import math
import sys
from pathlib import Path

import torch

own = False
TYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
S135, S360, L8B = (9, 3, 64), (15, 5, 64), (32, 8, 128)
LAYOUTS = (S135, S360, L8B, (8, 8, 64), (16, 1, 128), (24, 1, 64), (5, 5, 128))
CHUNK = 16                                              # slots that lie side by side for a value dim


def _rotary(dtype, layout, batch, seq, context, part=None, pairs='half', scaled=False, back=False, ragged=True, name=None):
    case = dict(op='rotary', dtype=dtype, heads=layout[0], kv_heads=layout[1], dim=layout[2], batch=batch, seq=seq,
                context=context, part=part or layout[2], pairs=pairs, scaled=scaled, back=back, ragged=ragged)
    return dict(case, name=name) if name else case


def _paged(op, dtype, layout, page, batch, seq, context, ragged=False, pairs='half', scaled=False, name=None):
    """context: slots that the longest sequence holds before the new rows."""
    case = dict(op=op, dtype=dtype, heads=layout[0], kv_heads=layout[1], dim=layout[2], page=page, batch=batch, seq=seq,
                context=context, ragged=ragged, part=layout[2], pairs=pairs, scaled=scaled)
    return dict(case, name=name) if name else case


def _adapters(dtype, N, K, rank, count, rows, kind, name=None):
    """kind: 'tokens' (a row a request, adapters in any order) or 'prompts' (runs of rows)."""
    case = dict(op='adapters', dtype=dtype, N=N, K=K, rank=rank, count=count, rows=rows, kind=kind)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decode step of a few chats with a 135M model: queries and keys of one token each; latency.
        _rotary('fp16', S135, 8, 1, 2047, name='rotary fp16 135m b8 s1'),
        # A long prompt with an 8B model, frequencies stretched for a long context: memory.
        _rotary('bf16', L8B, 1, 8192, 24576, scaled=True, ragged=False, name='rotary bf16 8b b1 s8192'),
        # The gradient of half-turned heads in pairs of neighbours, five ragged prompts.
        _rotary('fp32', (8, 8, 64), 5, 1111, 0, part=32, pairs='neighbours', back=True, name='rotary fp32 back b5 s1111'),
        # The prompts of four requests into their pages.
        _paged('append', 'bf16', L8B, 64, 4, 4100, 0, ragged=True, name='append bf16 8b b4 s4100'),
        # A chunk of a chat's prompt behind what is held, small pages.
        _paged('append', 'fp16', S135, 16, 1, 500, 1003, name='append fp16 135m b1 s500'),
        # The smallest step: one short chat with a 135M model; latency.
        _paged('step', 'fp16', S135, 16, 1, 1, 149, name='step fp16 135m b1 n150'),
        # A step of a full small-model batch, sequences of every length.
        _paged('step', 'fp16', S135, 64, 32, 1, 1983, ragged=True, name='step fp16 135m b32 n1984'),
        # One long document with an 8B model: a single token's work spread over the whole chip.
        _paged('attention', 'bf16', L8B, 128, 1, 1, 130998, name='attention bf16 8b b1 n130999'),
        # A full serving batch of an 8B model, sequences of every length: the cache's bandwidth.
        _paged('attention', 'fp16', L8B, 16, 64, 1, 8191, ragged=True, name='attention fp16 8b b64 n8192'),
        # The o projection of a 135M model, a few requests with an adapter each; latency.
        _adapters('fp16', 576, 576, 8, 4, 5, 'tokens', name='adapters fp16 576x576 r8 m5'),
        # A full serving batch, nearly every request with an adapter of its own.
        _adapters('fp16', 4096, 4096, 16, 64, 64, 'tokens', name='adapters fp16 4096x4096 r16 m64'),
        # Prompts of seven requests beside an 8B model's gate projection.
        _adapters('bf16', 14336, 4096, 32, 7, 4001, 'prompts', name='adapters bf16 14336x4096 r32 m4001'),
    ]


def _size(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, int(low * ((high + 1) / low) ** rng.random()))


def draw(rng):
    op = rng.choice(('rotary', 'append', 'attention', 'attention', 'step', 'step', 'adapters', 'adapters'))
    dtype, layout, ragged = rng.choice(('fp16', 'bf16')), rng.choice(LAYOUTS), rng.random() < 0.6
    pairs, scaled, batch = rng.choice(('half', 'neighbours')), rng.random() < 0.4, _size(rng, 1, 64)
    if op == 'rotary':
        rows = (1 << 24) // (batch * (layout[0] + layout[1]) * layout[2])       # (the largest listed one has 2.5 times that in 16 bits)
        part = rng.choice((layout[2], layout[2] // 2, layout[2] // 4, 40))
        return _rotary(rng.choice(('fp16', 'bf16', 'fp32')), layout, batch, _size(rng, 1, max(1, min(8192, rows))),
                       _size(rng, 1, 131072) - 1, part, pairs, scaled, rng.random() < 0.3, ragged)
    if op == 'adapters':
        N, K = rng.choice(((576, 576), (1536, 576), (576, 1536), (960, 2560), (1000, 264), (4096, 4096), (14336, 4096), (4096, 14336)))
        rank, kind = rng.choice((8, 16, 24, 32, 64, 128)), rng.choice(('tokens', 'tokens', 'prompts'))
        if kind == 'tokens':
            return _adapters(dtype, N, K, rank, _size(rng, 1, 64), _size(rng, 1, 96), kind)
        return _adapters(dtype, N, K, rank, _size(rng, 1, 12), _size(rng, 20, min(8192, (1 << 27) // (N + K) // max(1, rank // 16))), kind)
    page = rng.choice((16, 32, 64, 128))
    row = batch * layout[1] * layout[2]
    if op == 'append':
        return _paged(op, dtype, layout, page, batch, _size(rng, 1, max(1, min(8192, (1 << 24) // row))), _size(rng, 1, 1024) - 1,
                      ragged, pairs, scaled)
    wide = max(1, layout[0] // layout[1] // 4)          # (query heads of a KV head: the listed ones have up to four)
    slots = max(64, min(131072, (1 << (28 if op == 'attention' else 26)) // row // wide))
    return _paged(op, dtype, layout, page, batch, 1, _size(rng, 1, slots) - 1, ragged, pairs, scaled)


# ---------------------------------------------------------------- inputs
def _spans(case):
    """(slots held before the call, new rows) of each sequence."""
    batch, seq, context = case['batch'], case['seq'], case['context']
    if not case['ragged']:
        return [(context, seq)] * batch
    spans = []
    for b in range(batch):
        part = (b * 40503 % 65536) / 65536              # spread over 0 .. 1; the first sequence is the longest
        spans.append((context - int(context * part), max(1, seq - int(seq * ((b * 25173) % 65536) / 65536))))
    return spans


def _pages(case):
    return [-(-(held + rows) // case['page']) for held, rows in _spans(case)]


def _frequencies(case, device):
    """Angles of a step of one position, in 64 bits: 10000 ** (-i / half), the slow ones of a scaled model eight times
    slower, with a ramp between."""
    half = case['part'] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    if case['scaled']:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f


def _scale(case):
    return 1.0 + 0.1 * math.log(8.0) if case['scaled'] else 1.0


def _projected(case, g, device, seq):
    """q, k, v [batch, seq, heads, D] as slices of one projection's rows, a few key dims of each head larger."""
    heads, kv, dim = case['heads'], case['kv_heads'], case['dim']
    rows = torch.randn((case['batch'], seq, (heads + 2 * kv) * dim), generator=g, device=device).to(TYPES[case['dtype']])
    q, k, v = (t.unflatten(-1, (-1, dim)) for t in rows.split((heads * dim, kv * dim, kv * dim), -1))
    loud = 1 + 5 * (torch.rand(kv, dim, generator=g, device=device) < 0.06)
    k.mul_(loud.to(k.dtype))
    v.mul_(0.7)
    return q, k, v


def prepare(case, seed):
    device = torch.device('cuda')
    g = torch.Generator(device=device).manual_seed(int(seed))
    dtype = TYPES[case['dtype']]
    state = dict(case=case)
    if case['op'] == 'adapters':
        state.update(_prepare_adapters(case, g, device, dtype))
    else:
        batch, seq, dim, kv = case['batch'], case['seq'], case['dim'], case['kv_heads']
        spans = _spans(case)
        state['frequencies'] = _frequencies(case, device)
        state['position'] = torch.tensor([h for h, _ in spans], device=device)
        state['q'], state['k'], state['v'] = _projected(case, g, device, seq)
        if case['op'] == 'rotary':
            state['out'] = torch.zeros(state['q'].shape, dtype=dtype, device=device)
            state['out_k'] = torch.zeros(state['k'].shape, dtype=dtype, device=device)
        else:
            held, page = _pages(case), case['page']
            pages = sum(held) + 3
            order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
            state['table'] = table = torch.full((batch, max(held)), -1, dtype=torch.int32, device=device)
            at = 0
            for b, n in enumerate(held):
                table[b, :n] = order[at:at + n]
                at += n
            if case['op'] == 'append':
                state['keys'] = torch.zeros((pages, kv, page, dim), dtype=dtype, device=device)
                state['values'] = torch.zeros((pages, kv, page // CHUNK, dim, CHUNK), dtype=dtype, device=device)
                state['rows'] = torch.tensor([r for _, r in spans], device=device) if case['ragged'] else None
            else:
                loud = 1 + 5 * (torch.rand(kv, 1, dim, generator=g, device=device) < 0.06)
                state['keys'] = torch.randn((pages, kv, page, dim), generator=g, device=device, dtype=dtype).mul_(loud.to(dtype))
                state['values'] = torch.randn((pages, kv, page // CHUNK, dim, CHUNK), generator=g, device=device, dtype=dtype).mul_(0.7)
                state['q'], state['k'], state['v'] = (state[n][:, 0] for n in 'qkv')
                state['out'] = torch.zeros(state['q'].shape, dtype=dtype, device=device)
    if own:
        _prepare_own(case, state)
    return state


def _prepare_adapters(case, g, device, dtype):
    N, K, rank, count, rows = (case[n] for n in ('N', 'K', 'rank', 'count', 'rows'))
    # float32 draws, so that every type's inputs are the same up to its rounding
    rand = lambda *shape: torch.randn(shape, generator=g, device=device)
    state = dict(x=rand(rows, K).to(dtype), y=rand(rows, N).to(dtype), out=torch.zeros((rows, N), dtype=dtype, device=device),
                 down=(rand(count, rank, K) * K ** -0.5).to(dtype), up=(rand(count, N, rank) * rank ** -0.5).to(dtype),
                 scales=torch.rand(count, generator=g, device=device) * 1.5 + 0.5)
    state['runs'] = runs = _runs(case)
    state['index'] = torch.tensor([a for first, last, a in runs for _ in range(first, last)], device=device)
    return state


def _runs(case):
    """(first row, behind the last, adapter) of each request."""
    rows, count = case['rows'], case['count']
    if case['kind'] == 'tokens':                        # every eighth without an adapter, the others in no order
        return [(m, m + 1, -1 if m % 8 == 7 else (m * 40503 + 7) % 65536 % count) for m in range(rows)]
    requests = min(count, rows)
    cut = [rows * i // requests - (i * 2654435761 >> 7) % max(1, rows // (2 * requests)) * (0 < i < requests) for i in range(requests + 1)]
    return [(a, b, -1 if i % 8 == 5 else i) for i, (a, b) in enumerate(zip(cut, cut[1:]))]


def _prepare_own(case, state):
    package = str(Path(__file__).resolve().parents[1] / 'torch-intel-npu_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    import lowbit_hip
    state['lb'] = lowbit_hip
    if case['op'] == 'adapters':
        state['adapters'] = lowbit_hip.Adapters(state['down'], state['up'], scales=state['scales'])
        if case['kind'] == 'tokens':                    # a decode loop keeps its call, over buffers that stay
            state['call'] = lowbit_hip.PreparedAdapters(state['y'], state['x'], state['adapters'], state['index'], state['out'])
        return
    state['rotary'] = lowbit_hip.Rotary(state['frequencies'], pairs=case['pairs'], scale=_scale(case))
    if case['op'] == 'rotary':
        if case['seq'] == 1:
            state['call'] = lowbit_hip.PreparedRotary(state['q'], state['position'], state['rotary'], state['out'], k=state['k'],
                                                      out_k=state['out_k'], back=case['back'])
        return
    state['cache'] = lowbit_hip.PagedKVCache(state['keys'], state['values'])
    if case['op'] != 'append':
        more = dict(k=state['k'], v=state['v'], rotary=state['rotary']) if case['op'] == 'step' else {}
        state['call'] = lowbit_hip.PreparedPagedAttention(state['q'], state['cache'], state['table'], state['position'],
                                                          state['out'], **more)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state['case']
    if not own:
        return _PLAIN[case['op']](state)
    lb, op = state['lb'], case['op']
    if 'call' in state:
        state['call'].run()
    elif op == 'rotary':
        lb.rotary(state['q'], state['position'], state['rotary'], k=state['k'], out=state['out'], out_k=state['out_k'], back=case['back'])
    elif op == 'append':
        lb.paged_append(state['cache'], state['k'], state['v'], state['table'], state['position'], rows=state['rows'],
                        rotary=state['rotary'])
    else:
        lb.adapters_add(state['y'], state['x'], state['adapters'], state['index'], out=state['out'])
    return _outputs(state)


def _outputs(state):
    op = state['case']['op']
    names = {'rotary': ('out', 'out_k'), 'append': ('keys', 'values'), 'step': ('out', 'keys', 'values')}.get(op, ('out',))
    return [state[n] for n in names]


def _turned(state, x, position):
    """x [batch, seq, heads, D] in 32 bits, turned; position [batch, seq].  Angles, their cosines and sines in 64 bits."""
    case = state['case']
    angle = position[..., None].double() * state['frequencies']
    cos, sin = ((f(angle) * _scale(case)).float()[:, :, None] for f in (torch.cos, torch.sin))
    if case.get('back'):
        sin = -sin
    part, x = case['part'], x.float()
    y = x.clone()
    if case['pairs'] == 'half':
        a, b = x[..., :part // 2], x[..., part // 2:part]
        y[..., :part // 2], y[..., part // 2:part] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:part:2], x[..., 1:part:2]
        y[..., 0:part:2], y[..., 1:part:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_rotary(state):
    seq = state['case']['seq']
    position = state['position'][:, None] + torch.arange(seq, device=state['q'].device)
    for out, x in ((state['out'], state['q']), (state['out_k'], state['k'])):
        out.copy_(_turned(state, x, position))
    return _outputs(state)


def _plain_append(state, k=None, v=None, rows=None):
    case, position, table = state['case'], state['position'], state['table']
    k = state['k'] if k is None else k
    v = state['v'] if v is None else v
    batch, seq = k.shape[:2]
    page = case['page']
    slot = position[:, None] + torch.arange(seq, device=k.device)
    at = table.long().gather(1, (slot // page).clamp(max=table.shape[1] - 1))
    live = torch.arange(seq, device=k.device) < (torch.full_like(position, seq) if state.get('rows') is None else state['rows'])[:, None]
    # Rows that are not appended write what their slot holds: sizes stay known without the device.
    at, off = torch.where(live, at, at[:, :1]), torch.where(live, slot % page, slot[:, :1] % page)
    k = _turned(state, k, slot).to(k.dtype)
    pick = torch.where(live, torch.arange(seq, device=k.device), 0)[..., None, None].expand(-1, -1, *k.shape[2:])
    state['keys'][at, :, off] = k.gather(1, pick)
    state['values'][at, :, off // CHUNK, :, off % CHUNK] = v.gather(1, pick)
    return _outputs(state)


def _plain_attention(state, q=None):
    case, position, table = state['case'], state['position'], state['table']
    q = state['q'].float() if q is None else q
    batch, heads, dim = q.shape
    kv, slots = case['kv_heads'], table.shape[1] * case['page']
    pages = table.long().clamp(min=0)
    k = state['keys'][pages].transpose(1, 2).reshape(batch, kv, slots, dim).float()
    v = state['values'][pages].permute(0, 2, 1, 3, 5, 4).reshape(batch, kv, slots, dim).float()
    score = torch.matmul(q.view(batch, kv, heads // kv, dim), k.transpose(2, 3).contiguous()) * dim ** -0.5
    unseen = torch.arange(slots, device=q.device) > position[:, None]
    score.masked_fill_(unseen[:, None, None], float('-inf'))
    score = torch.exp(score - score.amax(-1, keepdim=True))
    state['out'].copy_((torch.matmul(score, v) / score.sum(-1, keepdim=True)).view(batch, heads, dim))
    return _outputs(state)


def _plain_step(state):
    _plain_append(state, state['k'][:, None], state['v'][:, None])
    return _plain_attention(state, _turned(state, state['q'][:, None], state['position'][:, None])[:, 0])


def _plain_adapters(state):
    x, y, down, up, index, out = (state[n] for n in ('x', 'y', 'down', 'up', 'index', 'out'))
    if state['case']['kind'] == 'prompts':              # a request's rows lie together: two products each
        for first, last, a in state['runs']:
            base = y[first:last].float()
            if a >= 0:
                base += state['scales'][a] * (x[first:last].float() @ down[a].float().T @ up[a].float().T)
            out[first:last] = base
        return _outputs(state)
    pick = index.clamp(min=0)
    z = torch.matmul(down[pick].float(), x.float()[..., None])
    delta = torch.matmul(up[pick].float(), z)[..., 0] * state['scales'][pick, None]
    out.copy_(y.float() + torch.where((index >= 0)[:, None], delta, torch.zeros_like(delta)))
    return _outputs(state)


_PLAIN = {'rotary': _plain_rotary, 'append': _plain_append, 'attention': _plain_attention, 'step': _plain_step,
          'adapters': _plain_adapters}


# ---------------------------------------------------------------- work, and the definition in 64 bits
def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'adapters':
        N, K, rank = case['N'], case['K'], case['rank']
        runs = _runs(case)
        with_one = sum(last - first for first, last, a in runs if a >= 0)
        used = len({a for _, _, a in runs if a >= 0})
        return {'bytes': size * (with_one * K + 2 * case['rows'] * N + used * rank * (N + K)) + 8 * case['rows'],
                'flops': 2 * with_one * rank * (N + K)}
    heads, kv, dim, batch, part = case['heads'], case['kv_heads'], case['dim'], case['batch'], case['part']
    spans = _spans(case)
    if case['op'] == 'rotary':
        rows = batch * case['seq'] * (heads + kv)
        return {'bytes': 2 * size * rows * dim, 'flops': 3 * rows * part}
    appended = sum(r for _, r in spans)
    wrote = 4 * size * kv * dim * appended              # k and v read and written
    if case['op'] == 'append':
        return {'bytes': wrote, 'flops': 3 * appended * kv * part}
    slots = sum(h + 1 for h, _ in spans)
    read = 2 * size * heads * dim * batch + 4 * sum(_pages(case))
    if case['op'] == 'attention':
        return {'bytes': read + 2 * size * kv * dim * slots, 'flops': 4 * heads * dim * slots}
    return {'bytes': read + 2 * size * kv * dim * (slots - batch) + wrote, 'flops': 4 * heads * dim * slots + 3 * batch * (heads + kv) * part}


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'adapters':
        x, y, scales = state['x'].double(), state['y'].double(), state['scales'].double()
        out = y.clone()
        for a in set(state['index'].tolist()) - {-1}:
            mine = (state['index'] == a).nonzero()[:, 0]
            down, up = state['down'][a].double(), state['up'][a].double()
            out[mine] += torch.einsum('mk,rk,nr->mn', x[mine], down, up) * scales[a]
        return [out]
    spans, part, kv, dim = _spans(case), case['part'], case['kv_heads'], case['dim']
    turn = torch.polar(torch.full_like(state['frequencies'], _scale(case)), state['frequencies'])

    def turned(x, first):
        """x [rows, heads, D] in 64 bits at positions first ..: pairs as complex numbers, times e^(i position frequency)."""
        x = x.double()
        at = torch.arange(first, first + len(x), device=x.device, dtype=torch.float64)
        by = torch.polar(turn.abs().expand(len(x), -1), at[:, None] * state['frequencies'])[:, None]
        by = by.conj() if case.get('back') else by
        if case['pairs'] == 'half':
            z = torch.complex(x[..., :part // 2], x[..., part // 2:part]) * by
            return torch.cat((z.real, z.imag, x[..., part:]), -1)
        z = torch.complex(x[..., :part].unflatten(-1, (-1, 2))[..., 0], x[..., :part].unflatten(-1, (-1, 2))[..., 1]) * by
        return torch.cat((torch.view_as_real(z).flatten(-2), x[..., part:]), -1)

    if case['op'] == 'rotary':
        return [torch.stack([turned(t[b], spans[b][0]) for b in range(case['batch'])]) for t in (state['q'], state['k'])]
    page = case['page']

    def place(t, b, slot):                              # the page and the place in it
        return int(state['table'][b, slot // page]), slot % page

    if case['op'] == 'append':
        keys, values = state['keys'].double(), state['values'].double()
        for b, (h, r) in enumerate(spans):
            k, v = turned(state['k'][b, :r], h), state['v'][b, :r].double()
            for first in range(h // page * page, h + r, page):
                id = int(state['table'][b, first // page])
                low, high = max(first, h), min(first + page, h + r)
                keys[id, :, low - first:high - first] = k[low - h:high - h].transpose(0, 1)
                by_slot = values[id].transpose(-1, -2).reshape(kv, page, dim).clone()
                by_slot[:, low - first:high - first] = v[low - h:high - h].transpose(0, 1)
                values[id] = by_slot.reshape(kv, page // CHUNK, CHUNK, dim).transpose(-1, -2)
        return [keys, values]
    out = torch.zeros(state['q'].shape, dtype=torch.float64, device=state['q'].device)
    step = case['op'] == 'step'
    keys, values = (state[n].double() if step else None for n in ('keys', 'values'))
    group = case['heads'] // kv
    for b, (h, _) in enumerate(spans):
        ids = state['table'][b, :h // page + 1].long()
        k = state['keys'][ids].double().transpose(0, 1).reshape(kv, -1, dim)[:, :h + 1]
        v = state['values'][ids].double().transpose(-1, -2).reshape(len(ids), kv, page, dim).transpose(0, 1).reshape(kv, -1, dim)[:, :h + 1]
        q = state['q'][b].double()
        if step:
            q = turned(state['q'][b][None], h)[0]
            id, off = int(ids[-1]), h % page
            keys[id, :, off] = turned(state['k'][b][None], h)[0]
            values[id, :, off // CHUNK, :, off % CHUNK] = state['v'][b].double()
            k, v = k.clone(), v.clone()
            k[:, h], v[:, h] = keys[id, :, off].to(state['keys'].dtype).double(), state['v'][b].double()   # as it is held
        s = (q.view(kv, group, dim) @ k.transpose(1, 2)) / dim ** 0.5
        out[b] = (torch.softmax(s, -1) @ v).view(-1, dim)
    return [out, keys, values] if step else [out]
