"""Operators over long histories and the tokens drawn after them, as cases that can be timed and checked.

A case is a dict of plain values; `kind` picks the operator:

  sparse  GPUCache.attend_sparse of one layer: each query attends to the `blocks` tiles of the indexed
          history that score highest for it, to everything appended after the index (`tail` generated
          tokens, a tile each) and to its own chunk;
  index   GPUCache.index: the elementwise bounds of every tile's keys, which those scores read;
  mass    GPUCache.attention_mass of one layer: what every token received of a chunk's softmax;
  evict   GPUCache.evict: per layer and KV head the `keep` tokens of the largest accumulated mass go to
          another cache (`sinks` first and `recent` last tokens stay), read back as values;
  sample  gpu_ops.sample: one token a row from logits and given random numbers.

Histories are a 16-bit text prefix followed by frames of `frame` tokens at 4, 8 or 16 bits (40/40/20),
the last one cut to fit `past`, then `tail` single tokens at 16 bits. Where `own` is false the operators
are computed in their plain form, from the codes, offsets and scales of the packed rows.
"""
import math
import os
import random
import sys

import torch

own = False

DIM, TILE = 64, 64
ROW_BYTES = {4: 40, 8: 72, 16: 128}  # payload and (offset, scale) of one 64-element row
DEVICE = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
    return [
        # one generated token over the default cache's full history: the smallest call, launches and latency
        dict(name='sparse_decode', kind='sparse', heads=5, q_heads=15, nq=1, past=8128, prefix=64, frame=64, tail=24,
             blocks=16, parts=1, precision='bf16', out='bf16'),
        # one generated token over hours of video: scoring two thousand tiles is most of the work
        dict(name='sparse_decode_long', kind='sparse', heads=8, q_heads=32, nq=1, past=131007, prefix=63, frame=64,
             tail=64, blocks=64, parts=1, precision='bf16', out='bf16'),
        # a frame whose queries choose each for itself
        dict(name='sparse_frame', kind='sparse', heads=5, q_heads=15, nq=64, past=32704, prefix=64, frame=64, tail=0,
             blocks=32, parts=1, precision='bf16', out='bf16'),
        # a long question of the small model over 78-token frames (a whole and a partial tile each), fp32 accurate
        dict(name='sparse_question', kind='sparse', heads=3, q_heads=9, nq=513, past=20011, prefix=39, frame=78, tail=9,
             blocks=24, parts=1, precision='fp32', out='fp32'),
        # the index of a whole cache after its frames were ingested
        dict(name='index_layers', kind='index', layers=32, heads=5, past=8128, prefix=64, frame=64),
        # a frame's attention counted over the default cache's full history
        dict(name='mass_frame', kind='mass', heads=5, q_heads=15, nq=64, past=8128, prefix=64, frame=64, tail=0, parts=1,
             precision='bf16'),
        # a generated token's attention counted over hours of video
        dict(name='mass_decode_long', kind='mass', heads=8, q_heads=32, nq=1, past=131007, prefix=63, frame=64, tail=64,
             parts=1, precision='fp32'),
        # a long prompt counts itself and the frames before it
        dict(name='mass_prompt', kind='mass', heads=5, q_heads=15, nq=2048, past=1000, prefix=40, frame=64, tail=0,
             parts=1, precision='bf16'),
        # half of the default cache's history leaves it (a quarter of its layers)
        dict(name='evict_frames', kind='evict', layers=8, heads=5, past=8128, prefix=64, frame=64, keep=4096, sinks=64,
             recent=512),
        # hours of video, 78 tokens a frame, cut to a quarter
        dict(name='evict_long', kind='evict', layers=4, heads=8, past=65531, prefix=41, frame=78, keep=16384, sinks=32,
             recent=2000),
        # the next token of one conversation
        dict(name='sample_one', kind='sample', rows=1, vocab=49280, logits='bf16', temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0),
        # the next tokens of many conversations over a large odd vocabulary, nothing cut by rank
        dict(name='sample_batch', kind='sample', rows=128, vocab=128003, logits='fp32', temperature=1.1, top_k=0, top_p=0.9,
             min_p=0.002),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def history(past):
        return dict(past=past, prefix=rng.randint(1, 128), frame=rng.choice([64, 78, 17, 128, 100]))

    kind = rng.choice(['sparse', 'sparse', 'sparse', 'index', 'mass', 'mass', 'evict', 'evict', 'sample', 'sample'])
    if kind in ('sparse', 'mass'):
        heads, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        nq = rng.choice([1, 1, spread(2, 512)])
        past = spread(200, min(131000, 90_000_000 // (nq * heads * group)))
        case = dict(kind=kind, heads=heads, q_heads=heads * group, nq=nq, **history(past), tail=rng.randint(0, 48),
                    parts=rng.choice([1, 1, 1, min(nq, 4)]), precision=rng.choice(['bf16', 'bf16', 'fp32']))
        if kind == 'sparse':
            case.update(blocks=rng.randint(1, 96), out=rng.choice(['bf16', 'bf16', 'fp32']))
        return case
    if kind == 'index':
        return dict(kind=kind, layers=rng.randint(1, 24), heads=rng.choice([1, 3, 5, 8]), **history(spread(200, 6000)))
    if kind == 'evict':
        past = spread(1500, 30000)
        return dict(kind=kind, layers=rng.randint(1, 6), heads=rng.choice([1, 3, 5, 8]), **history(past),
                    keep=rng.randint(past // 2, past - 1), sinks=rng.randint(0, 64), recent=rng.randint(0, past // 5))
    return dict(kind=kind, rows=spread(1, 96), vocab=spread(1000, 120000), logits=rng.choice(['bf16', 'fp32']),
                temperature=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, 0, spread(2, 500)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]))


def segments_of(case):
    """(lengths, bits) of the history before the tail: the prefix at 16 bits, then frames at mixed widths."""
    past, prefix, frame = case['past'] - case.get('tail', 0), case['prefix'], case['frame']
    past = max(past, 1)
    lengths = [min(prefix, past)]
    while sum(lengths) < past:
        lengths.append(min(frame, past - sum(lengths)))
    bits = [16] + random.Random(case['past']).choices([4, 8, 16], weights=[.4, .4, .2], k=len(lengths) - 1)
    return lengths, bits


def tail_of(case):
    return case['past'] - sum(segments_of(case)[0])


def tiles_of(lengths):
    """(first token, rows) of every tile of up to 64 tokens of these segments."""
    tiles, start = [], 0
    for n in lengths:
        tiles += [(start + i, min(TILE, n - i)) for i in range(0, n, TILE)]
        start += n
    return tiles


def history_bytes(case):
    """Packed bytes of one row of every token of the history, K alone."""
    lengths, bits = segments_of(case)
    return sum(n * ROW_BYTES[b] for n, b in zip(lengths, bits)) + tail_of(case) * ROW_BYTES[16]


def part_bounds(case):
    return [case['nq'] * i // case['parts'] for i in range(case['parts'])] + [case['nq']]


def work(case):
    kind = case['kind']
    if kind == 'sample':  # the logits once; an exponential and a sum for each
        n = case['rows'] * case['vocab']
        return dict(bytes=n * (2 if case['logits'] == 'bf16' else 4), flops=4 * n)
    H, past = case['heads'], case['past']
    if kind in ('sparse', 'mass'):
        Hq, nq, t = case['q_heads'], case['nq'], tail_of(case)
        seen = sum((m + 1) for a, b in zip(part_bounds(case), part_bounds(case)[1:]) for m in range(b - a))
        chunk = (Hq + 2 * H) * nq * DIM * 2
        if kind == 'mass':  # every key once, scores and a sum of each key's column
            return dict(bytes=H * history_bytes(case) + chunk + 4 * H * (past + nq),
                        flops=2 * DIM * Hq * (nq * past + seen))
        lengths, bits = segments_of(case)
        T = len(tiles_of(lengths))
        read = min(1.0, nq * case['blocks'] / T)  # of the indexed history, at most
        keys = min(case['blocks'], T) * (past - t) / T + t
        return dict(bytes=2 * H * (read * (history_bytes(case) - t * 128) + t * 128) + 4 * DIM * H * T + chunk
                    + Hq * nq * DIM * (2 if case['out'] == 'bf16' else 4),
                    flops=4 * DIM * H * nq * T + 4 * DIM * Hq * (nq * keys + seen))
    L = case['layers']
    if kind == 'index':
        return dict(bytes=L * H * (history_bytes(case) + 4 * DIM * len(tiles_of(segments_of(case)[0]))), flops=2 * L * H * past * DIM)
    keep = case['keep']
    # kept rows read and written packed and their values once more, masses read and kept, indices written
    row = 2 * history_bytes(case) / past
    return dict(bytes=L * H * (keep * (2 * row + 2 * 2 * DIM) + 4 * past + 8 * keep), flops=L * H * past)


def quantize(x, bits):
    """Codes, offsets and scales of rows [..., 64] at widths `bits` [tokens] (8 where a row is kept at 16)."""
    x = x.float()
    levels = torch.where(bits == 4, 15, 255)
    offset = x.amin(-1)
    span = x.amax(-1) - offset
    scale = torch.where(span > 0, (span.double() / levels).float(), torch.ones_like(span))
    codes = ((x - offset[..., None]).double() / scale[..., None]).float().round()
    return torch.minimum(codes, levels[:, None].float()).to(torch.uint8), offset, scale


def keys_and_values(gen, layers, heads, tokens, frame):
    """K and V [layers, heads, tokens, 64] bf16: N(0, 1) with four channels of a head eight times as large, keys
    about a centre that a frame's tokens share."""
    def rows():
        x = torch.randn((layers, heads, tokens, DIM), generator=gen, device=DEVICE)
        loud = torch.rand((layers, heads, 1, DIM), generator=gen, device=DEVICE).argsort(-1) < 4
        return x, torch.where(loud, 8.0, 1.0)
    k, gain = rows()
    centre = torch.randn((layers, heads, -(-tokens // frame), DIM), generator=gen, device=DEVICE)
    k += centre.repeat_interleave(frame, 2)[:, :, :tokens]
    v, gain_v = rows()
    return (k * gain).to(torch.bfloat16), (v * gain_v).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case['kind'] == 'sample':
        x = torch.randn((case['rows'], case['vocab']), generator=gen, device=DEVICE) * 2.5
        return dict(case=case, logits=x.to(DTYPES[case['logits']]),
                    u=torch.rand(case['rows'], generator=gen, device=DEVICE))
    layers, heads, past, nq = case.get('layers', 1), case['heads'], case['past'], case.get('nq', 0)
    lengths, bits = segments_of(case)
    k, v = keys_and_values(gen, layers, heads, past + nq, case['frame'])
    state = dict(case=case)
    if nq:
        state['q'] = (torch.randn((1, case['q_heads'], nq, DIM), generator=gen, device=DEVICE) * 0.5).to(torch.bfloat16)
        state['k'], state['v'] = k[0, :, past:][None].contiguous(), v[0, :, past:][None].contiguous()
    if case['kind'] == 'evict':  # masses as they accumulate: a few heavy tokens, many light ones
        state['weights'] = torch.rand((layers, heads, past), generator=gen, device=DEVICE).pow(-0.7).sub(1).contiguous()
    if own:
        state['cache'] = cache_of(state, k, v, lengths, bits)
        if case['kind'] == 'evict':
            state['into'] = empty_cache(case)
        return state
    tail = tail_of(case)
    width = torch.tensor([b for n, b in zip(lengths, bits) for _ in range(n)] + [16] * tail, device=DEVICE)
    state['width'] = width
    for name, x in (('keys', k), ('values', v)):
        x = x[:, :, :past]
        state[name] = (*quantize(x, width), x.contiguous())
    tiles = tiles_of(lengths)
    first = torch.tensor([t[0] for t in tiles], device=DEVICE)
    rows = torch.tensor([t[1] for t in tiles], device=DEVICE)
    # tokens of every tile, a partial one's last token repeated; the tile of every token
    state['tile_tokens'] = first[:, None] + torch.minimum(torch.arange(TILE, device=DEVICE), rows[:, None] - 1)
    state['tile_of'] = torch.repeat_interleave(torch.arange(len(tiles), device=DEVICE), rows)
    if case['kind'] == 'sparse':
        state['bounds'] = plain_bounds(state)
    return state


# ---- the framework's operators ---------------------------------------------------------------------------------

def dkv():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'dynamic-kv-cache_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    from dkv import gpu_cache, gpu_ops
    return gpu_cache, gpu_ops


def empty_cache(case):
    return dkv()[0].GPUCache(None, layers=case.get('layers', 1), heads=case['heads'],
                             max_tokens=case['past'] + case.get('nq', 0), precision=case.get('precision', 'bf16'))


def cache_of(state, k, v, lengths, bits):
    """The cache that a program holds before the call: the history packed, and, where the call reads it, indexed
    before the tail; the chunk appended, as attend() wants it."""
    case, past = state['case'], state['case']['past']
    cache, n = empty_cache(case), sum(lengths)
    cache.append_batch(k[:, :, :n], v[:, :, :n], bits, lengths)
    if case['kind'] == 'sparse':
        cache.index()
    if past > n:
        cache.append_batch(k[:, :, n:past], v[:, :, n:past], [16] * (past - n), [1] * (past - n))
    if 'q' in state:
        cache.select(16)
        cache.append(state['k'], state['v'], 0)
    if 'weights' in state:
        cache.mass().copy_(state['weights'])
    return cache


def run_own(state):
    case, cache = state['case'], state.get('cache')
    if case['kind'] == 'sample':
        return dkv()[1].sample(state['logits'], state['u'], temperature=case['temperature'], top_k=case['top_k'],
                               top_p=case['top_p'], min_p=case['min_p'])
    if case['kind'] == 'index':
        cache.index(first=0)
        low, high = cache.tile_bounds()
        return dict(low=low, high=high)
    if case['kind'] == 'evict':
        kept = cache.evict(case['keep'], sinks=case['sinks'], recent=case['recent'], into=state['into'])
        rows = [kept.materialize(layer) for layer in range(case['layers'])]
        return dict(kept=kept.kept, mass=kept.mass(), k=[r[0] for r in rows], v=[r[1] for r in rows])
    parts = part_bounds(case) if case['parts'] > 1 else None
    if case['kind'] == 'mass':
        return cache.attention_mass(state['q'], state['k'], 0, case['past'], segments=parts)
    return cache.attend_sparse(state['q'], state['k'], state['v'], 0, case['past'], case['blocks'],
                               out_dtype=DTYPES[case['out']], segments=parts)


# ---- the plain forms ---------------------------------------------------------------------------------------------

def unpacked(state, name, precision):
    """The packed rows' values [layers, heads, tokens, 64] in fp32, rounded to bf16 where the cache's precision has
    attention round them."""
    codes, offset, scale, raw = state[name]
    x = torch.where((state['width'] == 16)[:, None], raw.float(), codes.float() * scale[..., None] + offset[..., None])
    return x.to(torch.bfloat16).float() if precision == 'bf16' else x


def plain_bounds(state):
    """(low, high) [tiles, layers, heads, 64] bf16 of the keys of every tile."""
    k = unpacked(state, 'keys', 'bf16')[:, :, state['tile_tokens']]
    return tuple(b.permute(2, 0, 1, 3).to(torch.bfloat16) for b in (k.amin(3), k.amax(3)))


def chunk_mask(case):
    """[nq, nq]: the chunk's tokens that a query sees, itself and those before it in its own part."""
    part = torch.zeros(case['nq'], dtype=torch.long, device=DEVICE)
    part[torch.tensor(part_bounds(case)[1:-1], dtype=torch.long, device=DEVICE)] = 1
    part = part.cumsum(0)
    return (part[:, None] == part[None]).tril()


def plain_scores(state, keys, visible):
    """Scaled scores [heads, group, nq, past + nq] of the queries, -inf where a key is not visible."""
    case, q, H = state['case'], state['q'].float(), state['case']['heads']
    q = q.view(H, -1, DIM)  # a KV head's query heads one after the other
    s = torch.matmul(q, torch.cat((keys, state['k'][0].float()), 1).transpose(1, 2)) * DIM ** -0.5
    s = s.view(H, -1, case['nq'], s.shape[-1])
    return s.masked_fill(~visible, -math.inf)


def plain_softmax(s):
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def plain_choice(state):
    """[heads, nq, indexed tokens]: whether a query attends to a token of the indexed history. A tile's score bounds
    the queries' scores over its keys, summed over the query heads of a KV head: sums in 64 bits, rounded to 32 at
    the end, so that equal scores are equal and the order of the sums does not choose."""
    case = state['case']
    low, high = (b[:, 0].permute(1, 2, 0).double() for b in state['bounds'])  # [heads, 64, tiles]
    q = state['q'][0].double().view(case['heads'], -1, case['nq'], DIM)
    score = (torch.matmul(q.clamp(min=0).sum(1), high) + torch.matmul(q.clamp(max=0).sum(1), low)).float()
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order[..., :case['blocks']], True)
    return chosen[..., state['tile_of']]


def plain_sparse(state):
    case, H, nq = state['case'], state['case']['heads'], state['case']['nq']
    keys, values = (unpacked(state, name, case['precision'])[0] for name in ('keys', 'values'))
    chosen = plain_choice(state)
    rest = torch.ones((H, nq, tail_of(case)), dtype=torch.bool, device=DEVICE)
    visible = torch.cat((chosen, rest, chunk_mask(case).expand(H, nq, nq)), 2)[:, None]
    p = plain_softmax(plain_scores(state, keys, visible))
    out = torch.matmul(p.view(H, -1, p.shape[-1]), torch.cat((values, state['v'][0].float()), 1))
    return out.view(1, case['q_heads'], nq, DIM).transpose(1, 2).to(DTYPES[case['out']])


def plain_mass(state):
    case = state['case']
    keys = unpacked(state, 'keys', case['precision'])[0]
    history = torch.ones((case['nq'], case['past']), dtype=torch.bool, device=DEVICE)
    p = plain_softmax(plain_scores(state, keys, torch.cat((history, chunk_mask(case)), 1)))
    return p.sum((1, 2))


def kept_counts(case):
    """(leading, trailing, {width: tokens kept}): the tokens of the segments that stay whole at either end, and how
    many of each width the segments between them keep, in proportion to what they hold (largest remainders)."""
    lengths, bits = segments_of(case)
    past, a, b = case['past'], 0, len(lengths)
    while a < b and sum(lengths[:a]) < case['sinks']:
        a += 1
    while b > a and sum(lengths[b:]) < case['recent']:
        b -= 1
    held = {}
    for n, w in zip(lengths[a:b], bits[a:b]):
        held[w] = held.get(w, 0) + n
    lead, trail = sum(lengths[:a]), sum(lengths[b:])
    total, left = sum(held.values()), case['keep'] - lead - trail
    keep = {w: left * n // total for w, n in held.items()}
    for w in sorted(held, key=lambda w: (-(left * held[w] % total), -w))[:left - sum(keep.values())]:
        keep[w] += 1
    return lead, past - trail, keep


def plain_evict(state):
    case, w = state['case'], state['weights']
    lead, end, keep = kept_counts(case)
    width, token = state['width'], torch.arange(case['past'], device=DEVICE)
    middle = (token >= lead) & (token < end)

    def heaviest(bits, n):  # the n heaviest of a width, in token order
        own_width = token[middle & (width == bits)]
        order = torch.sort(w[..., own_width], dim=-1, descending=True, stable=True).indices[..., :n]
        return own_width[order.sort(-1).values]
    every = w.shape[:2]
    kept = torch.cat([token[:lead].expand(*every, -1)] + [heaviest(b, n) for b, n in keep.items()]
                     + [token[end:].expand(*every, -1)], -1)
    rows = [unpacked(state, name, 'bf16').to(torch.bfloat16).gather(2, kept[..., None].expand(*kept.shape, DIM))
            for name in ('keys', 'values')]
    return dict(kept=kept.int(), mass=w.gather(2, kept), k=[r[None] for r in rows[0]], v=[r[None] for r in rows[1]])


def plain_sample(state):
    case = state['case']
    x = state['logits'].double()
    x, token = torch.sort(x, dim=-1, descending=True, stable=True)
    if case['top_k']:
        x, token = x[:, :case['top_k']], token[:, :case['top_k']]
    w = torch.exp((x - x[:, :1]) / case['temperature'])
    if case['top_p'] < 1:  # a token stays while those before it hold less than top_p
        total = w.cumsum(-1)
        w = torch.where(total - w < case['top_p'] * total[:, -1:], w, 0)
    w = torch.where(w >= case['min_p'], w, 0)
    by_token = torch.zeros(state['logits'].shape, dtype=torch.float64, device=DEVICE).scatter_(1, token, w)
    total = by_token.cumsum(-1)
    return (total <= state['u'].double()[:, None] * total[:, -1:]).sum(-1)


def run(state):
    if own:
        return run_own(state)
    kind = state['case']['kind']
    if kind == 'sparse':
        return plain_sparse(state)
    if kind == 'index':
        low, high = plain_bounds(state)
        return dict(low=low, high=high)
    if kind == 'mass':
        return plain_mass(state)
    return plain_evict(state) if kind == 'evict' else plain_sample(state)


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------

def exact_rows(state, name, layer, head, precision):
    codes, offset, scale, raw = (x[layer, head] for x in state[name])
    x = codes.float() * scale[:, None] + offset[:, None]
    x[state['width'] == 16] = raw[state['width'] == 16].float()
    return (x.bfloat16() if precision == 'bf16' else x).double()


def exact_attention(state):
    """For each KV head: (probabilities [group, nq, past + nq], values [past + nq, 64])."""
    case = state['case']
    H, nq, past = case['heads'], case['nq'], case['past']
    G, T = case['q_heads'] // H, len(state['tile_tokens'])
    q = state['q'][0].double().view(H, G, nq, DIM)
    bounds, m = part_bounds(case), torch.arange(nq, device=DEVICE)
    seen = torch.zeros((nq, nq), dtype=torch.bool, device=DEVICE)
    for a, b in zip(bounds, bounds[1:]):
        seen[a:b, a:b] = m[None, a:b] <= m[a:b, None]
    for h in range(H):
        k = torch.cat((exact_rows(state, 'keys', 0, h, case['precision']), state['k'][0, h].double()))
        v = torch.cat((exact_rows(state, 'values', 0, h, case['precision']), state['v'][0, h].double()))
        mask = torch.ones((nq, past + nq), dtype=torch.bool, device=DEVICE)
        mask[:, past:] = seen
        if case['kind'] == 'sparse' and case['blocks'] < T:
            low, high = (b[:, 0, h].double() for b in state['bounds'])
            score = torch.zeros((nq, T), dtype=torch.float64, device=DEVICE)
            for g in range(G):
                for at in range(0, nq, 32):
                    x = q[h, g, at:at + 32, None]
                    score[at:at + 32] += torch.maximum(x * low, x * high).sum(-1)
            rank = score.float().neg().argsort(dim=-1, stable=True).argsort(-1)
            mask[:, :len(state['tile_of'])] = (rank < case['blocks'])[:, state['tile_of']]
        s = torch.einsum('gmd,td->gmt', q[h], k) / 8
        yield torch.softmax(s.masked_fill(~mask, -math.inf), -1), v


def exact(case, seed):
    state = prepare(case, seed)
    kind = case['kind']
    if kind == 'sparse':
        out = torch.cat([torch.einsum('gmt,td->gmd', p, v) for p, v in exact_attention(state)])
        return out.transpose(0, 1)[None]
    if kind == 'mass':
        return torch.stack([p.sum((0, 1)) for p, _ in exact_attention(state)])
    if kind == 'index':
        low = torch.empty((len(state['tile_tokens']), case['layers'], case['heads'], DIM), dtype=torch.float64, device=DEVICE)
        high = torch.empty_like(low)
        tiles = tiles_of(segments_of(case)[0])
        for layer in range(case['layers']):
            for h in range(case['heads']):
                k = exact_rows(state, 'keys', layer, h, 'bf16')[state['tile_tokens']]
                low[:, layer, h], high[:, layer, h] = k.amin(1), k.amax(1)
        assert len(tiles) == len(low)
        return dict(low=low, high=high)
    if kind == 'evict':
        lead, end, keep = kept_counts(case)
        kept, mass, ks, vs = [], [], [], []
        for layer in range(case['layers']):
            for h in range(case['heads']):
                w = state['weights'][layer, h].double()
                stay = torch.zeros(case['past'], dtype=torch.bool, device=DEVICE)
                order = list(range(lead))
                for b, n in keep.items():
                    rank = w.masked_fill(state['width'] != b, -1)
                    rank[:lead] = rank[end:] = -1
                    stay = rank.neg().argsort(dim=-1, stable=True)[:n].sort().values
                    order += stay.tolist()
                order += range(end, case['past'])
                at = torch.tensor(order, device=DEVICE)
                kept.append(at), mass.append(w[at])
                ks.append(exact_rows(state, 'keys', layer, h, 'bf16')[at])
                vs.append(exact_rows(state, 'values', layer, h, 'bf16')[at])

        def shaped(x):
            return torch.stack(x).unflatten(0, (case['layers'], case['heads']))
        return dict(kept=shaped(kept), mass=shaped(mass), k=list(shaped(ks)[:, None]), v=list(shaped(vs)[:, None]))
    tokens = []
    for x, u in zip(state['logits'].double(), state['u'].tolist()):
        w = ((x - x.max()) / case['temperature']).exp()
        order = x.neg().argsort(dim=-1, stable=True)[:case['top_k'] or None]
        if case['top_p'] < 1:
            c = w[order].cumsum(0)
            order = order[:int((c < case['top_p'] * c[-1]).sum()) + 1]
        order = order[w[order] >= case['min_p']].sort().values
        c = w[order].cumsum(0)
        tokens.append(order[int((c <= u * c[-1]).sum())])
    return torch.stack(tokens)
