"""The paged cache's operators (``vesta.paged.PagedCache``), as cases that can be timed and compared.

A case is one call that a serving program makes between two layers, or between two steps, on sequences
of different lengths whose key and value rows lie in pages of one pool:

* ``kind='append'``: the new tokens' key and value rows go into the pages (rounded to the pool's type).
  Results: the pool.
* ``kind='attend'``: attention of each sequence's new tokens (``counts``) over all its ``lengths``
  positions, the new ones causally. Results: the output rows; with ``weights`` also the attention weight
  that each position has received so far.
* ``kind='evict'``: each sequence keeps its ``recent`` last positions and those that received the most
  weight, ``keep`` in all, for each layer and head, in other pages. Results: the pool, the new lengths,
  the kept positions and their weights.

``context`` is the longest context before the new tokens and ``tokens`` the most new tokens; the
sequences' own numbers lie between ``ragged`` (a part of 1) times these and these, the first sequence
having the most. Pages lie in the pool in random order, as after some time of serving.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False      # False: the plain forms; True: the framework's operators

_DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def _case(name, kind, seqs, context, tokens, heads, group, width, dtype, page, ragged=1.0, query='', weights=False,
          layers=1, keep=0, recent=0):
    """``dtype``: the pool's type; ``query``: the new rows' or the queries' own (default: the pool's)."""
    return dict(name=name, kind=kind, seqs=seqs, context=context, tokens=tokens, heads=heads, group=group, width=width,
                dtype=dtype, query=query or dtype, page=page, ragged=ragged, weights=weights, layers=layers, keep=keep,
                recent=recent)


def listed():
    return [
        # the benchmark's 8 rows of GPT-2 small, a decode step's new rows: the smallest call, latency alone
        _case('append_8x1', 'append', 8, 391, 1, 12, 1, 64, 'f16', 64, query='f32'),
        # prompts for a server's batch, ragged, into pages of 16
        _case('append_32x700', 'append', 32, 300, 700, 8, 1, 128, 'bf16', 16, ragged=0.3),
        # one user of GPT-2 small, one token: latency alone
        _case('decode_1_f32', 'attend', 1, 700, 1, 12, 1, 64, 'f16', 64, query='f32'),
        # a server's batch of ragged conversations, four query heads to a key head
        _case('decode_64_gqa', 'attend', 64, 4000, 1, 8, 4, 128, 'bf16', 16, ragged=0.1),
        # two very long documents asked one question each: few rows, a long axis
        _case('decode_2_long', 'attend', 2, 100003, 1, 8, 4, 128, 'f16', 64, ragged=0.9),
        # GPT-2 small's prompts of the benchmark, the activations in 32 bits as the layered engine has them
        _case('chunk_8x128_f32', 'attend', 8, 0, 128, 12, 1, 64, 'f16', 64, query='f32'),
        # chunked prefill of the largest model's 25 heads: ragged chunks after ragged contexts
        _case('chunk_6x512', 'attend', 6, 450, 512, 25, 1, 64, 'f16', 16, ragged=0.05),
        # a long document's next chunk: the most work
        _case('chunk_1x4096_long', 'attend', 1, 27001, 4096, 8, 4, 128, 'bf16', 64),
        # decode steps of GPT-2 medium that keep account of the weight each position receives
        _case('weigh_32x1', 'attend', 32, 1000, 1, 16, 1, 64, 'f16', 32, ragged=0.2, weights=True),
        # prompts that do
        _case('weigh_4x1999', 'attend', 4, 0, 1999, 8, 4, 128, 'bf16', 64, ragged=0.5, weights=True),
        # GPT-2 small's full caches halved, in all layers
        _case('evict_8x1024', 'evict', 8, 1024, 0, 12, 1, 64, 'f16', 32, ragged=0.4, layers=12, keep=512, recent=64),
        # long conversations cut to a quarter
        _case('evict_3x30000', 'evict', 3, 30011, 0, 8, 1, 128, 'bf16', 64, ragged=0.6, layers=2, keep=8001, recent=500),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(('append', 'attend', 'attend', 'attend', 'evict'))
    width = rng.choice((64, 128))
    heads, group = rng.choice(((12, 1), (16, 1), (25, 1), (8, 4), (4, 7), (1, 16), (2, 3)))
    dtype = rng.choice(('f16', 'bf16'))
    query = rng.choice(('f32', 'f16')) if dtype == 'f16' and kind != 'evict' else dtype
    page = rng.choice((8, 16, 32, 64, 128))
    ragged = rng.choice((0.05, 0.5, 1.0))
    shape = dict(heads=heads, group=group, width=width, dtype=dtype, query=query, page=page, ragged=ragged)
    row = heads * width
    if kind == 'append':
        tokens = _spread(rng, 1, 4000)
        seqs = _spread(rng, 1, max(1, min(64, 24 * 1024 * 1024 // (row * tokens))))
        return _case('', kind, seqs, _spread(rng, 1, 1000), tokens, **shape)
    if kind == 'evict':
        context = _spread(rng, 40, 30000)
        layers = rng.choice((1, 2, 5))
        seqs = _spread(rng, 1, max(1, min(16, 160 * 1024 * 1024 // (row * context * layers))))
        keep = max(1, int(context * rng.uniform(0.1, 0.9)))
        return _case('', kind, seqs, context, 0, layers=layers, keep=keep, recent=rng.randrange(0, min(keep, 600) + 1),
                     **shape)
    weights = rng.random() < 0.3
    if rng.random() < 0.5:      # a decode step
        context = _spread(rng, 1, 100000)
        seqs = _spread(rng, 1, max(1, min(128, 200 * 1024 * 1024 // (row * context))))
        return _case('', kind, seqs, context, 1, weights=weights, **shape)
    tokens = _spread(rng, 2, 4096)
    context = 0 if rng.random() < 0.4 else _spread(rng, 1, 24000)
    pairs = tokens * (context + tokens) * group * row
    seqs = _spread(rng, 1, max(1, min(32, int(4e11) // (2 * pairs), 4 * 1024 * 1024 // (tokens * group * heads))))
    return _case('', kind, seqs, context, tokens, weights=weights, **shape)


def _numbers(case):
    """Each sequence's new tokens and its whole length: the case's own, whatever the seed."""
    rng = random.Random(1000003 * case['seqs'] + 1009 * case['context'] + case['tokens'])
    least = case['ragged']

    def some(most, low):
        return [most] + [max(low, int(round(most * rng.uniform(least, 1.0)))) for _ in range(case['seqs'] - 1)]

    counts = some(case['tokens'], 1) if case['tokens'] else [0] * case['seqs']
    return counts, [c + n for c, n in zip(counts, some(case['context'], 0))]


def _inputs(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed) * 2 + 1)
    counts, lengths = _numbers(case)
    page, heads, width, layers = case['page'], case['heads'], case['width'], case['layers']
    B, M = case['seqs'], sum(counts)
    # a server's tables have room beyond the present lengths: here two pages
    wide = [-(-n // page) + 2 for n in lengths]
    to_wide = -(-case['keep'] // page)
    pages = sum(wide) + B * to_wide + 3
    order = torch.randperm(pages, generator=gen, device='cuda').int()
    table = torch.full((B, max(wide)), -1, dtype=torch.int32, device='cuda')
    at = 0
    for b, n in enumerate(wide):
        table[b, :n] = order[at:at + n]
        at += n
    to = order[at:at + B * to_wide].reshape(B, to_wide).contiguous()

    def normal(shape, dtype, scale=1.0):
        t = torch.empty(shape, dtype=_DTYPES[dtype], device='cuda')
        t.normal_(0.0, scale, generator=gen)
        return t

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device='cuda')

    s = dict(case=case, counts=counts, lens=lengths, table=table, to=to, lengths=ints(lengths),
             starts=ints([sum(counts[:b]) for b in range(B + 1)]))
    pool = (layers, pages, page, heads, width)
    s['keys'], s['vals'] = normal(pool, case['dtype']), normal(pool, case['dtype'])
    if case['kind'] == 'append':
        s['k'], s['v'] = (normal((M, heads, width), case['query'], 1.5) for _ in range(2))
    if case['kind'] == 'attend':
        # scores of a spread between a flat and a peaked softmax
        s['q'] = normal((M, heads * case['group'], width), case['query'], 1.8)
    S = table.shape[1] * page
    if case['weights'] or case['kind'] == 'evict':
        # sums of softmax weights: spread over orders of magnitude, some positions never looked at
        w = torch.empty((layers, B, heads, S), device='cuda').normal_(0.0, 2.0, generator=gen).exp_()
        w.masked_fill_(torch.rand((layers, B, heads, S), generator=gen, device='cuda') < 0.03, 0.0)
        s['weight'] = w if case['kind'] == 'evict' else w[0]
        s['weight_out'] = torch.zeros(w.shape[:-1] + (to_wide * page,), device='cuda') if case['kind'] == 'evict' \
            else torch.zeros_like(w[0])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / 'vesta-gpu_amd'))
        from vesta.paged import PagedCache
        layers, pages, page, heads, width = s['keys'].shape
        cache = PagedCache(pages, heads, width, layers=layers, page=page, dtype=case['dtype'])
        cache.keys.copy_(s['keys'])
        cache.vals.copy_(s['vals'])
        s['cache'], s['keys'], s['vals'] = cache, cache.keys, cache.vals
    return s


def _slots(s, table, b, n):
    """The pool rows (page, slot) of sequence b's positions 0 .. n - 1."""
    page = s['case']['page']
    p = torch.arange(n, device='cuda')
    return table[b].long()[p // page], p % page


def _plain_append(s):
    for b, (c, n) in enumerate(zip(s['counts'], s['lens'])):
        i0 = sum(s['counts'][:b])
        pages, slots = (t[n - c:] for t in _slots(s, s['table'], b, n))
        for pool, new in ((s['keys'], s['k']), (s['vals'], s['v'])):
            pool[0, pages, slots] = new[i0:i0 + c].to(pool.dtype)
    return dict(keys=s['keys'], vals=s['vals'])


def _attend(s, b, i0, keys, vals, dtype):
    """Sequence b's attention in ``dtype``: yields (first key head, heads, output [heads, group, count, width],
    weights received [heads, length])."""
    case = s['case']
    c, n, G, E = s['counts'][b], s['lens'][b], case['group'], case['width']
    pages, slots = _slots(s, s['table'], b, n)
    hidden = torch.arange(n, device='cuda')[None, :] > torch.arange(n - c, n, device='cuda')[:, None]
    some = max(1, min(case['heads'], (1 << 28) // (G * c * n)))
    for h in range(0, case['heads'], some):
        hs = min(some, case['heads'] - h)
        k, v = (t[0, :, :, h:h + hs][pages, slots].to(dtype).transpose(0, 1) for t in (keys, vals))
        q = s['q'][i0:i0 + c, h * G:(h + hs) * G].to(dtype).reshape(c, hs, G, E).permute(1, 2, 0, 3)
        z = (q.reshape(hs, G * c, E) @ k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(E))
        z = z.view(hs, G, c, n).masked_fill(hidden, -math.inf)
        e = torch.exp(z - z.amax(-1, keepdim=True))
        del z
        w = e / e.sum(-1, keepdim=True)
        del e
        o = (w.view(hs, G * c, n) @ v.contiguous()).view(hs, G, c, E)
        yield h, hs, o, (w.sum((1, 2)) if case['weights'] else None)


def _plain_attend(s, dtype=torch.float32, rounded=True):
    case = s['case']
    out = torch.empty_like(s['q'], dtype=s['q'].dtype if rounded else dtype)
    got = s['weight'].to(dtype) if case['weights'] else None
    for b, (c, n) in enumerate(zip(s['counts'], s['lens'])):
        i0 = sum(s['counts'][:b])
        for h, hs, o, w in _attend(s, b, i0, s['keys'], s['vals'], dtype):
            out[i0:i0 + c, h * case['group']:(h + hs) * case['group']] = \
                o.permute(2, 0, 1, 3).reshape(c, hs * case['group'], -1).to(out.dtype)
            if w is not None:
                got[b, h:h + hs, n - c:n] = 0
                got[b, h:h + hs, :n] += w
                got[b, h:h + hs, n:] = 0
    return dict(out=out, weight=got) if case['weights'] else dict(out=out)


def _plain_evict(s):
    case = s['case']
    L, H, keep, page = case['layers'], case['heads'], case['keep'], case['page']
    kept_all = torch.full((L, case['seqs'], H, keep), -1, dtype=torch.int32, device='cuda')
    weight = torch.zeros_like(s['weight_out'])
    for b, n in enumerate(s['lens']):
        m, last = min(keep, n), min(case['recent'], min(keep, n))
        w = s['weight'][:, b, :, :n].clone()
        w[..., n - last:] = math.inf
        kept = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :m].sort(-1).values
        kept_all[:, b, :, :m] = kept.int()
        weight[:, b, :, :m] = torch.gather(s['weight'][:, b], -1, kept)
        src = s['table'][b].long()[kept // page], kept % page                       # [L, H, m]
        dst = tuple(t.expand(L, H, m) for t in _slots(s, s['to'], b, m))
        at = (torch.arange(L, device='cuda')[:, None, None].expand(L, H, m),
              torch.arange(H, device='cuda')[None, :, None].expand(L, H, m))
        for pool in (s['keys'], s['vals']):
            pool[at[0], dst[0], dst[1], at[1]] = pool[at[0], src[0], src[1], at[1]]
    lengths = torch.clamp(s['lengths'], max=keep)
    return dict(keys=s['keys'], vals=s['vals'], lengths=lengths, kept=kept_all, weight=weight)


def run(state):
    s, case = state, state['case']
    if not own:
        return {'append': _plain_append, 'attend': _plain_attend, 'evict': _plain_evict}[case['kind']](s)
    cache = s['cache']
    if case['kind'] == 'append':
        cache.append(s['k'], s['v'], s['table'], s['starts'], s['lengths'])
        return dict(keys=cache.keys, vals=cache.vals)
    if case['kind'] == 'evict':
        lengths, weight, kept = cache.evict(s['weight'], s['table'], s['lengths'], case['keep'], s['to'],
                                            recent=case['recent'], weight_out=s['weight_out'])
        return dict(keys=cache.keys, vals=cache.vals, lengths=lengths, kept=kept, weight=weight)
    if case['weights']:
        out, weight = cache.attend(s['q'], s['table'], s['starts'], s['lengths'], most=case['tokens'],
                                   weight=s['weight'])      # kept in place, pass after pass, as the plain form does
        return dict(out=out, weight=weight)
    return dict(out=cache.attend(s['q'], s['table'], s['starts'], s['lengths'], most=case['tokens']))


def work(case):
    counts, lengths = _numbers(case)
    M, positions, B = sum(counts), sum(lengths), case['seqs']
    size, qsize = (4 if case[k] == 'f32' else 2 for k in ('dtype', 'query'))
    row = case['heads'] * case['width']
    if case['kind'] == 'append':
        return {'bytes': 2 * M * row * (size + qsize), 'flops': 0}
    if case['kind'] == 'evict':
        kept = sum(min(case['keep'], n) for n in lengths)
        nbytes = case['layers'] * (2 * 2 * kept * row * size + case['heads'] * (4 * positions + 8 * kept))
        return {'bytes': nbytes, 'flops': 0}
    pairs = sum(c * n - c * (c - 1) // 2 for c, n in zip(counts, lengths))
    nbytes = 2 * M * row * case['group'] * qsize + 2 * positions * row * size
    if case['weights']:
        nbytes += 4 * case['heads'] * (2 * positions - M)
    return {'bytes': nbytes, 'flops': 4 * pairs * row * case['group']}


def _exact_attend(s):
    """The definition in 64 bits, one key head and some queries at a time."""
    case = s['case']
    G, E, page = case['group'], case['width'], case['page']
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    weight = s['weight'].double() if case['weights'] else None
    first = 0
    for b in range(case['seqs']):
        c, n = s['counts'][b], s['lens'][b]
        rows = [s['table'][b, :-(-n // page)].long(), slice(None)]
        if weight is not None:
            weight[b, :, n - c:] = 0.0
        for h in range(case['heads']):
            k, v = (p[0][rows[0], :, h].reshape(-1, E)[:n].double() for p in (s['keys'], s['vals']))
            kt = k.t().contiguous()
            step = max(1, (1 << 26) // (G * n))
            for j in range(0, c, step):
                m = min(step, c - j)
                q = s['q'][first + j:first + j + m, h * G:(h + 1) * G].double().reshape(m * G, E)
                score = (q @ kt / math.sqrt(E)).view(m, G, n)
                for_row = torch.arange(n - c + j, n - c + j + m, device='cuda').view(m, 1, 1)
                score = torch.where(torch.arange(n, device='cuda') <= for_row, score, -math.inf)
                p = torch.softmax(score, -1)
                out[first + j:first + j + m, h * G:(h + 1) * G] = (p.view(m * G, n) @ v).view(m, G, E)
                if weight is not None:
                    weight[b, h, :n] += p.sum((0, 1))
        first += c
    return dict(out=out, weight=weight) if case['weights'] else dict(out=out)


def _exact_append(s):
    case = s['case']
    pools = [p.double() for p in (s['keys'], s['vals'])]
    first = 0
    for b in range(case['seqs']):
        c, n = s['counts'][b], s['lens'][b]
        ids = s['table'][b].tolist()
        done = 0
        while done < c:                      # a page's part at a time
            at = n - c + done
            slot = at % case['page']
            m = min(case['page'] - slot, c - done)
            for pool, new in zip(pools, (s['k'], s['v'])):
                pool[0, ids[at // case['page']], slot:slot + m] = new[first + done:first + done + m].double()
            done += m
        first += c
    return dict(keys=pools[0], vals=pools[1])


def _exact_evict(s):
    case = s['case']
    page, keep = case['page'], case['keep']
    pools = [p.double() for p in (s['keys'], s['vals'])]
    kept = torch.full((case['layers'], case['seqs'], case['heads'], keep), -1, dtype=torch.int32, device='cuda')
    weight = torch.zeros(s['weight_out'].shape, dtype=torch.float64, device='cuda')
    lengths = []
    for b in range(case['seqs']):
        n = s['lens'][b]
        m = min(keep, n)
        last = min(case['recent'], m)
        lengths.append(m)
        src = (s['table'][b].long()[:, None] * page + torch.arange(page, device='cuda')).reshape(-1)
        dst = (s['to'][b].long()[:, None] * page + torch.arange(page, device='cuda')).reshape(-1)[:m]
        for layer in range(case['layers']):
            for h in range(case['heads']):
                w = s['weight'][layer, b, h, :n]
                old = w[:n - last]
                # the least weight kept, all above it, and the first of those that have just it
                take = m - last
                mask = torch.zeros(n, dtype=torch.bool, device='cuda')
                mask[n - last:] = True
                if take:
                    least = torch.sort(old, descending=True).values[take - 1]
                    above = old > least
                    same = old == least
                    mask[:n - last] = above | (same & (same.cumsum(0) <= take - above.sum()))
                pos = mask.nonzero()[:, 0]
                kept[layer, b, h, :m] = pos.int()
                weight[layer, b, h, :m] = w[pos].double()
                for pool, old_pool in zip(pools, (s['keys'], s['vals'])):
                    flat = old_pool[layer].reshape(-1, case['heads'], case['width'])
                    pool[layer].view(-1, case['heads'], case['width'])[dst, h] = flat[src[pos], h].double()
    return dict(keys=pools[0], vals=pools[1], lengths=torch.tensor(lengths, dtype=torch.int32, device='cuda'),
                kept=kept, weight=weight)


def exact(case, seed):
    s = _inputs(case, seed)
    return {'append': _exact_append, 'attend': _exact_attend, 'evict': _exact_evict}[case['kind']](s)
