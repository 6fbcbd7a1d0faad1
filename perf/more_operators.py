"""A key/value cache held in 8 bits (``vesta.paged8.PagedCache8``) and log probabilities (``vesta.logprobs.logprobs``),
as cases that can be timed and compared.

The cache holds each 32 values of a row as 8-bit elements with one power of two: ``form='i8'`` whole numbers of
+-127 with the least power such that none is clipped, ``form='e4m3'`` 8-bit floats (4 bits of exponent, 3 of fraction,
up to 448) likewise. A case is one call that a serving program makes:

* ``kind='append'``: the new tokens' key and value rows go into the pages. Results: the pool's elements and powers.
* ``kind='read'``: the new tokens' rows of the pool come back as values. Results: those rows.
* ``kind='attend'``: causal attention of each sequence's new tokens over all its positions. Results: the output rows.
* ``kind='logprobs'``: of ``rows`` rows of logits, the log probability of each one's given tokens, the entropy, and
  the ``top`` most likely tokens with theirs. Results: all of these.

``context`` is the longest context before the new tokens and ``tokens`` the most new tokens; the sequences' own numbers
lie between ``ragged`` (a part of 1) times these and these, the first sequence having the most. Pages lie in the pool in
random order, as after some time of serving. ``allowed`` is the share of the vocabulary that a row's mask (of a grammar,
say) leaves; of masked cases one row is left nothing.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False      # False: the plain forms; True: the framework's operators

_DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BLOCK = 32
# the least and largest power of two of a block's elements, for rows that are read as f16 or bf16: every value is one
# of theirs
_POWERS = {('i8', 'f16'): (-24, 9), ('i8', 'bf16'): (-126, 119), ('e4m3', 'f16'): (-15, 7), ('e4m3', 'bf16'): (-117, 119)}
_BIAS = {'i8': 133, 'e4m3': 127}      # what is held is the power and this (an i8 element counts 64ths)


def _cache(name, kind, seqs, context, tokens, heads, group, width, dtype, form, page, ragged=1.0, query=''):
    """``dtype``: what the pool's rows are read as; ``query``: the new rows', the queries' or the results' own."""
    return dict(name=name, kind=kind, seqs=seqs, context=context, tokens=tokens, heads=heads, group=group, width=width,
                dtype=dtype, form=form, query=query or dtype, page=page, ragged=ragged)


def _logits(name, rows, vocab, dtype, given=1, top=0, allowed=1.0):
    return dict(name=name, kind='logprobs', rows=rows, vocab=vocab, dtype=dtype, given=given, top=top, allowed=allowed)


def listed():
    return [
        # the benchmark's 8 rows of GPT-2 small, a decode step's new rows: the smallest call, latency alone
        _cache('append_8x1', 'append', 8, 391, 1, 12, 1, 64, 'f16', 'i8', 64, query='f32'),
        # prompts for a server's batch, ragged, into pages of 16
        _cache('append_32x700', 'append', 32, 300, 700, 8, 1, 128, 'bf16', 'e4m3', 16, ragged=0.3),
        # one page's worth of a conversation taken out to be looked at
        _cache('read_1x64', 'read', 1, 500, 64, 16, 1, 64, 'f16', 'e4m3', 32, query='f32'),
        # whole conversations leave the 8-bit cache for one of 16 bits
        _cache('read_24x2000', 'read', 24, 0, 2000, 25, 1, 64, 'f16', 'i8', 64, ragged=0.2),
        # one user of GPT-2 small, one token: latency alone
        _cache('decode_1_f32', 'attend', 1, 700, 1, 12, 1, 64, 'f16', 'i8', 64, query='f32'),
        # a server's batch of ragged conversations, four query heads to a key head
        _cache('decode_96_gqa', 'attend', 96, 6000, 1, 8, 4, 128, 'bf16', 'e4m3', 16, ragged=0.1),
        # two very long documents asked one question each: few rows, a long axis
        _cache('decode_2_long', 'attend', 2, 120001, 1, 8, 4, 128, 'f16', 'i8', 64, ragged=0.9),
        # chunked prefill of the largest model's 25 heads: ragged chunks after ragged contexts
        _cache('chunk_6x512', 'attend', 6, 450, 512, 25, 1, 64, 'f16', 'i8', 16, ragged=0.05),
        # a long document's next chunk: the most work
        _cache('chunk_1x4096_long', 'attend', 1, 18001, 4096, 8, 4, 128, 'bf16', 'i8', 64),
        # the benchmark's 8 rows after a decode step: the chosen tokens and five alternatives
        _logits('logprobs_8', 8, 50257, 'f32', top=5),
        # prompts of a batch scored, each token by the row before it
        _logits('logprobs_8192', 8192, 50257, 'f32'),
        # a server's step over a larger vocabulary: four candidates a row, a mask that leaves a fifth, 20 alternatives
        _logits('logprobs_200_masked', 200, 128001, 'bf16', given=4, top=20, allowed=0.2),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(('append', 'read', 'attend', 'attend', 'attend', 'logprobs', 'logprobs'))
    if kind == 'logprobs':
        vocab = _spread(rng, 500, 200000)
        rows = _spread(rng, 1, max(1, min(8192, 400 * 1000 * 1000 // vocab)))
        return _logits('', rows, vocab, rng.choice(('f32', 'f16', 'bf16')), given=rng.choice((1, 1, 2, 5)),
                       top=rng.choice((0, 0, 1, 5, 20, 64)), allowed=rng.choice((1.0, 1.0, 0.3, 0.001)))
    width = rng.choice((64, 128))
    heads, group = rng.choice(((12, 1), (16, 1), (25, 1), (8, 4), (4, 7), (1, 16), (2, 3)))
    dtype = rng.choice(('f16', 'bf16'))
    query = rng.choice(('f32', 'f16')) if dtype == 'f16' else dtype if kind == 'attend' else rng.choice(('f32', 'bf16'))
    shape = dict(heads=heads, group=group, width=width, dtype=dtype, form=rng.choice(('i8', 'e4m3')), query=query,
                 page=rng.choice((8, 16, 32, 64, 128)), ragged=rng.choice((0.05, 0.5, 1.0)))
    row = heads * width
    if kind != 'attend':
        tokens = _spread(rng, 1, 4000)
        seqs = _spread(rng, 1, max(1, min(64, 24 * 1024 * 1024 // (row * tokens))))
        return _cache('', kind, seqs, _spread(rng, 1, 1000), tokens, **shape)
    if rng.random() < 0.5:      # a decode step
        context = _spread(rng, 1, 120000)
        seqs = _spread(rng, 1, max(1, min(128, 200 * 1024 * 1024 // (row * context))))
        return _cache('', kind, seqs, context, 1, **shape)
    tokens = _spread(rng, 2, 4096)
    context = 0 if rng.random() < 0.4 else _spread(rng, 1, 18000)
    pairs = tokens * (context + tokens) * group * row
    seqs = _spread(rng, 1, max(1, min(32, int(3e11) // (2 * pairs), 4 * 1024 * 1024 // (tokens * group * heads))))
    return _cache('', kind, seqs, context, tokens, **shape)


def _numbers(case):
    """Each sequence's new tokens and its whole length: the case's own, whatever the seed."""
    rng = random.Random(1000003 * case['seqs'] + 1009 * case['context'] + case['tokens'])
    least = case['ragged']

    def some(most, low):
        return [most] + [max(low, int(round(most * rng.uniform(least, 1.0)))) for _ in range(case['seqs'] - 1)]

    counts = some(case['tokens'], 1)
    return counts, [c + n for c, n in zip(counts, some(case['context'], 0))]


# ---------------------------------------------------------------- the held form, in torch operations
def _hold(x, form, dtype):
    """``x`` [.., width] (f32) as elements [.., width] and powers [.., width / 32]. A block's power is the least with
    which its largest value rounds to an element (i8: below 127.5, e4m3: below 464; of zeros the least), within ``_POWERS``; elements are
    rounded to nearest, a tie to even. All steps are exact but the rounding."""
    x = x.unflatten(-1, (-1, _BLOCK))
    part, exp = torch.frexp(x.abs().amax(-1, keepdim=True))         # the largest is part 2^exp, 1/2 <= part < 1
    up, bits = (127.5 / 128, 7) if form == 'i8' else (464 / 512, 9)
    low, high = _POWERS[form, dtype]
    power = torch.where(part > 0, exp - bits + (part >= up).int(), low).clamp(low, high)
    y = x * torch.exp2(-power.float())
    if form == 'i8':
        held = y.round().clamp(-127, 127).to(torch.int8)
    else:
        step = torch.exp2((torch.frexp(y)[1].clamp_min(-5) - 4).float())     # 2^(exponent - 3), subnormals' 2^-9
        held = ((y / step).round() * step).clamp(-448, 448).to(torch.float8_e4m3fn)
    return held.flatten(-2), (power.squeeze(-1) + _BIAS[form]).to(torch.uint8)


def _values(held, powers, form, dtype=torch.float32):
    """What elements and powers stand for."""
    x = held.to(dtype).unflatten(-1, (-1, _BLOCK))
    return (x * torch.exp2((powers.int() - _BIAS[form]).to(dtype)).unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) * 2 + 1)


def _logit_inputs(case, seed):
    gen = _gen(seed)
    M, V = case['rows'], case['vocab']
    x = torch.empty((M, V), device='cuda').normal_(0.0, 1.0, generator=gen)
    # rows between nearly certain of a token and nearly flat
    x *= torch.exp(torch.empty((M, 1), device='cuda').uniform_(-1.0, 1.6, generator=gen))
    if case['allowed'] < 1:
        x.masked_fill_(torch.rand((M, V), generator=gen, device='cuda') >= case['allowed'], -math.inf)
        x[M // 2].fill_(-math.inf)
    x = x.to(_DTYPES[case['dtype']])
    # tokens that were chosen by it, and others'
    given = torch.randint(V, (M, case['given']), generator=gen, device='cuda', dtype=torch.int32)
    given[:, 0] = torch.where(torch.rand(M, generator=gen, device='cuda') < 0.5, x.argmax(1).int(), given[:, 0])
    return dict(case=case, logits=x, given=given)


def _inputs(case, seed):
    if case['kind'] == 'logprobs':
        return _logit_inputs(case, seed)
    gen = _gen(seed)
    counts, lengths = _numbers(case)
    page, heads, width = case['page'], case['heads'], case['width']
    B, M = case['seqs'], sum(counts)
    # a server's tables have room beyond the present lengths: here two pages
    wide = [-(-n // page) + 2 for n in lengths]
    pages = sum(wide) + 3
    order = torch.randperm(pages, generator=gen, device='cuda').int()
    table = torch.full((B, max(wide)), -1, dtype=torch.int32, device='cuda')
    at = 0
    for b, n in enumerate(wide):
        table[b, :n] = order[at:at + n]
        at += n

    def normal(*shape, scale=1.0):
        return torch.empty(shape, device='cuda').normal_(0.0, scale, generator=gen)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device='cuda')

    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    s = dict(case=case, counts=counts, lens=lengths, table=table, lengths=ints(lengths), starts=ints(starts))
    # a head's dims differ in magnitude, keys' by more
    dims = normal(heads, 1, width, scale=0.7).exp_(), normal(heads, 1, width, scale=0.2).exp_()
    for name, d in zip(('keys', 'vals'), dims):
        held, powers = [], []
        some = max(1, (1 << 27) // (page * heads * width))
        for first in range(0, pages, some):
            x = normal(min(some, pages - first), heads, page, width) * d
            h, p = _hold(x.to(_DTYPES[case['dtype']]).float(), case['form'], case['dtype'])
            held.append(h)
            powers.append(p)
        s[name], s[name[0] + 'scales'] = (torch.cat(t)[None] for t in (held, powers))
    if case['kind'] == 'append':
        s['k'], s['v'] = (normal(M, heads, width, scale=1.5).mul_(d.squeeze(1)).to(_DTYPES[case['query']]) for d in dims)
    elif case['kind'] == 'read':
        s['k'], s['v'] = (torch.zeros(M, heads, width, dtype=_DTYPES[case['query']], device='cuda') for _ in range(2))
    else:
        # scores of a spread between a flat and a peaked softmax
        s['q'] = normal(M, heads * case['group'], width, scale=1.4).to(_DTYPES[case['query']])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / 'vesta-gpu_amd'))
        if case['kind'] == 'logprobs':
            from vesta.logprobs import logprobs
            s['logprobs'] = logprobs
            return s
        from vesta.paged8 import PagedCache8
        _, pages, heads, page, width = s['keys'].shape
        cache = PagedCache8(pages, heads, width, page=page, dtype=case['dtype'], form=case['form'])
        for name in ('keys', 'vals', 'kscales', 'vscales'):
            getattr(cache, name).copy_(s[name])
            s[name] = getattr(cache, name)
        s['cache'] = cache
    return s


# ---------------------------------------------------------------- the plain forms
def _places(s):
    """The page and slot of each new token."""
    counts = (s['starts'][1:] - s['starts'][:-1]).long()
    M = sum(s['counts'])
    b = torch.repeat_interleave(torch.arange(len(counts), device='cuda'), counts, output_size=M)
    pos = torch.arange(M, device='cuda') - s['starts'][b] + s['lengths'][b] - counts[b]
    page = s['case']['page']
    return b, s['table'][b, pos // page].long(), pos % page


def _plain_append(s):
    case = s['case']
    _, pages, slots = _places(s)
    for new, name in (('k', 'keys'), ('v', 'vals')):
        held, powers = _hold(s[new].float(), case['form'], case['dtype'])
        s[name].view(torch.uint8)[0, pages, :, slots] = held.view(torch.uint8)
        s[new + 'scales'][0, pages, :, slots] = powers
    return {name: s[name] for name in ('keys', 'vals', 'kscales', 'vscales')}


def _plain_read(s):
    case = s['case']
    _, pages, slots = _places(s)
    for new, name in (('k', 'keys'), ('v', 'vals')):
        held = s[name].view(torch.uint8)[0, pages, :, slots].view(s[name].dtype)
        s[new].copy_(_values(held, s[new + 'scales'][0, pages, :, slots], case['form']))
    return dict(k=s['k'], v=s['v'])


def _plain_attend(s):
    """All sequences together, padded to the longest and the most new tokens."""
    case = s['case']
    G, H, E, B, C, S = case['group'], case['heads'], case['width'], case['seqs'], max(s['counts']), max(s['lens'])
    counts = (s['starts'][1:] - s['starts'][:-1]).long()
    lengths = s['lengths'].long()
    p = torch.arange(S, device='cuda')
    pages = s['table'][:, p // case['page']].long().clamp_min(0)
    slots = (p % case['page']).expand(B, S)
    there = p < lengths[:, None]
    k, v = (_values(s[name].view(torch.uint8)[0, pages, :, slots].view(s[name].dtype),
                    s[name[0] + 'scales'][0, pages, :, slots], case['form']) for name in ('keys', 'vals'))
    k, v = (t.masked_fill_(~there[:, :, None, None], 0.0).transpose(1, 2) for t in (k, v))        # [B, H, S, E]
    j = torch.arange(C, device='cuda')
    row = (s['starts'][:-1].long()[:, None] + j).clamp_max(s['q'].shape[0] - 1)
    q = s['q'].float()[row].view(B, C, H, G, E).permute(0, 2, 3, 1, 4).reshape(B, H, G * C, E)
    z = torch.matmul(q * (1.0 / math.sqrt(E)), k.transpose(2, 3).contiguous()).view(B, H, G, C, S)
    hidden = p > (lengths - counts)[:, None, None] + j[:, None]                                  # [B, C, S]
    z.masked_fill_(hidden[:, None, None], -math.inf)
    z = torch.exp_(z.sub_(z.amax(-1, keepdim=True)))
    z.div_(z.sum(-1, keepdim=True))
    o = torch.matmul(z.view(B, H, G * C, S), v.contiguous()).view(B, H, G, C, E).permute(0, 3, 1, 2, 4)
    return dict(out=o.reshape(B, C, H * G, E)[j < counts[:, None]].to(s['q'].dtype))


def _plain_logprobs(s):
    x, k, M = s['logits'].float(), s['case']['top'], s['case']['rows']
    top = x.amax(1, keepdim=True)
    d = x - torch.where(top == -math.inf, 0.0, top)                  # -inf for all of a row that allows nothing
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total).clamp_min(-1e30)
    out = dict(given=torch.gather(d, 1, s['given'].long()) - log_total)
    shared = (e * d.clamp_min(-1e30)).sum(1, keepdim=True)
    out['entropy'] = torch.where(total > 0, log_total - shared / total, 0.0).squeeze(1)
    del e
    if k:
        # the order of the values, then of the ids from the lowest, as one whole number
        bits = (x + 0.0).view(torch.int32)
        bits = bits ^ ((bits >> 31) & 0x7fffffff)
        key = (bits.long() << 32) - torch.arange(x.shape[1], device='cuda')
        ids = (-torch.topk(key, k, dim=1).values) & 0xffffffff
        out['top'], out['ids'] = torch.gather(d, 1, ids) - log_total, ids.int()
    return out


def run(state):
    s, case = state, state['case']
    kind = case['kind']
    if not own:
        return {'append': _plain_append, 'read': _plain_read, 'attend': _plain_attend,
                'logprobs': _plain_logprobs}[kind](s)
    if kind == 'logprobs':
        got = s['logprobs'](s['logits'], s['given'], top=case['top'])
        out = dict(given=got.given, entropy=got.entropy)
        return {**out, 'top': got.top, 'ids': got.ids} if case['top'] else out
    cache = s['cache']
    batch = s['table'], s['starts'], s['lengths']
    if kind == 'append':
        cache.append(s['k'], s['v'], *batch)
        return {name: s[name] for name in ('keys', 'vals', 'kscales', 'vscales')}
    if kind == 'read':
        cache.read(s['k'], s['v'], *batch)
        return dict(k=s['k'], v=s['v'])
    return dict(out=cache.attend(s['q'], *batch, most=case['tokens']))


def work(case):
    sizes = {'f32': 4, 'f16': 2, 'bf16': 2}
    if case['kind'] == 'logprobs':
        M = case['rows']
        # a product and a sum of the total, and of the entropy
        return {'bytes': M * (case['vocab'] * sizes[case['dtype']] + 8 * case['given'] + 4 + 8 * case['top']),
                'flops': 4 * M * case['vocab']}
    counts, lengths = _numbers(case)
    M, positions, size = sum(counts), sum(lengths), sizes[case['query']]
    row = case['heads'] * case['width']
    held = row + row // _BLOCK
    if case['kind'] != 'attend':
        return {'bytes': 2 * M * (row * size + held), 'flops': 0}
    pairs = sum(c * n - c * (c - 1) // 2 for c, n in zip(counts, lengths))
    return {'bytes': 2 * M * row * case['group'] * size + 2 * positions * held, 'flops': 4 * pairs * row * case['group']}


# ---------------------------------------------------------------- from the definitions, in 64 bits
_E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]


def _exact_hold(x, form, dtype):
    """The elements and powers of ``x`` (64 bits) by trying each power from the least on, and each element's neighbours."""
    x = x.unflatten(-1, (-1, _BLOCK))
    low, high = _POWERS[form, dtype]
    most = x.abs().amax(-1, keepdim=True)
    bound = 127.5 if form == 'i8' else 464.0
    edges = bound * 2.0 ** torch.arange(low, high, dtype=torch.float64, device='cuda')       # at or past the nth: a larger power
    power = low + torch.searchsorted(edges, most, right=True)
    y = x * 2.0 ** -power.double()
    if form == 'i8':
        held = torch.round(y).clamp(-127, 127)
    else:
        table = torch.tensor(_E4M3, dtype=torch.float64, device='cuda')
        # of two neighbours the nearer, of equally near ones the one whose last bit is 0: the even code
        up = torch.searchsorted(table, y.abs()).clamp(1, len(_E4M3) - 1)
        over, under = table[up] - y.abs(), y.abs() - table[up - 1]
        code = torch.where((over < under) | ((over == under) & (up % 2 == 0)), up, up - 1)
        held = table[code] * torch.where(y < 0, -1.0, 1.0)
    return held.flatten(-2), (power.squeeze(-1) + _BIAS[form]).to(torch.uint8)


def _exact_append(s):
    case = s['case']
    out = dict(keys=s['keys'], vals=s['vals'], kscales=s['kscales'].clone(), vscales=s['vscales'].clone())
    for name in ('keys', 'vals'):
        out[name] = out[name].clone() if case['form'] == 'i8' else out[name].double()
    first = 0
    for b in range(case['seqs']):
        c, n = s['counts'][b], s['lens'][b]
        ids = s['table'][b].tolist()
        done = 0
        while done < c:                      # a page's part at a time
            at = n - c + done
            slot = at % case['page']
            m = min(case['page'] - slot, c - done)
            for name, new in (('keys', s['k']), ('vals', s['v'])):
                h, p = _exact_hold(new[first + done:first + done + m].double(), case['form'], case['dtype'])
                where = 0, ids[at // case['page']], slice(None), slice(slot, slot + m)
                out[name][where] = h.transpose(0, 1).to(out[name].dtype)
                out[name[0] + 'scales'][where] = p.transpose(0, 1)
            done += m
        first += c
    return out


def _rows(s, name, b, h=slice(None)):
    """Sequence b's rows of the pool in 64 bits, [.., length, width]."""
    case, n = s['case'], s['lens'][b]
    ids = s['table'][b, :-(-n // case['page'])].long()
    held, powers = s[name][0].view(torch.uint8)[ids][:, h].view(s[name].dtype), s[name[0] + 'scales'][0][ids][:, h]
    factor = 2.0 ** (powers.double() - _BIAS[case['form']])
    x = (held.double().unflatten(-1, (-1, _BLOCK)) * factor[..., None]).flatten(-2)
    x = x if x.dim() == 4 else x[:, None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_read(s):
    out = {new: torch.cat([_rows(s, name, b)[:, n - c:].transpose(0, 1)
                           for b, (c, n) in enumerate(zip(s['counts'], s['lens']))])
           for new, name in (('k', 'keys'), ('v', 'vals'))}
    return out


def _exact_attend(s):
    """The definition, one key head and some queries at a time."""
    case = s['case']
    G, E = case['group'], case['width']
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device='cuda')
    first = 0
    for b in range(case['seqs']):
        c, n = s['counts'][b], s['lens'][b]
        for h in range(case['heads']):
            k, v = (_rows(s, name, b, h)[0] for name in ('keys', 'vals'))
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
        first += c
    return dict(out=out)


def _exact_logprobs(s):
    case = s['case']
    got = []
    some = max(1, (1 << 27) // case['vocab'])
    for i in range(0, case['rows'], some):
        x = s['logits'][i:i + some].double()
        lp = torch.log_softmax(x, 1)
        none = torch.isneginf(x).all(1)
        lp[none] = -math.inf
        p = lp.exp()
        part = [lp.gather(1, s['given'][i:i + some].long()), -torch.where(p > 0, p * lp, 0.0).sum(1)]
        if case['top']:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case['top']]
            part += [lp.gather(1, order), order.int()]
        got.append(part)
    return dict(zip(('given', 'entropy', 'top', 'ids'), (torch.cat(t) for t in zip(*got))))


def exact(case, seed):
    s = _inputs(case, seed)
    return {'append': _exact_append, 'read': _exact_read, 'attend': _exact_attend, 'logprobs': _exact_logprobs}[case['kind']](s)
