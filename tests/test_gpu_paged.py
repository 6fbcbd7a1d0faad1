"""The paged cache's operators on the GPU (vesta/paged.py) against plain PyTorch in 64 bits: lengths and chunks around
the edges of the kernels' tiles, empty sequences and rows, pages inside and across tiles, every kind and head width.
Pool rows that no sequence holds are NaN, table entries past a length are no page."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
# pg_wide wherever it is made (not for f32 queries of width 128)
WIDE = {(64, False): (0, 0, 0), (128, False): (0, 0, 0), (64, True): (0, 0, 0), (128, True): (1 << 30, 1 << 30, 0)}
KINDS = [('f16', 'f16'), ('bf16', 'bf16'), ('f16', 'f32')]        # cache, queries


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('no GPU')


@pytest.fixture(params=('rule', 'rows of 16', 'rows of 128', 'rows of 256'))
def blocks(request, monkeypatch):
    """Attention as the rule has it, or by the kernel for few or for many rows throughout."""
    from vesta import paged
    if request.param != 'rule':
        monkeypatch.setattr(paged, 'FEW_ROWS', 1 << 30 if request.param == 'rows of 16' else 0)
        monkeypatch.setattr(paged, 'WIDE_FROM', WIDE)
        monkeypatch.setattr(paged, 'TWICE', (1 << 30, 0, 0))
    if request.param == 'rows of 256':               # of width 128, the others as 128
        monkeypatch.setattr(paged, 'TWICE', (0, 0, 0))
        monkeypatch.setattr(paged, 'WIDE_SPLIT', 1 << 30)


def _gen(*seed):
    return torch.Generator(device='cuda').manual_seed(sum(1009 ** i * int(s) for i, s in enumerate(seed)) % (1 << 31))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


class Batch:
    """Sequences of ``lengths`` with ``counts`` new tokens each in a cache of random pages, all rows drawn."""

    def __init__(self, counts, lengths, heads=3, group=1, width=64, page=16, dtype='f16', query=None, layers=1, spare=1,
                 seed=0, to_rows=0):
        from vesta.paged import PagedCache
        gen = _gen(seed, sum(lengths), len(lengths), heads, width, page)
        self.counts, self.lens, self.group, self.page = counts, lengths, group, page
        B, M = len(counts), sum(counts)
        wide = [-(-n // page) + spare for n in lengths]
        to_wide = -(-to_rows // page)
        pages = sum(wide) + B * to_wide + 2
        self.cache = PagedCache(pages, heads, width, layers=layers, page=page, dtype=dtype)
        order = torch.randperm(pages, generator=gen, device='cuda').int()
        self.table = torch.full((B, max(wide)), -7, dtype=torch.int32, device='cuda')
        self.cache.keys.fill_(math.nan)
        self.cache.vals.fill_(math.nan)
        at = 0
        for b, n in enumerate(wide):
            m = -(-lengths[b] // page)
            self.table[b, :m] = order[at:at + m]
            at += n
            for pool in (self.cache.keys, self.cache.vals):
                rows = torch.randn(layers, lengths[b], heads, width, generator=gen, device='cuda')
                p = torch.arange(lengths[b], device='cuda')
                pool[:, self.table[b].long()[p // page], p % page] = rows.to(pool.dtype)
        self.to = order[at:at + B * to_wide].reshape(B, to_wide).contiguous()
        self.starts, self.lengths = _ints([sum(counts[:b]) for b in range(B + 1)]), _ints(lengths)
        self.q = torch.randn(M, heads * group, width, generator=gen, device='cuda').mul_(1.5).to(DT[query or dtype])
        self.gen = gen

    def rows(self, b, pool, layer=0):
        """Sequence b's rows of ``pool`` in 64 bits, [heads, length, width]."""
        p = torch.arange(self.lens[b], device='cuda')
        return pool[layer][self.table[b].long()[p // self.page], p % self.page].double().permute(1, 0, 2).contiguous()

    def want(self, scale=None, layer=0):
        """Outputs, the bound of their errors, the weights received and theirs, in 64 bits.

        A score (in units of log 2) is off by the fp32 additions of its E products and its own roundings: (E + 6)
        half steps of the sum of its terms' magnitudes (three planes of an fp32 query carry 24 bits: 2 more), the
        exponential by 2^-22; a weight by that times log 2, and by its rounding to the cache's type (fp32 queries:
        three planes cut off to 2^-23) in the output's numerator; weights below 2^-14 of the largest of their tile
        have fp16's fixed step, 2^-25. Sums over n positions are off by one half step an addition in the longest
        chain: tiles of 16 to 64 one after another, their parts, joins: (n / 16 + 48). The output is rounded once."""
        G, E, M = self.group, self.cache.width, self.q.shape[0]
        H = self.cache.heads
        scale = 1 / math.sqrt(E) if scale is None else scale
        out = torch.zeros(M, H * G, E, dtype=torch.float64, device='cuda')
        bound = torch.zeros_like(out)
        S = self.table.shape[1] * self.page
        got = torch.zeros(len(self.counts), H, S, dtype=torch.float64, device='cuda')
        gerr = torch.zeros_like(got)
        f16, f32 = self.cache.dtype == torch.float16, self.q.dtype == torch.float32
        u = 2.0 ** -24
        up = 2.0 ** -23 if f32 else torch.finfo(self.cache.dtype).eps / 2
        i0 = 0
        for b, (c, n) in enumerate(zip(self.counts, self.lens)):
            if c and n:
                k, v = self.rows(b, self.cache.keys, layer), self.rows(b, self.cache.vals, layer)
                q = self.q[i0:i0 + c].double().view(c, H, G, E).permute(1, 2, 0, 3).reshape(H, G * c, E)
                z = (q @ k.transpose(1, 2).contiguous()).view(H, G, c, n) * scale
                mag = (q.abs() @ k.abs().nan_to_num(0, 0, 0).transpose(1, 2).contiguous()).view(H, G, c, n) * scale
                pos = torch.arange(n - c, n, device='cuda')[:, None]
                hidden = torch.arange(n, device='cuda')[None] > pos
                z = z.masked_fill(hidden, -math.inf)
                p = torch.softmax(z, -1)
                p = torch.where(hidden.expand_as(p), torch.zeros_like(p), p)
                top = z.amax(-1, keepdim=True).abs().nan_to_num(0, 0, 0)
                dw = ((E + 8) * mag + 4 * top) * u + 2.0 ** -22          # relative error of a weight, both its parts
                chain = (n / 16 + 48) * u
                worst = (p * dw).sum(-1, keepdim=True)                   # ... of their sum
                vis = v[:, None, None].expand(H, G, c, n, E) if H * G * c * n * E < 1 << 27 else None
                if vis is not None:
                    vm = torch.where(hidden[..., None], torch.zeros((), dtype=v.dtype, device='cuda'), vis)
                    o = (p[..., None] * vm).sum(-2)
                    va = vm.abs().nan_to_num(0, 0, 0)
                    a = (p[..., None] * va).sum(-2)
                    da = ((p * dw)[..., None] * va).sum(-2)
                    floor = va.sum(-2) if f16 else torch.zeros_like(o)
                else:
                    o, a, da, floor = ((w.reshape(H, G * c, n) @ x).view(H, G, c, E) for w, x in
                                       ((p, v), (p, v.abs()), (p * dw, v.abs()), ((~hidden).double().expand_as(p) * f16,
                                                                                 v.abs())))
                e = (up + 2 * chain) * a + da + worst * a + 2.0 ** -25 * floor
                seen = (pos >= 0).view(1, 1, c, 1)
                o, e = torch.where(seen, o, torch.zeros_like(o)), torch.where(seen, e, torch.zeros_like(e))
                out[i0:i0 + c] = o.permute(2, 0, 1, 3).reshape(c, H * G, E)
                bound[i0:i0 + c] = e.permute(2, 0, 1, 3).reshape(c, H * G, E)
                w = torch.where(seen, p, torch.zeros_like(p))
                got[b, :, :n] = w.sum((1, 2))
                gerr[b, :, :n] = (w * (dw + worst + chain + (G * c / 16 + 16) * u)).sum((1, 2))
            i0 += c
        ur = u if f32 else torch.finfo(self.q.dtype).eps / 2
        bound = bound + ur * (out.abs().nan_to_num(0, 0, 0) + bound) + (2.0 ** -25 if self.q.dtype == DT['f16'] else 0)
        return out, bound, got, gerr

    def attend(self, **kw):
        return self.cache.attend(self.q, self.table, self.starts, self.lengths, **kw)


def _close(got, want, bound):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() - bound)
    bad = ~(off <= 0)
    assert not bad.any(), f'{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: ' \
                          f'{got[bad][0].item()} for {want[bad][0].item()}, bound {bound[bad][0].item():.3g}'


# counts, lengths: one token each, around tiles of 16, 32, 64, 128; ragged chunks; sequences of nothing; padded rows
SHAPES = [
    ([1], [1]),
    ([1, 1, 1, 1, 1], [2, 63, 64, 65, 129]),
    ([1, 1, 0, 1], [31, 0, 40, 33]),
    ([3], [3]),
    ([16, 17, 1, 0, 31], [16, 50, 128, 9, 300]),
    ([130, 2, 64], [130, 260, 64]),
    ([33, 5], [40, 3]),
    ([1, 200, 1, 1], [1000, 333, 7, 0]),
]


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width,group,page', [(64, 1, 16), (128, 4, 64), (64, 3, 8), (128, 1, 1), (64, 16, 128)])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_attend(blocks, dtype, query, width, group, page, shape):
    counts, lengths = SHAPES[shape]
    b = Batch(counts, lengths, 2, group, width, page, dtype, query, seed=shape)
    want, bound, got, gerr = b.want()
    _close(b.attend(), want, bound)
    _close(b.attend(most=max(counts)), want, bound)
    S = b.table.shape[1] * page
    old = torch.rand(len(counts), 2, S + 3, generator=b.gen, device='cuda')
    new = torch.full((len(counts), 2, S), -1.0, device='cuda')
    out, w = b.attend(weight=old, weight_out=new)
    _close(out, want, bound)
    for i, (c, n) in enumerate(zip(counts, lengths)):
        got[i, :, :max(n - c, 0)] += old[i, :, :max(n - c, 0)].double()
    _close(w, got, gerr + got.abs() * 2.0 ** -23)
    assert b.attend(weight=old)[1] is old
    _close(old[:, :, :S], got, gerr + got.abs() * 2.0 ** -23)
    assert not old[:, :, S:].any()
    b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
def test_sequences_of_many_tiles(blocks, dtype, query, width):
    """Tiles of several sequences in the order of their steps: ragged ones, one that begins long before its rows, one
    without any, one whose first rows are padding, one of padding alone."""
    b = Batch([650, 0, 333, 701, 1, 290, 90], [650, 50, 1200, 500, 2000, 290, 0], 2, 2, width, 16, dtype, query)
    want, bound, got, gerr = b.want()
    for most in (None, 701):
        out, w = b.attend(most=most, weight=torch.zeros_like(got, dtype=torch.float32))
        _close(out, want, bound)
        _close(w, got, gerr)
        _close(b.attend(most=most), want, bound)
    b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
def test_attend_long(blocks, dtype, query):
    """Contexts of some thousands, few and many sequences, and a scale of the caller's."""
    for counts, lengths, heads, group in (([1], [5000], 1, 1), ([1, 1], [3001, 64], 4, 4), ([7], [4100], 2, 2),
                                          ([1] * 40, [50 * i for i in range(40)], 2, 1), ([300], [2300], 1, 2)):
        b = Batch(counts, lengths, heads, group, 64, 32, dtype, query)
        want, bound, got, gerr = b.want(scale=0.3)
        out, w = b.attend(scale=0.3, weight=torch.zeros_like(got, dtype=torch.float32))
        _close(out, want, bound)
        _close(w, got, gerr)
        _close(b.attend(scale=0.3, most=max(counts)), want, bound)
    b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('counts,lengths', [([5, 20], [40, 70]), ([140], [200])])
def test_values_not_finite(blocks, dtype, query, width, counts, lengths):
    """An infinity or a NaN in a key or value reaches the tokens that see its position, and no other: the outputs of
    those that see none of it are what they are without it, those that do see it get what the formula gives."""
    b = Batch(counts, lengths, 2, 2, width, 16, dtype, query)
    where = []
    for i, (c, n) in enumerate(zip(counts, lengths)):
        for pos, pool, value in ((n - 1, b.cache.vals, math.inf), (n - 3, b.cache.vals, -math.inf),
                                 (n - 4, b.cache.vals, math.nan), (n - 2, b.cache.keys, math.nan)):
            where.append((i, pos, pool, value))
            pool[0, b.table[i, pos // 16], pos % 16, 0, 3] = value
    want, bound, *_ = b.want()
    i0 = 0
    out = b.attend()
    for i, (c, n) in enumerate(zip(counts, lengths)):
        seen = slice(i0, i0 + c - 4)                       # tokens before all of it, and head 1: finite
        assert want[seen].isfinite().all() and want[i0:i0 + c, 2:].isfinite().all()
        i0 += c
    _close(out, want, bound)


@pytest.mark.parametrize('dtype,query', KINDS)
def test_infinite_value_seen_by_all(blocks, dtype, query):
    b = Batch([1, 40], [70, 200], 2, 1, 64, 16, dtype, query)
    for i in range(2):
        b.cache.vals[0, b.table[i, 0], 3, 1, 5] = -math.inf
    want, bound, *_ = b.want()
    assert (want[:, 1, 5] == -math.inf).all() and want.isinf().sum() == 41
    _close(b.attend(), want, bound)


def test_infinite_key_fp32(blocks):
    """A key with an infinity: scores of +-inf, whatever the planes of the query hold: weight 0, or all NaN."""
    b = Batch([9], [100], 1, 1, 64, 16, 'f16', 'f32')
    b.cache.keys[0, b.table[0, 1], 2, 0, 7] = math.inf
    b.q[:, 0, 7] = _ints([0]).float() - 1e-20             # -inf scores: the position has no weight
    want, bound, got, gerr = b.want()
    out, w = b.attend(weight=torch.zeros_like(got, dtype=torch.float32))
    assert want.isfinite().all()
    _close(out, want, bound)
    _close(w, got, gerr)
    b.q[3, 0, 7] = 1.0                                    # +inf: no softmax
    out = b.attend()
    assert out[3].isnan().all() and out[:3].isfinite().all() and out[4:].isfinite().all()


@pytest.mark.parametrize('scale', (1e-30, 1e30))
def test_fp32_queries_of_any_size(blocks, scale):
    b = Batch([4, 1], [60, 33], 2, 1, 128, 16, 'f16', 'f32')
    b.q.mul_(scale)
    want, bound, *_ = b.want(scale=0.1 / scale)
    _close(b.attend(scale=0.1 / scale), want, bound)


@pytest.mark.parametrize('dtype,query', KINDS)
def test_rows_behind_the_last_are_left(blocks, dtype, query):
    counts, lengths = [3, 1], [10, 70]
    b = Batch(counts, lengths, 2, 2, 64, 16, dtype, query)
    want, bound, *_ = b.want()
    q = torch.cat((b.q, b.q.new_full((5, 4, 64), math.nan)))
    out = torch.full_like(q, 7.0)
    assert b.cache.attend(q, b.table, b.starts, b.lengths, out=out) is out
    _close(out[:4], want, bound)
    assert (out[4:] == 7.0).all()
    rows = torch.ones(9, 2, 64, device='cuda')
    before = b.cache.keys.clone(), b.cache.vals.clone()
    b.cache.append(rows, rows, b.table, b.starts, b.lengths)
    changed = (b.cache.keys.isnan() != before[0].isnan()) | (b.cache.keys != before[0]) & ~before[0].isnan()
    assert int(changed.any(-1).any(-1).sum()) <= 4
    b.cache.check()


def test_strided_queries_and_outputs(blocks):
    """Queries that are a part of a fused projection, outputs into a wider row."""
    b = Batch([3, 20, 1], [3, 50, 90], 2, 2, 64, 16)
    want, bound, *_ = b.want()
    wide = torch.randn(24, 8, 64, device='cuda').half()
    wide[:, 2:6] = b.q
    out = torch.zeros(24, 3, 4, 64, device='cuda', dtype=torch.float16)
    b.cache.attend(wide[:, 2:6], b.table, b.starts, b.lengths, out=out[:, 1])
    _close(out[:, 1], want, bound)
    assert not out[:, 0].any() and not out[:, 2].any()
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    _close(b.cache.attend(heads_first, b.table, b.starts, b.lengths), want, bound)


@pytest.mark.parametrize('dtype,new', [('f16', 'f16'), ('f16', 'f32'), ('bf16', 'bf16'), ('bf16', 'f32')])
@pytest.mark.parametrize('width,page', [(64, 16), (128, 1), (64, 64)])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_append(dtype, new, width, page, shape):
    counts, lengths = SHAPES[shape]
    b = Batch(counts, lengths, 3, 1, width, page, dtype, layers=2)
    M = sum(counts)
    k, v = (torch.randn(M, 3, width, generator=b.gen, device='cuda').mul_(3).to(DT[new]) for _ in range(2))
    want = [b.cache.keys.clone(), b.cache.vals.clone()]
    i0 = 0
    for i, (c, n) in enumerate(zip(counts, lengths)):
        for j in range(c):
            s = n - c + j
            if s >= 0:
                for pool, rows in zip(want, (k, v)):
                    pool[1, b.table[i, s // page], s % page] = rows[i0 + j].to(pool.dtype)
        i0 += c
    b.cache.append(k, v, b.table, b.starts, b.lengths, layer=1)
    for pool, w in zip((b.cache.keys, b.cache.vals), want):
        assert torch.equal(pool.view(torch.int16), w.view(torch.int16))
    b.cache.check()


def _evicted(weight, n, keep, recent):
    """Which positions stay, in order, by their definition: a stable sort on the host."""
    m = min(keep, n)
    last = min(recent, m)
    old = weight[:n - last].tolist()
    rank = sorted(range(n - last), key=lambda s: (-math.inf if math.isnan(old[s]) else -old[s], not math.isnan(old[s]), s))
    return sorted(rank[:m - last]) + list(range(n - last, n))


@pytest.mark.parametrize('dtype', ('f16', 'bf16'))
@pytest.mark.parametrize('width,page,to_spare', [(64, 16, 0), (128, 1, 3), (64, 128, 1)])
@pytest.mark.parametrize('keep,recent', [(1, 0), (1, 1), (7, 7), (40, 0), (64, 10), (100, 300), (1500, 16)])
def test_evict(dtype, width, page, to_spare, keep, recent):
    lengths = [0, 1, 39, 40, 64, 101, 1025, 2300]
    b = Batch([0] * 8, lengths, 2, 1, width, page, dtype, layers=2, to_rows=keep + to_spare * page)
    S = b.table.shape[1] * page
    w = torch.randn(2, 8, 2, S, generator=b.gen, device='cuda').exp_()
    w[:, :, 0] = (w[:, :, 0] * 3).round_()                       # many ties, zeros among them
    w[1, 7, 1, 5:900:7] = 0.25
    w[0, 7, 1, 5] = math.inf
    w[0, 7, 1, 1000] = math.nan
    w[0, 6, 1, 8] = -0.0
    w[0, 6, 1, 9] = -3.0
    for i, n in enumerate(lengths):
        w[:, i, :, n:] = 1e30                                    # not looked at
    before = b.cache.keys.clone(), b.cache.vals.clone()
    new, wo, kept = b.cache.evict(w, b.table, b.lengths, keep, b.to, recent=recent)
    assert new.tolist() == [min(n, keep) for n in lengths]
    pools = [(p.clone(), a) for p, a in zip(before, (b.cache.keys, b.cache.vals))]
    for layer in range(2):
        for i, n in enumerate(lengths):
            for h in range(2):
                want = _evicted(w[layer, i, h].cpu(), n, keep, recent)
                m = len(want)
                assert kept[layer, i, h, :m].tolist() == want and (kept[layer, i, h, m:] == -1).all()
                src = torch.tensor(want, dtype=torch.long, device='cuda')
                dst = torch.arange(m, device='cuda')
                assert torch.equal(wo[layer, i, h, :m].nan_to_num(5), w[layer, i, h][src].nan_to_num(5))
                assert not wo[layer, i, h, m:].any()
                for p, _ in pools:
                    p[layer, b.to[i].long()[dst // page], dst % page, h] = \
                        p[layer, b.table[i].long()[src // page], src % page, h]
    for p, got in pools:
        assert torch.equal(p.view(torch.int16), got.view(torch.int16))
    b.cache.check()


def test_bad_contents_raise_after(blocks):
    """What the host cannot see: replaced by something possible, and check() says so (once)."""
    b = Batch([2, 3], [40, 20], 2, 1, 64, 16)
    good = b.table, b.starts, b.lengths
    rows = b.q

    def calls(table, starts, lengths):
        b.cache.attend(b.q, table, starts, lengths)
        b.cache.append(rows, rows, table, starts, lengths)

    t = b.table.clone()
    t[1, 0] = b.cache.pages
    t2 = b.table.clone()
    t2[0, 1] = -1
    for args, text in (((t, *good[1:]), 'page id'), ((t2, *good[1:]), 'page id'),
                       ((good[0], _ints([0, 2, 900]), good[2]), 'starts'),
                       ((good[0], _ints([0, 4, 2]), good[2]), 'starts'),
                       ((good[0], _ints([-1, 2, 5]), good[2]), 'starts'),
                       ((good[0], _ints([0, 5, 0]), good[2]), 'starts'),
                       ((*good[:2], _ints([40, 1 << 30])), 'length'), ((*good[:2], _ints([-3, 20])), 'length')):
        calls(*args)
        with pytest.raises(RuntimeError, match=text):
            b.cache.check()
        b.cache.check()
    # starts that ask for more parts than there can be: left out, none past the workspaces
    n = 70
    many = Batch([1] * n, [300] * n, 2, 1, 64, 16)
    odd = _ints([0 if i % 2 else n for i in range(n + 1)])
    w = torch.zeros(n, 2, many.table.shape[1] * 16, device='cuda')
    many.cache.attend(many.q, many.table, odd, many.lengths, weight=w)
    with pytest.raises(RuntimeError, match='starts'):
        many.cache.check()
    b.cache.attend(b.q, *good, most=1)
    with pytest.raises(RuntimeError, match='most'):
        b.cache.check()
    w = torch.ones(1, 2, 2, b.table.shape[1] * 16, device='cuda')
    b.cache.evict(w, b.table, _ints([40, 99999]), 5, _ints([[0], [1]]))
    with pytest.raises(RuntimeError, match='length'):
        b.cache.check()
    b.cache.evict(w, b.table, b.lengths, 5, _ints([[-1], [b.cache.pages]]))
    with pytest.raises(RuntimeError, match='page id'):
        b.cache.check()


def test_pages_shared_to_read(blocks):
    """Two sequences with the same first pages; each appends to its own."""
    b = Batch([1, 1], [33, 33], 2, 1, 64, 16)
    b.table[1, :2] = b.table[0, :2]
    rows = torch.randn(2, 2, 64, device='cuda').half()
    b.cache.append(rows, rows, b.table, b.starts, b.lengths)
    want, bound, *_ = b.want()
    _close(b.attend(), want, bound)


def test_a_long_pool(blocks):
    """Row offsets past 2^31 bytes and elements in a layer."""
    from vesta.paged import PagedCache
    c = PagedCache(pages=40000, heads=8, width=128, page=64, dtype='bf16')     # 2.6e9 elements
    table = _ints([[39999, 1, 32768], [17, 39998, 0]])
    starts, lengths = _ints([0, 130, 260]), _ints([130, 130])
    k, v = (torch.randn(260, 8, 128, generator=_gen(i), device='cuda').bfloat16() for i in range(2))
    q = torch.randn(260, 16, 128, generator=_gen(3), device='cuda').bfloat16()
    c.append(k, v, table, starts, lengths)
    assert torch.equal(c.keys[0, 39999, 5], k[5]) and torch.equal(c.vals[0, 39998, 63], v[130 + 127])
    small = PagedCache(pages=6, heads=8, width=128, page=64, dtype='bf16')
    t2 = _ints([[0, 1, 2], [3, 4, 5]])
    small.append(k, v, t2, starts, lengths)
    assert torch.equal(c.attend(q, table, starts, lengths), small.attend(q, t2, starts, lengths))
    w = torch.rand(1, 2, 8, 192, generator=_gen(4), device='cuda')
    to = _ints([[39990], [39991]])
    new, _, kept = c.evict(w, table, lengths, 50, to, recent=3)
    for h in range(8):
        assert torch.equal(c.vals[0, 39991, :50, h], v[130 + kept[0, 1, h].long(), h])
    c.check()


def test_other_stream_and_graph():
    """Captured calls replay on new contents; two graphs and eager calls in between share nothing."""
    b = Batch([1, 1, 1], [50, 700, 3], 2, 2, 64, 16, spare=2, layers=1)
    rows = torch.randn(3, 2, 64, device='cuda').half()
    w = torch.zeros(3, 2, b.table.shape[1] * 16, device='cuda')
    for i, n in enumerate(b.lens):                          # every page of the table's room may be used
        m = -(-n // 16)
        b.table[i, m:m + 1] = b.cache.pages - 1 - i
    q2 = b.q.clone()

    def step():
        b.cache.append(rows, rows, b.table, b.starts, b.lengths)
        return b.cache.attend(b.q, b.table, b.starts, b.lengths, most=1), \
            b.cache.attend(q2, b.table, b.starts, b.lengths, weight=w, weight_out=torch.empty_like(w), most=1)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    side = torch.cuda.Stream()
    for k in range(4):
        rows.normal_()
        b.q.normal_()
        q2.normal_()
        w.uniform_()
        want = step()
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            eager = step()
        torch.cuda.synchronize()
        for got in (eager, *(got for _, got in graphs)):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1][0])
            assert torch.equal(got[1][1], want[1][1])
        b.lengths -= torch.tensor([1, 1, 0], dtype=torch.int32, device='cuda')
    b.cache.check()


def test_two_threads():
    """Calls of two threads, each on its own stream: each gets its own answer."""
    import threading
    bs = [Batch([1, 9], [40 + 200 * i, 80], 2, 1, 64, 16, seed=i) for i in range(2)]
    wants = [b.attend() for b in bs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(bs[i].attend(), wants[i]):
                    bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_serving_run():
    """The operators as a server uses them: prompts, decode steps that count weights, eviction when the cache is full,
    decoding on, against a plain 64-bit model of the same rows (which keeps what the operators kept)."""
    from vesta.paged import PagedCache
    H, E, page, keep = 2, 64, 16, 40
    rng = random.Random(5)
    gen = _gen(11)
    cache = PagedCache(64, H, E, page=page, dtype='f16')
    free = list(range(64))
    rng.shuffle(free)
    prompts = [37, 5, 61]
    table = torch.full((3, 5), -1, dtype=torch.int32, device='cuda')
    rows = [[torch.empty(0, H, E, dtype=torch.float64, device='cuda') for _ in range(2)] for _ in range(3)]
    w = torch.zeros(1, 3, H, 5 * page, device='cuda')
    lens = [0, 0, 0]
    for step in range(30):
        counts = prompts if step == 0 else [1, 1 if step != 4 else 0, 1]
        if max(lens) + 1 > 70:                                   # full: everyone goes to 40 positions
            to = _ints([[free.pop() for _ in range(3)] for _ in range(3)])
            old = table.clone()
            lengths, w, kept = cache.evict(w, table, _ints(lens), keep, to, recent=8)
            for b in range(3):
                m = int(lengths[b])
                assert m == min(lens[b], keep)
                for j in range(2):
                    at = kept[0, b, :, :m].long().t()[:, :, None].expand(m, H, E)
                    rows[b][j] = torch.gather(rows[b][j], 0, at)
                lens[b] = m
            free += [p for p in old.flatten().tolist() if p >= 0]
            table = torch.cat((to, torch.full((3, 2), -1, dtype=torch.int32, device='cuda')), 1).contiguous()
            w = torch.cat((w, torch.zeros(1, 3, H, 2 * page, device='cuda')), -1).contiguous()
        lens = [n + c for n, c in zip(lens, counts)]
        for b in range(3):
            for p in range(-(-lens[b] // page)):
                if int(table[b, p]) < 0:
                    table[b, p] = free.pop()
        M = sum(counts)
        k, v, q = (torch.randn(M, H, E, generator=gen, device='cuda') for _ in range(3))
        starts, lengths = _ints([sum(counts[:b]) for b in range(4)]), _ints(lens)
        cache.append(k, v, table, starts, lengths)
        out, _ = cache.attend(q, table, starts, lengths, weight=w[0])
        i0 = 0
        for b, c in enumerate(counts):
            for j, new in enumerate((k, v)):
                rows[b][j] = torch.cat((rows[b][j], new[i0:i0 + c].half().double()))
            K, V = (r.transpose(0, 1).contiguous() for r in rows[b])
            z = q[i0:i0 + c].double().transpose(0, 1).contiguous() @ K.transpose(1, 2).contiguous() / 8
            n = lens[b]
            z = z.masked_fill(torch.arange(n, device='cuda') > torch.arange(n - c, n, device='cuda')[:, None], -math.inf)
            want = (torch.softmax(z, -1) @ V).transpose(0, 1)
            # fp32 queries: scores (of up to about 6) to 70 half steps of their terms' sum (up to about 12)
            # twice, and as many of the values: 2^-24 * 70 * 12 * 2 * 4 = 4e-4; measured far below
            assert (out[i0:i0 + c].double() - want).abs().max().item() < 4e-4 if c else True
            i0 += c
    cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
def test_every_variant(monkeypatch, dtype, query, width):
    """The same batch through every kernel that a rule may pick: two, four or eight waves, positions dealt to parts or not,
    blocks of 16, 128 or 256 rows, weights from kept scores or made again, in slices of the rows or not."""
    from vesta import paged
    b = Batch([1, 40, 1, 3], [700, 333, 2500, 3], 2, 2, width, 16, dtype, query)
    want, bound, got, gerr = b.want()
    base = dict(EIGHT_WAVES=0, TWO_WAVES=0, WIDE_FROM=WIDE, TWICE=(1 << 30, 0, 0), SPLIT={64: 1 << 30, 128: 1 << 30},
                WIDE_SPLIT=1 << 30, FEW_ROWS=1 << 20, SCORES_ROWS=1 << 30)
    parts = dict(SPLIT={64: 0, 128: 0}, WIDE_SPLIT=0)
    for kw in ({}, dict(EIGHT_WAVES=1 << 20), dict(TWO_WAVES=1 << 20), parts, {**parts, 'TARGET': 16, 'PART_STEPS': 1},
               dict(SCORES_MAX=0), dict(SCORES_ROWS=2), dict(EIGHT_WAVES=1 << 20, SCORES_ROWS=40),
               dict(FEW_ROWS=0), dict(FEW_ROWS=0, **parts), dict(FEW_ROWS=0, WEIGH_BLOCKS=1),
               dict(FEW_ROWS=0, WIDE_TARGET=1 << 12, WIDE_PART_STEPS=1, WEIGH_BLOCKS=1 << 20, **parts),
               dict(RUN=1), dict(WIDE_RUN=64, FEW_ROWS=0), dict(WIDE_RUN=3, FEW_ROWS=0),
               dict(TWICE=(0, 0, 0), FEW_ROWS=0), dict(TWICE=(0, 0, 0), FEW_ROWS=0, WEIGH_BLOCKS=1 << 20)):
        for name, value in {**base, **kw}.items():
            monkeypatch.setattr(paged, name, value)
        out, w = b.attend(weight=torch.zeros_like(got, dtype=torch.float32))
        _close(out, want, bound)
        _close(w, got, gerr)
        _close(b.attend(), want, bound)
        monkeypatch.undo()
    b.cache.check()


def test_many_sequences(blocks):
    """More sequences than a wave has lanes, most of them without new tokens."""
    n = 150
    counts = [1 if i % 3 == 0 else 0 for i in range(n)]
    counts[149], counts[64] = 40, 5
    lengths = [3 * i + c for i, c in enumerate(counts)]
    b = Batch(counts, lengths, 1, 1, 64, 16)
    want, bound, got, gerr = b.want()
    for most in (None, 40):
        out, w = b.attend(most=most, weight=torch.zeros_like(got, dtype=torch.float32))
        _close(out, want, bound)
        _close(w, got, gerr)
    counts = [1] * n
    b = Batch(counts, [40 * i + 1 for i in range(n)], 1, 2, 64, 16)
    want, bound, got, gerr = b.want()
    _close(b.attend(most=1), want, bound)
    b.cache.check()


@pytest.mark.parametrize('n', (9000, 40000))
def test_evict_long(n):
    """More positions than a block holds in registers."""
    b = Batch([0, 0], [n, 300], 1, 1, 64, 64, to_rows=n // 2)
    w = torch.randn(1, 2, 1, b.table.shape[1] * 64, generator=b.gen, device='cuda').exp_()
    w[0, 0, 0, 17::5] = 0.5
    w[0, 0, 0, 16::3] = 0.0
    for keep, recent in ((n // 2, 100), (n // 2 - 5, 0), (301, 7)):
        new, wo, kept = b.cache.evict(w, b.table, b.lengths, keep, b.to, recent=recent)
        for i in range(2):
            want = _evicted(w[0, i, 0].cpu(), b.lens[i], keep, recent)
            assert int(new[i]) == len(want) and kept[0, i, 0, :len(want)].tolist() == want
            src, dst = torch.tensor(want, device='cuda'), torch.arange(len(want), device='cuda')
            assert torch.equal(wo[0, i, 0, :len(want)], w[0, i, 0][src])
            assert torch.equal(b.cache.keys[0, b.to[i].long()[dst // 64], dst % 64],
                               b.cache.keys[0, b.table[i].long()[src // 64], src % 64])
    b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('below', (16.5, 24.5, 25.5, 29.5))
def test_a_long_tail_keeps_its_mass(blocks, dtype, query, width, below):
    """One position in 32 takes nearly all of the softmax and has value 0, all others weigh 2^-below of it and have a
    value of 4096: the output is theirs alone, in whatever part, step and wave they come.

    A tail weight is off by its rounding to 16 bits, half a step of itself, or half of fp16's fixed step where it is
    small: 2^-25, of a largest weight of 2^9 at least, so 2^-34 of the largest (bf16 has none; fp32 queries' planes
    carry 24 bits of it); by 2^-22 and 4 half steps of the largest score's fp32 exponent (below half steps of 32 at
    most) otherwise, as is the sum; the sums of up to 3000 positions by a half step each."""
    counts, lengths = [1, 140, 3], [3000, 700, 96]
    b = Batch(counts, lengths, 2, 2, width, 16, dtype, query)
    for i, n in enumerate(lengths):
        p = torch.arange(n, device='cuda')
        at = b.table[i].long()[p // 16], p % 16
        b.cache.keys[0][at] = 0.0
        b.cache.vals[0][at] = 4096.0
        top = p % 32 == 0
        b.cache.keys[0, at[0][top], at[1][top], :, 5] = 1.0
        b.cache.vals[0, at[0][top], at[1][top]] = 0.0
    b.q.zero_()
    b.q[:, :, 5] = 1.0
    scale = below * math.log(2)
    want, *_ = b.want(scale=scale)
    w = 2.0 ** -below
    u = 2.0 ** -24
    rounded = 0.0 if query == 'f32' else max(torch.finfo(DT[dtype]).eps / 2, 2.0 ** -34 / w if dtype == 'f16' else 0.0)
    rel = rounded + 2 * (2.0 ** -22 + 4 * 32 * u) + 3000 * u
    ur = u if query == 'f32' else torch.finfo(DT[query]).eps / 2
    bound = want * (rel + ur) * 1.01 + (2.0 ** -25 if query == 'f16' else 0.0)
    assert (want[0] > 0).all()
    _close(b.attend(scale=scale), want, bound)
    _close(b.attend(scale=scale, most=140), want, bound)


@pytest.mark.parametrize('dtype,query', KINDS)
def test_scores_of_many_millions(blocks, dtype, query):
    """Scores whose fp32 steps are whole numbers, two of them equal: their weights stay in their types' range, equal, and
    each is rounded once (fp32 queries: sums, the exponential's 2^-22 aside, which both have alike, and a division)."""
    b = Batch([1, 40], [70, 200], 2, 1, 64, 16, dtype, query)
    for pool in (b.cache.keys, b.cache.vals):
        pool.nan_to_num_(0.0).zero_()
    for i in range(2):
        for s, v in ((3, 2.0), (50, 4.0)):
            b.cache.keys[0, b.table[i, s // 16], s % 16] = 1000.0
            b.cache.vals[0, b.table[i, s // 16], s % 16] = v
    b.q.fill_(1000.0)
    # log2(e) 6.4e7 times the scale: between 2^24 and 2^27
    for scale in (0.1, 0.21, 0.33, 0.57, 0.77, 1.0, 1.13):
        out = b.attend(scale=scale)
        want = torch.full(out.shape, 3.0, dtype=torch.float64, device='cuda')
        rounded = 8 * 2.0 ** -24 if query == 'f32' else torch.finfo(DT[dtype]).eps
        _close(out, want, want * rounded * 1.01)
    b.cache.check()


@pytest.mark.parametrize('new', ('f16', 'f32'))
def test_an_impossible_sequence_appends_nothing(new):
    """A length past the table or starts that cannot be: the cache's rows stay, those of the other sequences come."""
    b = Batch([2, 3, 1], [16, 48, 16], 2, 1, 64, 16, spare=0)
    b.table[0, 1:], b.table[2, 1:] = b.table[1, 1], b.table[1, 2]      # stale entries behind their own page
    rows = torch.randn(6, 2, 64, generator=b.gen, device='cuda').to(DT[new])
    good = b.starts, b.lengths
    # (starts, lengths, the sequences that are stored)
    for starts, lengths, stored in ((good[0], _ints([49, 48, 16]), (1, 2)), (good[0], _ints([16, 1 << 30, 16]), (0, 2)),
                                    (good[0], _ints([16, -1, 99]), (0,)), (_ints([-1, 2, 5, 6]), good[1], (1, 2)),
                                    (_ints([0, 2, 5, 7]), good[1], (0, 1)), (_ints([0, 2, 5, 4]), good[1], (0, 1))):
        before = b.cache.keys.clone(), b.cache.vals.clone()
        b.cache.append(rows, -rows, b.table, starts, lengths)
        for sign, pool, want in zip((1, -1), (b.cache.keys, b.cache.vals), before):
            for i in stored:
                for j, s in enumerate(range(b.lens[i] - b.counts[i], b.lens[i])):
                    want[0, b.table[i, s // 16], s % 16] = sign * rows[int(good[0][i]) + j].half()
            assert torch.equal(pool.view(torch.int16), want.view(torch.int16))
        with pytest.raises(RuntimeError, match='length|starts'):
            b.cache.check()
        rows = rows + 1


def test_check_waits_for_other_streams():
    """An error of a call that another stream has not reached yet is found, and only once."""
    b = Batch([2], [40], 2, 1, 64, 16)
    x = torch.randn(8192, 8192, device='cuda').bfloat16()
    bad = _ints([1 << 20])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
            x @ x                                        # some 15 ms
        b.cache.append(b.q, b.q, b.table, b.starts, bad)
    with pytest.raises(RuntimeError, match='length'):
        b.cache.check()
    b.cache.check()


@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('parts', (False, True))
@pytest.mark.parametrize('kept', (False, True))
@pytest.mark.parametrize('base', (512.0, 0.75))
def test_every_bit_of_fp32_queries(blocks, monkeypatch, width, parts, kept, base):
    """Outputs and received weights to the last bits of 24, by every kernel (what is lost without a plane, and the bounds:
    paged_planes.py, whose own test plants that on the CPU)."""
    import paged_planes as pp
    from vesta import paged
    if parts:
        for name, value in dict(SPLIT={64: 0, 128: 0}, WIDE_SPLIT=0, PART_STEPS=1, WIDE_PART_STEPS=1, TARGET=16).items():
            monkeypatch.setattr(paged, name, value)
    monkeypatch.setattr(paged, 'SCORES_ROWS', 1 << 30 if kept else 0)
    G = 2
    b = Batch([1, 200, 3], [2, 300, 140], 2, G, width, 16, 'f16', 'f32')
    for pool in (b.cache.keys, b.cache.vals):
        pool.nan_to_num_(0.0).zero_()
    b.cache.keys[..., 2] = -1000.0
    for i in range(3):
        b.cache.keys[0, b.table[i, 0], :2] = 0.0
        for s, v in ((0, 1.0), (1, -1.0)):
            b.cache.keys[0, b.table[i, 0], s, :, s] = 1.0
            b.cache.vals[0, b.table[i, 0], s] = v
    x = pp.gaps(204 * 2 * G, width, base).view(204, 2 * G)
    b.q.zero_()
    b.q[:, :, 0], b.q[:, :, 2] = base, 1.0
    b.q[:, :, 1] = (base - x).to(b.q)
    assert torch.equal(b.q[:, :, 1].double().cpu(), base - x)
    out, bound, w0, w1, rel = pp.answer(x, base)
    got, w = b.attend(scale=pp.SCALE, weight=torch.zeros(3, 2, b.table.shape[1] * 16, device='cuda'))
    wide = [t.cuda()[..., None].expand(204, 2 * G, width) for t in (out, bound)]
    _close(got, *wide)
    _close(b.attend(scale=pp.SCALE), *wide)
    rows = [0, 1, 201, 204]
    for i in range(3):
        for s, one in ((0, w0), (1, w1)):
            want = one[rows[i]:rows[i + 1]].reshape(-1, 2, G).sum((0, 2)).cuda()
            _close(w[i, :, s], want, want * (rel + G * b.counts[i] * 2.0 ** -24))
    assert not w[:, :, 2:].any()
    b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('parts', (False, True))
def test_a_nan_far_below_the_largest_score(blocks, monkeypatch, dtype, query, width, parts):
    """A visible NaN reaches the output whatever its position's weight, also one that fp32 has as 0: 0 * NaN."""
    from vesta import paged
    if parts:
        for name, value in dict(SPLIT={64: 0, 128: 0}, WIDE_SPLIT=0, PART_STEPS=1, WIDE_PART_STEPS=1, TARGET=64).items():
            monkeypatch.setattr(paged, name, value)
    for counts, lengths in (([1, 3], [3000, 200]), ([140], [1500])):
        b = Batch(counts, lengths, 2, 1, width, 16, dtype, query)
        b.q.zero_()
        b.q[:, :, 0] = 1.0
        for i in range(len(counts)):
            for s in range(112):
                b.cache.keys[0, b.table[i, s // 16], s % 16, :, 0] = -400.0
        b.cache.vals[0, b.table[:, 0].long(), 10, 0, 3] = math.nan
        want, bound, *_ = b.want(scale=1.0)
        assert want[:, 0, 3].isnan().all() and want.isnan().sum() == len(want)
        _close(b.attend(scale=1.0), want, bound)
        b.cache.keys[0, b.table[:, 0].long(), 12, 1, 5] = math.nan
        got, w = b.attend(scale=1.0, weight=torch.zeros(len(counts), 2, b.table.shape[1] * 16, device='cuda'))
        assert got[:, 1].isnan().all() and got[:, 0].isnan().sum() == len(want)
        assert w[:, 1, :100].isnan().all() and not w[:, 0].isnan().any()


def test_an_empty_table():
    """Sequences that can hold nothing: their tokens see nothing, as padded rows do."""
    from vesta.paged import PagedCache
    for dtype, query in KINDS:
        c = PagedCache(2, 2, 64, page=16, dtype=dtype)
        q = torch.ones(5, 4, 64, device='cuda', dtype=DT[query])
        out, w = c.attend(q, torch.empty(2, 0, dtype=torch.int32, device='cuda'), _ints([0, 2, 5]), _ints([0, 0]),
                          weight=torch.ones(2, 2, 7, device='cuda'))
        assert not out.any() and not w.any()
        c.append(q[:, :2], q[:, :2], torch.empty(2, 0, dtype=torch.int32, device='cuda'), _ints([0, 2, 5]), _ints([0, 0]))
        c.check()
