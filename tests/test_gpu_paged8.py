"""The cache in 8 bits on the GPU (vesta/paged8.py): what it holds bit by bit, what it reads back, and its attention
against plain PyTorch in 64 bits on the held values, with the bounds of the 16-bit cache's tests: its operands are these
values exactly. Pool rows that no sequence holds are NaN, table entries past a length are no page."""
import math

import pytest
import torch

import held8
from test_gpu_paged import DT, KINDS, SHAPES, WIDE, Batch, _close, _gen, _gpu, _ints, blocks  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = ('i8', 'e4m3')


def _bytes(t):
    return t.view(torch.uint8)


class Batch8(Batch):
    def __init__(self, counts, lengths, heads=3, group=1, width=64, page=16, dtype='f16', form='i8', query=None, layers=1,
                 spare=1, seed=0):
        from vesta.paged8 import PagedCache8
        gen = _gen(seed, sum(lengths), len(lengths), heads, width, page)
        self.counts, self.lens, self.group, self.page, self.form, self.dt = counts, lengths, group, page, form, dtype
        wide = [-(-n // page) + spare for n in lengths]
        pages = sum(wide) + 2
        self.cache = PagedCache8(pages, heads, width, layers=layers, page=page, dtype=dtype, form=form)
        order = torch.randperm(pages, generator=gen, device='cuda').int()
        self.table = torch.full((len(counts), max(wide)), -7, dtype=torch.int32, device='cuda')
        self.pools = ((self.cache.keys, self.cache.kscales), (self.cache.vals, self.cache.vscales))
        for held, powers in self.pools:
            _bytes(held).fill_(127)
            powers.fill_(255 if form == 'i8' else held8.BIAS[form])
        at = 0
        for b, n in enumerate(wide):
            m = -(-lengths[b] // page)
            self.table[b, :m] = order[at:at + m]
            at += n
            for held, powers in self.pools:
                rows = torch.randn(layers, lengths[b], heads, width, generator=gen, device='cuda')
                rows *= torch.randn(width, generator=gen, device='cuda').exp()
                self.put(b, held, powers, *held8.hold(rows, form, dtype))
        self.starts, self.lengths = _ints([sum(counts[:b]) for b in range(len(counts) + 1)]), _ints(lengths)
        self.q = torch.randn(sum(counts), heads * group, width, generator=gen, device='cuda').mul_(0.8).to(DT[query or dtype])
        self.gen = gen

    def place(self, b):
        p = torch.arange(self.lens[b], device='cuda')
        return self.table[b].long()[p // self.page], p % self.page

    def put(self, b, held, powers, code, byte):
        pages, slots = self.place(b)
        _bytes(held)[:, pages, :, slots] = code.transpose(0, 1)
        powers[:, pages, :, slots] = byte.transpose(0, 1)

    def rows(self, b, pool, layer=0):
        pages, slots = self.place(b)
        powers = self.cache.kscales if pool is self.cache.keys else self.cache.vscales
        return held8.values(_bytes(pool)[layer][pages, :, slots], powers[layer][pages, :, slots],
                            self.form).permute(1, 0, 2).contiguous()


def _same(got, want):
    """The same values, bit by bit but for the NaNs' own and the zeros' sign."""
    assert got.shape == want.shape
    same = (got.double() == want) | (got.isnan() & want.isnan())
    assert bool(same.all()), f'{int((~same).sum())} of {same.numel()}, first at {(~same).nonzero()[0].tolist()}: ' \
                             f'{got[~same][0].item()} for {want[~same][0].item()}'


def _difficult(dtype, new, gen):
    """Blocks of 32 values, [n, 64]: of every magnitude, at the edges between two powers and two elements, zeros and
    values that are not finite among them."""
    top = 16 if new == 'f16' else 127
    x = torch.randn(4000, 64, generator=gen, device='cuda')
    x *= torch.exp2(torch.randint(-30 if new == 'f16' else -140, top, (4000, 1), generator=gen, device='cuda').float())
    near = torch.tensor([127.5, 464.0, 127.0, 448.0, 255.0, 256.0, 1.0, 8.5, 9.5, 0.5, 1.5, 2.5, 63.75, 232.0],
                        device='cuda')
    y = near[torch.randint(14, (4000, 64), generator=gen, device='cuda')]
    y = torch.nextafter(y, y + torch.randint(-1, 2, y.shape, generator=gen, device='cuda'))
    y *= torch.exp2(torch.randint(-16, 8, (4000, 2), generator=gen, device='cuda').float()).repeat_interleave(32, 1)
    z = torch.randint(-1023, 1024, (2000, 64), generator=gen, device='cuda').float() / 8
    w = x[:200].clone()
    w[::3, 5] = math.nan
    w[1::3, 40] = math.inf
    w[2::3, 0] = -math.inf
    w[::2, 32:] = 0
    return torch.cat((x, y, z, w, torch.zeros(1, 64, device='cuda'), -torch.zeros(1, 64, device='cuda'))).to(DT[new])


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,new', [('f16', 'f16'), ('f16', 'f32'), ('bf16', 'bf16'), ('bf16', 'f32')])
def test_what_is_held(dtype, new, form):
    """Every rounding, power and limit as defined, and reading it back gives the values it stands for."""
    from vesta.paged8 import PagedCache8
    x = _difficult(dtype, new, _gen(3))
    n = x.shape[0]
    cache = PagedCache8(n // 64 + 1, 1, 64, page=64, dtype=dtype, form=form)
    table, starts, lengths = torch.arange(n // 64 + 1, dtype=torch.int32, device='cuda')[None], _ints([0, n]), _ints([n])
    k, v = x[:, None].contiguous(), x.flip(0)[:, None].contiguous()
    cache.append(k, v, table, starts, lengths)
    for held, powers, rows in ((cache.keys, cache.kscales, k), (cache.vals, cache.vscales, v)):
        code, byte = held8.hold(rows[:, 0], form, dtype)
        assert torch.equal(powers[0, :, 0].reshape(-1, 2)[:n], byte)
        got = _bytes(held)[0, :, 0].reshape(-1, 64)[:n]
        nan = (byte == 255).repeat_interleave(32, -1)                # its elements are any
        if form == 'e4m3':                                           # either of the two NaNs
            nan = (code & 127 == 127) & (got & 127 == 127)
        assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, code))
        values = held8.values(code, byte, form)
        fine = values.to(DT[dtype]).double()
        assert torch.equal(fine.nan_to_num(7.0), values.nan_to_num(7.0))     # each is a value of the cache's type
        # half a step: of a block's largest or, e4m3, of the value, and the limits' own
        r = rows[:, 0].double()
        big = r.abs().nan_to_num(0, 0, 0).unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)
        ok = r.isfinite() & values.isfinite()
        least = 2.0 ** (held8.LOW[form, dtype] - (1 if form == 'i8' else 10))
        most = (127 if form == 'i8' else 448) * 2.0 ** held8.HIGH[form, dtype]
        off = (values - r.clamp(-most, most)).abs()
        # (the least power: the largest is at least 127.5 / 2 or 464 / 2 of it; subnormals' half step is 2^-10)
        bound = big.clamp_max(2 * most) / 127.5 if form == 'i8' else torch.maximum(r.abs() / 16, big * 2.0 ** -10 / 232)
        assert bool((off <= bound + least)[ok].all())
    for t in (DT[dtype], torch.float32):
        a, b = (torch.full((n, 1, 64), 7.0, dtype=t, device='cuda') for _ in range(2))
        assert cache.read(a, b, table, starts, lengths)[0] is a
        _same(a[:, 0], held8.values(*held8.hold(k[:, 0], form, dtype), form))
        _same(b[:, 0], held8.values(*held8.hold(v[:, 0], form, dtype), form))
    cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype', ('f16', 'bf16'))
def test_every_element_of_every_power(form, dtype):
    """All codes with all bytes that appending may leave are read exactly."""
    from vesta.paged8 import PagedCache8
    low, high = (held8.BIAS[form] + d[form, dtype] for d in (held8.LOW, held8.HIGH))
    powers = torch.arange(low, high + 1, device='cuda').tolist() + ([255] if form == 'i8' else [])
    cache = PagedCache8(len(powers), 1, 64, page=4, dtype=dtype, form=form)
    code = torch.arange(256, device='cuda', dtype=torch.uint8)
    code = torch.where(code == 128, 0, code) if form == 'i8' else code       # (no whole number is held as -128)
    for pool, byte in ((cache.keys, cache.kscales), (cache.vals, cache.vscales)):
        _bytes(pool).copy_(code.view(1, 1, 1, 4, 64).expand(pool.shape))
        byte.copy_(torch.tensor(powers, dtype=torch.uint8, device='cuda').view(1, -1, 1, 1, 1).expand(byte.shape))
    n = 4 * len(powers)
    table = torch.arange(len(powers), dtype=torch.int32, device='cuda')[None]
    for t in (DT[dtype], torch.float32):
        k, v = (torch.empty(n, 1, 64, dtype=t, device='cuda') for _ in range(2))
        cache.read(k, v, table, _ints([0, n]), _ints([n]))
        want = held8.values(_bytes(cache.keys)[0, :, 0], cache.kscales[0, :, 0], form).view(n, 64)
        _same(k[:, 0], want)
        _same(v[:, 0], want)


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,new', [('f16', 'f16'), ('f16', 'f32'), ('bf16', 'bf16'), ('bf16', 'f32')])
@pytest.mark.parametrize('width,page', [(64, 16), (128, 1), (64, 64)])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_append_and_read(dtype, new, form, width, page, shape):
    counts, lengths = SHAPES[shape]
    b = Batch8(counts, lengths, 3, 1, width, page, dtype, form, layers=2)
    M = sum(counts)
    wide = torch.randn(M + 2, 7, width, generator=b.gen, device='cuda').mul_(3).to(DT[new])
    k, v = wide[:, :3], wide[:, 4:]
    want = [[_bytes(t).clone() for t in pool] for pool in b.pools]
    back = [torch.full((M + 2, 3, width), 7.0, dtype=torch.float64, device='cuda') for _ in range(2)]
    i0 = 0
    for i, (c, n) in enumerate(zip(counts, lengths)):
        for j in range(c):
            s = n - c + j
            for (pool, powers), rows, to in zip(want, (k, v), back):
                to[i0 + j] = 0
                if s >= 0:
                    code, byte = held8.hold(rows[i0 + j], form, dtype)
                    pool[1, b.table[i, s // page], :, s % page] = code
                    powers[1, b.table[i, s // page], :, s % page] = byte
                    to[i0 + j] = held8.values(code, byte, form)
        i0 += c
    b.cache.append(k, v, b.table, b.starts, b.lengths, layer=1)
    for pool, w in zip(b.pools, want):
        for t, x in zip(pool, w):
            assert torch.equal(_bytes(t), x)
    out = torch.full((M + 2, 9, width), 7.0, dtype=DT[new], device='cuda')
    b.cache.read(out[:, 1:4], out[:, 5:8], b.table, b.starts, b.lengths, layer=1)
    _same(out[:, 1:4], back[0])
    _same(out[:, 5:8], back[1])
    assert (out[:, [0, 4, 8]] == 7).all()
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width,group,page', [(64, 1, 16), (128, 4, 64), (64, 3, 8), (128, 1, 1), (64, 16, 128)])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_attend(blocks, dtype, query, form, width, group, page, shape):  # noqa: F811
    counts, lengths = SHAPES[shape]
    b = Batch8(counts, lengths, 2, group, width, page, dtype, form, query, seed=shape)
    want, bound, *_ = b.want()
    _close(b.attend(), want, bound)
    _close(b.attend(most=max(counts)), want, bound)
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
def test_sequences_of_many_tiles(blocks, dtype, query, form, width):  # noqa: F811
    b = Batch8([650, 0, 333, 701, 1, 290, 90], [650, 50, 1200, 500, 2000, 290, 0], 2, 2, width, 16, dtype, form, query)
    want, bound, *_ = b.want()
    for most in (None, 701):
        _close(b.attend(most=most), want, bound)
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
def test_attend_long(blocks, dtype, query, form):  # noqa: F811
    for counts, lengths, heads, group in (([1], [5000], 1, 1), ([1, 1], [3001, 64], 4, 4), ([7], [4100], 2, 2),
                                          ([1] * 40, [50 * i for i in range(40)], 2, 1), ([300], [2300], 1, 2)):
        b = Batch8(counts, lengths, heads, group, 64, 32, dtype, form, query)
        want, bound, *_ = b.want(scale=0.3)
        _close(b.attend(scale=0.3), want, bound)
        _close(b.attend(scale=0.3, most=max(counts)), want, bound)
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
def test_every_variant(monkeypatch, dtype, query, form, width):
    """The same batch through every kernel that a rule may pick: two, four or eight waves, positions dealt to parts or
    not, blocks of 16, 128 or 256 rows."""
    from vesta import paged
    b = Batch8([1, 40, 1, 3], [700, 333, 2500, 3], 2, 2, width, 16, dtype, form, query)
    want, bound, *_ = b.want()
    base = dict(EIGHT_WAVES=0, TWO_WAVES=0, WIDE_FROM=WIDE, TWICE=(1 << 30, 0, 0), SPLIT={64: 1 << 30, 128: 1 << 30},
                WIDE_SPLIT=1 << 30, FEW_ROWS=1 << 20)
    parts = dict(SPLIT={64: 0, 128: 0}, WIDE_SPLIT=0)
    for kw in ({}, dict(EIGHT_WAVES=1 << 20), dict(TWO_WAVES=1 << 20), parts, {**parts, 'TARGET': 16, 'PART_STEPS': 1},
               dict(FEW_ROWS=0), dict(FEW_ROWS=0, **parts), dict(FEW_ROWS=0, WIDE_TARGET=1 << 12, WIDE_PART_STEPS=1, **parts),
               dict(RUN=1), dict(WIDE_RUN=64, FEW_ROWS=0), dict(TWICE=(0, 0, 0), FEW_ROWS=0)):
        for name, value in {**base, **kw}.items():
            monkeypatch.setattr(paged, name, value)
        _close(b.attend(), want, bound)
        monkeypatch.undo()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('counts,lengths', [([5, 20], [40, 70]), ([140], [200])])
def test_values_not_finite(blocks, dtype, query, form, width, counts, lengths):  # noqa: F811
    """What is held of a NaN reaches the tokens that see its position, and no other."""
    b = Batch8(counts, lengths, 2, 2, width, 16, dtype, form, query)
    for i, (c, n) in enumerate(zip(counts, lengths)):
        for pos, (pool, powers) in ((n - 1, b.pools[1]), (n - 2, b.pools[0])):
            at = 0, b.table[i, pos // 16], 0, pos % 16
            _bytes(pool)[at][35] = 127
            powers[at][1] = 255 if form == 'i8' else powers[at][1]
    want, bound, *_ = b.want()
    out = b.attend()
    i0 = 0
    for i, (c, n) in enumerate(zip(counts, lengths)):
        assert want[i0:i0 + c - 2].isfinite().all() and want[i0:i0 + c, 2:].isfinite().all()
        assert want[i0 + c - 2:i0 + c, :2].isnan().any()
        i0 += c
    _close(out, want, bound)


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
def test_small_and_large_values(blocks, dtype, query, form):  # noqa: F811
    """Held values at both ends of their type: their least steps, their largest sizes."""
    for power in (-22, 12) if dtype == 'f16' else (-110, 100):
        b = Batch8([3, 40], [40, 200], 2, 1, 64, 16, dtype, form, query)
        for i, n in enumerate(b.lens):
            rows = torch.randn(1, n, 2, 64, generator=b.gen, device='cuda') * 2.0 ** power
            b.put(i, *b.pools[1], *held8.hold(rows, form, dtype))
        want, bound, *_ = b.want()
        if dtype == 'f16':
            # the matrix cores add products as if a subnormal operand were 2^-14: 1 * 2^-24 + 2^-15 * 2^-24 is 2^-24, where
            # 2^-14 * 2^-24 still counts (exactly so on the card); each addition is off by a half step of 2^-14 times
            # the weights, whose sum is 1
            bound = bound + 2.0 ** -14 * (max(b.lens) / 16 + 48) * 2.0 ** -24
        _close(b.attend(), want, bound)


@pytest.mark.parametrize('form', FORMS)
def test_a_long_pool(blocks, form):  # noqa: F811
    """Row offsets past 2^31 bytes in a layer."""
    from vesta.paged8 import PagedCache8
    c = PagedCache8(pages=40000, heads=8, width=128, page=64, dtype='bf16', form=form)     # 2.6e9 elements
    table = _ints([[39999, 1, 32768], [17, 39998, 0]])
    starts, lengths = _ints([0, 130, 260]), _ints([130, 130])
    k, v = (torch.randn(260, 8, 128, generator=_gen(i), device='cuda').bfloat16() for i in range(2))
    q = torch.randn(260, 16, 128, generator=_gen(3), device='cuda').bfloat16()
    c.append(k, v, table, starts, lengths)
    small = PagedCache8(pages=6, heads=8, width=128, page=64, dtype='bf16', form=form)
    t2 = _ints([[0, 1, 2], [3, 4, 5]])
    small.append(k, v, t2, starts, lengths)
    assert torch.equal(_bytes(c.keys)[0, 39999], _bytes(small.keys)[0, 0])
    assert torch.equal(c.vscales[0, 39998], small.vscales[0, 4])
    assert torch.equal(c.attend(q, table, starts, lengths), small.attend(q, t2, starts, lengths))
    a, b = c.read(torch.empty_like(k), torch.empty_like(v), table, starts, lengths)
    x, y = small.read(torch.empty_like(k), torch.empty_like(v), t2, starts, lengths)
    assert torch.equal(a, x) and torch.equal(b, y)
    c.check()


def test_bad_contents_raise_after(blocks):  # noqa: F811
    """What the host cannot see: replaced by something possible, and check() says so (once); nothing is appended for a
    sequence that cannot be, and its rows are read as zeros."""
    b = Batch8([2, 3], [40, 20], 2, 1, 64, 16)
    good = b.table, b.starts, b.lengths
    t, t2 = b.table.clone(), b.table.clone()
    t[1, 0] = t[1, 1] = b.cache.pages
    t2[0, 2] = -1
    for args, text, lost in (((t, *good[1:]), 'page id', slice(2, 5)), ((t2, *good[1:]), 'page id', slice(0, 2)),
                             ((good[0], _ints([0, 2, 900]), good[2]), 'starts', slice(2, 5)),
                             ((good[0], _ints([0, 4, 2]), good[2]), 'starts', slice(4, 5)),
                             ((good[0], _ints([-1, 2, 5]), good[2]), 'starts', slice(0, 2)),
                             ((*good[:2], _ints([40, 1 << 30])), 'length', slice(2, 5)),
                             ((*good[:2], _ints([-3, 20])), 'length', slice(0, 2))):
        before = [[_bytes(x).clone() for x in pool] for pool in b.pools]
        b.cache.attend(b.q, *args)
        with pytest.raises(RuntimeError, match=text):
            b.cache.check()
        k, v = (torch.ones(5, 2, 64, device='cuda') for _ in range(2))
        b.cache.read(k, v, *args)
        assert not k[lost].any() and not v[lost].any()
        with pytest.raises(RuntimeError, match=text):
            b.cache.check()
        b.cache.append(b.q, b.q, *args)
        with pytest.raises(RuntimeError, match=text):
            b.cache.check()
        b.cache.check()
        # (starts of 0, 4 and 2 are four new tokens of the first sequence, which can be)
        rows = {(int(b.table[i, (n - c + j) // 16]), (n - c + j) % 16)
                for i, (c, n) in enumerate(zip((4, 3), b.lens)) for j in range(c)}
        for pool, old in zip(b.pools, before):
            for x, y in zip(pool, old):
                changed = (_bytes(x) != y).flatten(-1).any(-1)[0].any(1)
                assert {tuple(at) for at in changed.nonzero().tolist()} <= rows


@pytest.mark.parametrize('form,dtype', [('i8', 'f16'), ('e4m3', 'bf16')])
@pytest.mark.parametrize('heads,page', [(8, 16), (16, 1), (24, 64), (12, 8)])
def test_heads_taken_together(form, dtype, heads, page):
    """Rows of 128 whose heads a wave of append may take eight of: what it leaves is the held form of each row, in its
    own place alone, from any strides; nothing of a sequence that cannot be."""
    counts, lengths = [1, 5, 0, 17, 3, 1, 2], [1, 70, 33, 17, 2, 400, 65]
    b = Batch8(counts, lengths, heads, 1, 128, page, dtype, form)
    wide = torch.randn(sum(counts) + 1, 2 * heads + 1, 128, generator=b.gen, device='cuda').to(DT[dtype])
    k, v = wide[:, :heads], wide[:, heads + 1:]
    for starts, lost in ((b.starts, ()), (torch.cat((b.starts[:-1], _ints([900]))), (6,))):
        want = [[_bytes(t).clone() for t in pool] for pool in b.pools]
        i0 = 0
        for i, (c, n) in enumerate(zip(counts, lengths)):
            for j in range(c):
                s = n - c + j
                if s >= 0 and i not in lost:
                    for (pool, powers), rows in zip(want, (k, v)):
                        code, byte = held8.hold(rows[i0 + j], form, dtype)
                        pool[0, b.table[i, s // page], :, s % page] = code
                        powers[0, b.table[i, s // page], :, s % page] = byte
            i0 += c
        b.cache.append(k, v, b.table, starts, b.lengths)
        for pool, w in zip(b.pools, want):
            for t, x in zip(pool, w):
                assert torch.equal(_bytes(t), x)
        if lost:
            with pytest.raises(RuntimeError, match='starts'):
                b.cache.check()
        wide.neg_()
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,query', KINDS)
@pytest.mark.parametrize('width,group', [(64, 1), (128, 4)])
def test_rows_loaded_past_the_cache(form, dtype, query, width, group, monkeypatch):
    """The pools of a long decode are loaded another way: the same results."""
    from vesta import paged, paged8
    b = Batch8([1, 1, 2, 0, 1], [900, 1, 333, 70, 2500], 3, group, width, 16, dtype, form, query)
    want, bound, *_ = b.want()
    monkeypatch.setattr(paged, 'EIGHT_WAVES', 0)
    for split in (1 << 30, 0):
        monkeypatch.setattr(paged, 'SPLIT', {64: split, 128: split})
        got = []
        for most in (1 << 60, 0):
            monkeypatch.setattr(paged8, 'ATTEND_PAST', most)
            got.append(b.cache.attend(b.q, b.table, b.starts, b.lengths, most=2))
        _close(got[0], want, bound)
        assert torch.equal(*got)
    b.cache.check()


def test_other_stream_and_graph():
    """Captured calls replay on new contents; two graphs and eager calls in between share nothing."""
    b = Batch8([1, 1, 1], [50, 700, 3], 2, 2, 64, 16, spare=2)
    rows = torch.randn(3, 2, 64, device='cuda').half()
    k, v = (torch.empty_like(rows) for _ in range(2))
    for i, n in enumerate(b.lens):                          # every page of the table's room may be used
        m = -(-n // 16)
        b.table[i, m:m + 1] = b.cache.pages - 1 - i
    q2 = b.q.float()

    def step(k, v):
        b.cache.append(rows, rows, b.table, b.starts, b.lengths)
        b.cache.read(k, v, b.table, b.starts, b.lengths)
        return b.cache.attend(b.q, b.table, b.starts, b.lengths, most=1), b.cache.attend(q2, b.table, b.starts, b.lengths), k, v

    step(k, v)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(torch.empty_like(k), torch.empty_like(v))
        graphs.append((g, got))
    side = torch.cuda.Stream()
    for n in range(4):
        rows.normal_()
        b.q.normal_()
        q2.normal_()
        want = step(k, v)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            eager = step(torch.empty_like(k), torch.empty_like(v))
        torch.cuda.synchronize()
        for got in (eager, *(got for _, got in graphs)):
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        b.lengths -= torch.tensor([1, 1, 0], dtype=torch.int32, device='cuda')
    b.cache.check()


@pytest.mark.parametrize('form', FORMS)
@pytest.mark.parametrize('dtype,new', [('f16', 'f16'), ('f16', 'f32'), ('bf16', 'bf16')])
@pytest.mark.parametrize('width', (64, 128))
def test_rows_behind_a_sequence_that_cannot_be(form, dtype, new, width):
    """Rows behind the last sequence's stay as they are, whatever its length or first start says; its own become 0."""
    b = Batch8([2, 3], [40, 20], 3, 1, width, 16, dtype, form)
    for starts, lengths, text in ((b.starts, _ints([40, 1 << 30]), 'length'), (b.starts, _ints([40, -1]), 'length'),
                                  (_ints([0, -2, 5]), b.lengths, 'starts')):
        k, v = (torch.full((40, 3, width), 7.0, device='cuda', dtype=DT[new]) for _ in range(2))
        b.cache.read(k, v, b.table, starts, lengths)
        assert (k[5:] == 7).all() and (v[5:] == 7).all()
        lost = slice(2, 5) if starts is b.starts else slice(0, 5)
        assert not k[lost].any() and not v[lost].any()
        with pytest.raises(RuntimeError, match=text):
            b.cache.check()


@pytest.mark.parametrize('dtype,query', KINDS)
def test_which_kernels_run(dtype, query, monkeypatch):
    """Of a long decode on both sides of the rule, and of rows whose heads are taken together."""
    from vesta import paged, paged8
    call, names = paged._Launcher.__call__, []

    def named(self, *a):
        names.append(self.name)
        return call(self, *a)

    monkeypatch.setattr(paged._Launcher, '__call__', named)
    b = Batch8([1, 1], [30000, 29000], 8, 1, 128, 64, dtype, 'i8', query)
    size = 2 * min(b.table.numel(), b.cache.pages) * 64 * 8 * 128
    for past, name in ((size, 'pg_attn'), (size - 1, 'pg_attn_past')):
        monkeypatch.setattr(paged8, 'ATTEND_PAST', past)
        b.cache.attend(b.q, b.table, b.starts, b.lengths, most=1)
        assert names[0] == name, names
        names.clear()
    rows = b.q.float() if query == 'f32' else b.q
    b.cache.append(rows, rows, b.table, b.starts, b.lengths)
    assert names == ['pg_append32' if query == 'f32' else 'pg_append16x8']
    b.cache.check()
