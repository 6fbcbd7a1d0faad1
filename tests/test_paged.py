"""CPU tests of the paged cache's calls (vesta/paged.py): what is refused, and
that every launch asked for covers what its kernel indexes. The launches are
recorded, not made."""
import pytest
import torch

from vesta import paged
from vesta.paged import PagedCache


class _Recorder:
    def __init__(self, log):
        self.log = log

    def __getattr__(self, name):
        def launch(grid, block, stream, *vals):
            assert len(vals) == len(paged.SIGNATURES[name]), name
            paged.struct.pack('@' + ''.join(paged._CODES[c] for c in paged.SIGNATURES[name]), *vals)
            self.log.append((name, grid, block, vals))
        return launch


class _Dry(PagedCache):
    """A cache on the CPU whose launches go into ``log``."""

    def __init__(self, *a, dtype='f16', **kw):
        kw = {**dict(width=64, layers=1, page=64), **kw}
        self._shape(*a, kw['width'], kw['layers'], kw['page'], dtype)
        self._allocate(torch.device('cpu'))
        self.log = []
        self._kind = {self.dtype: _Recorder(self.log)}
        if dtype == 'f16':
            self._kind[torch.float32] = _Recorder(self.log)

    def _enter(self):
        return 0, None


def _last(c, *names):
    """The arguments of the last launch of one of ``names``."""
    return [vals for name, _, _, vals in c.log if name in names][-1]


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _batch(B=2, N=3, M=5):
    return torch.zeros(B, N, dtype=torch.int32), _ints(*[0] * B, M), _ints(*[M] * B)


def _rows(M, H, E=64, dtype=torch.float16):
    return torch.zeros(M, H, E, dtype=dtype)


@pytest.mark.parametrize('bad', [dict(pages=0), dict(heads=0), dict(layers=0), dict(page=0), dict(page=48),
                                 dict(page=1 << 17), dict(width=80), dict(dtype='f32'), dict(pages=1 << 25),
                                 dict(heads=1 << 25)])
def test_shapes_refused(bad):
    with pytest.raises(ValueError):
        PagedCache(**{**dict(pages=4, heads=2), **bad})


def test_no_gpu_raises():
    if torch.cuda.is_available():
        pytest.skip('a GPU is present')
    with pytest.raises(RuntimeError, match='no GPU'):
        PagedCache(4, 2)


def test_append_refusals():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    k = _rows(5, 3)
    c.append(k, k, table, starts, lengths)
    assert [e[0] for e in c.log] == ['pg_append16']
    c.append(k.float(), k.float(), table, starts, lengths)
    assert c.log[-1][0] == 'pg_append32' and c.log[-1][1] * 256 >= 5 * 3 * 8
    n = len(c.log)
    for args, err in (((k.double(), k, table, starts, lengths), TypeError),
                      ((k.bfloat16(), k, table, starts, lengths), TypeError),
                      ((k, k.float(), table, starts, lengths), TypeError),
                      ((k, _rows(4, 3), table, starts, lengths), ValueError),
                      ((_rows(5, 2), _rows(5, 2), table, starts, lengths), ValueError),
                      ((_rows(5, 3, 32), _rows(5, 3, 32), table, starts, lengths), ValueError),
                      ((k[0], k[0], table, starts, lengths), ValueError),
                      ((k, k, table.long(), starts, lengths), TypeError),
                      ((k, k, table.t(), starts, lengths), TypeError),
                      ((k, k, table[0], starts, lengths), ValueError),
                      ((k, k, table, starts[:2], lengths), ValueError),
                      ((k, k, table, starts, lengths[:1]), ValueError),
                      ((k, k, table, starts, lengths.long()), TypeError),
                      ((k, k, table, starts, lengths, 1), ValueError),
                      ((k, k, table, starts, lengths, -1), ValueError)):
        with pytest.raises(err):
            c.append(*args)
    assert len(c.log) == n


def test_strides():
    """Any strides of the rows and heads, as the columns of one product's output; not of the values in a row."""
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    qkv = torch.zeros(5, 9, 64, dtype=torch.float16)
    q, k, v = qkv[:, :3], qkv[:, 3:6], qkv[:, 6:]
    c.append(k, v, table, starts, lengths)
    assert c.log[-1][3][2:6] == (9 * 64, 64, 9 * 64, 64)
    c.attend(q, table, starts, lengths)
    attn = ('pg_attn2', 'pg_attn', 'pg_attn8', 'pg_wide')
    assert _last(c, *attn)[1:3] == (9 * 64, 64)
    c.attend(torch.zeros(3, 5, 64, dtype=torch.float16).transpose(0, 1), table, starts, lengths)
    assert _last(c, *attn)[1:3] == (64, 5 * 64)
    odd = torch.zeros(5 * 3 * 64 + 4, dtype=torch.float16)
    for bad in (odd[4:].view(5, 3, 64), torch.zeros(5, 3, 128, dtype=torch.float16)[:, :, ::2],
                torch.zeros(5, 3, 68, dtype=torch.float16)[:, :, :64]):
        with pytest.raises(ValueError):
            c.append(bad, k, table, starts, lengths)
        with pytest.raises(ValueError):
            c.attend(bad, table, starts, lengths)
        with pytest.raises(ValueError):
            c.attend(q, table, starts, lengths, out=bad)


@pytest.mark.parametrize('width,rows,pages,kernel,threads', [
    (64, 500, 20, 'pg_wide', 256), (128, 500, 20, 'pg_wide8', 512), (128, 500, 10, 'pg_wide', 256),
    (128, 60, 40, 'pg_wide', 256)])
def test_rows_of_a_block(width, rows, pages, kernel, threads):
    """Many rows over many positions take blocks of 256 rows at width 128; each tile has a block of the grid."""
    B, H, G = 32, 8, 4
    c = _Dry(8, H, width=width)
    table = torch.zeros(B, pages, dtype=torch.int32)
    starts = torch.arange(B + 1, dtype=torch.int32) * rows
    q = torch.zeros(B * rows, H * G, width, dtype=torch.float16)
    c.attend(q, table, starts, _ints(*[64 * pages] * B), most=rows)
    name, grid, block, vals = c.log[-1]
    assert (name, block) == (kernel, threads)
    tile = 64 * threads // 128
    assert grid >= B * H * -(-rows * G // tile) and grid % 8 == 0


@pytest.mark.parametrize('width,B,pages,parts', [(128, 1, 17, True), (128, 24, 17, False), (128, 24, 70, True),
                                                 (64, 1, 31, False), (64, 1, 40, True), (64, 16, 70, False),
                                                 (64, 16, 90, True), (64, 64, 60, False), (64, 64, 70, True)])
def test_positions_in_parts(width, B, pages, parts):
    """One token a sequence: in one block where there are tiles enough for the chip, in parts over long tables."""
    c = _Dry(8, 8, width=width)
    c.attend(torch.zeros(B, 8, width, dtype=torch.float16), torch.zeros(B, pages, dtype=torch.int32),
             torch.arange(B + 1, dtype=torch.int32), _ints(*[64 * pages] * B), most=1)
    assert (c.log[-1][0] == 'pg_join') == parts
    assert c.log[0][1] > B * 8


def test_attend_refusals():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    q = _rows(5, 6)
    w = torch.zeros(2, 3, 3 * 64)
    for kw, err in ((dict(q=_rows(5, 4)), ValueError), (dict(q=_rows(5, 0)), ValueError),
                    (dict(q=q.bfloat16()), TypeError), (dict(q=q.double()), TypeError), (dict(scale=0.0), ValueError),
                    (dict(scale=-1.0), ValueError), (dict(scale=float('nan')), ValueError),
                    (dict(scale=float('inf')), ValueError), (dict(most=0), ValueError), (dict(most=1.5), TypeError),
                    (dict(scale=1e39), ValueError), (dict(scale=1e-40), ValueError), (dict(out=q), ValueError),
                    (dict(layer=0.0), TypeError),
                    (dict(out=q.float()), TypeError), (dict(out=_rows(4, 6)), ValueError),
                    (dict(out=_rows(1, 6).expand(5, 6, 64)), ValueError),
                    (dict(out=_rows(5, 1).expand(5, 6, 64)), ValueError), (dict(q=None), TypeError),
                    (dict(table=None), TypeError), (dict(lengths=[1, 2]), TypeError), (dict(weight=3), TypeError),
                    (dict(weight=w.half()), TypeError), (dict(weight=w[:, :, :-1]), TypeError),
                    (dict(weight=w[:, :, :-1].contiguous()), ValueError), (dict(weight=w[:1]), ValueError),
                    (dict(weight=w[None]), ValueError), (dict(weight_out=w), ValueError),
                    (dict(weight=w, weight_out=w[:, :, :64].contiguous()), ValueError)):
        with pytest.raises(err):
            c.attend(**{**dict(q=q, table=table, starts=starts, lengths=lengths), **kw})
    assert not c.log
    with pytest.raises(TypeError):
        _Dry(8, 3, dtype='bf16').attend(q.float(), table, starts, lengths)


def test_attend_results():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    for dtype in (torch.float16, torch.float32):
        q = _rows(5, 6, dtype=dtype)
        out = c.attend(q, table, starts, lengths)
        assert out.shape == q.shape and out.dtype == dtype
        assert c.attend(q, table, starts, lengths, out=out) is out
    w = torch.zeros(2, 3, 3 * 64)
    assert c.attend(q, table, starts, lengths, weight=w)[1] is w
    w2 = torch.zeros(2, 3, 200)
    assert c.attend(q, table, starts, lengths, weight=w, weight_out=w2)[1] is w2


def test_nothing_to_do():
    """No tokens, no sequences, no pages in the table: no launch that would read what is not there."""
    c = _Dry(8, 3)
    for B, M, N in ((2, 0, 3), (0, 0, 3), (0, 4, 3), (2, 4, 0)):
        table = torch.zeros(B, N, dtype=torch.int32)
        starts, lengths = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        c.append(_rows(M, 3), _rows(M, 3), table, starts, lengths)
        assert not c.log
        assert c.attend(_rows(M, 6), table, starts, lengths).shape == (M, 6, 64)
        assert not c.log or M and B
        c.log.clear()
        w = torch.zeros(B, 3, N * 64)
        c.attend(_rows(M, 6), table, starts, lengths, weight=w)
        assert all(grid for _, grid, *_ in c.log) and (w.numel() or not any('weigh' in e[0] or 'given' in e[0] for e in c.log))
        c.log.clear()


def test_evict_refusals():
    c = _Dry(8, 3, layers=2)
    table, _, lengths = _batch()
    to = torch.zeros(2, 1, dtype=torch.int32)
    w = torch.zeros(2, 2, 3, 192)
    ok = dict(weight=w, table=table, lengths=lengths, keep=50, to=to)
    new, wo, kept = c.evict(**ok)
    assert new.shape == (2,) and wo.shape == (2, 2, 3, 64) and kept.shape == (2, 2, 3, 50)
    assert [e[0] for e in c.log] == ['pg_select', 'pg_move']
    for kw, err in ((dict(to=table), ValueError), (dict(keep=2.0), TypeError), (dict(recent=None), TypeError),
                    (dict(keep=0), ValueError), (dict(keep=65), ValueError), (dict(recent=-1), ValueError),
                    (dict(weight=w[:1]), ValueError), (dict(weight=w[..., :100].contiguous()), ValueError),
                    (dict(weight=w.half()), TypeError), (dict(to=to[:1]), ValueError), (dict(to=to.long()), TypeError),
                    (dict(weight_out=w[..., :32].contiguous()), ValueError), (dict(weight_out=w), ValueError),
                    (dict(lengths=lengths[:1]), ValueError)):
        with pytest.raises(err):
            c.evict(**{**ok, **kw})
    assert len(c.log) == 2


@pytest.mark.parametrize('kind', paged.KINDS)
@pytest.mark.parametrize('width', paged.WIDTHS)
def test_kernels_compile(width, kind):
    from vesta.launch import compile_code
    code = compile_code(paged.paged_source(width, kind))
    key = b'.vgpr_spill_count'                        # of every kernel: a MessagePack number after the key
    spills = [code[i + len(key)] for i in range(len(code)) if code.startswith(key, i)]
    assert len(spills) == len(paged.kernels_of(width, kind)) and not any(spills)


def test_starts_are_needed():
    """Only eviction does without them: the kernels of the others read them."""
    c = _Dry(8, 3)
    table, _, lengths = _batch()
    k = _rows(5, 3)
    for call in (lambda: c.append(k, k, table, None, lengths), lambda: c.attend(k, table, None, lengths),
                 lambda: c.attend(k, table, None, lengths, weight=torch.zeros(2, 3, 192))):
        with pytest.raises(TypeError, match='starts'):
            call()
    assert not c.log


def test_extend_needs_starts():
    from vesta.gpt2 import VestaGPT2
    c = _Dry(8, 3)
    m = object.__new__(VestaGPT2)
    m.L, m.H, m.E, m.D, m.W = 1, 3, 64, 192, dict(wte=torch.zeros(5, 192, dtype=torch.float16),
                                                  fcw=torch.zeros(1, 192, 768, dtype=torch.float16))
    m._pf = m._paged = None
    table, _, lengths = _batch()
    with pytest.raises(TypeError, match='starts'):
        m.extend(c, _ints(*[0] * 5), _ints(*[0] * 5), table, None, lengths)


def test_whole_numbers_of_any_type():
    """A NumPy number of few bits, as comes out of an array, does not overflow in the addresses and sizes made of it."""
    import numpy as np
    c = _Dry(np.int32(64), np.int8(3), layers=np.int8(40), page=np.int16(64))
    for n in (c.pages, c.heads, c.layers, c.page, c.width):
        assert type(n) is int
    table, starts, lengths = _batch()
    k = _rows(5, 3)
    c.append(k, k, table, starts, lengths, layer=np.int8(39))
    assert c.log[-1][3][6] - c.keys.data_ptr() == 39 * 64 * 64 * 3 * 64 * 2
    c.attend(k, table, starts, lengths, layer=np.int16(39))
    assert c.log[-1][3][3] - c.keys.data_ptr() == 39 * 64 * 64 * 3 * 64 * 2
    q = _rows(2 * 100, 3 * 32)
    starts, lengths = _ints(0, 100, 200), _ints(100, 100)
    c.attend(q, table, starts, lengths, most=100)
    want = c.log[-1]
    c.attend(q, table, starts, lengths, most=np.int8(100))
    assert c.log[-1][:3] == want[:3] and c.log[-1][3][11:21] == want[3][11:21]
    w = torch.zeros(40, 2, 3, 192)
    to = torch.zeros(2, 2, dtype=torch.int32)
    c.evict(w, table, lengths, 120, to, 9)
    want = [e[1:3] for e in c.log[-2:]]
    c.evict(w, table, lengths, np.int8(120), to, np.int8(9))
    assert [e[1:3] for e in c.log[-2:]] == want


def test_evict_numbers_past_32_bits():
    """More recent positions than there can be are all of them; more kept ones than a kernel can count are refused."""
    c = _Dry(8, 1, page=1 << 16)
    w, table, lengths = torch.zeros(1, 1, 1, 1 << 16), torch.zeros(1, 1, dtype=torch.int32), _ints(9)
    c.evict(w, table, lengths, 5, torch.ones(1, 1, dtype=torch.int32), recent=1 << 40)
    assert [e[0] for e in c.log] == ['pg_select', 'pg_move'] and c.log[0][3][7] == 5
    for keep in (5, 1 << 31):
        with pytest.raises(ValueError, match='2.31'):
            c.evict(w, table, lengths, keep, torch.ones(1, 1 << 15, dtype=torch.int32))


def _view(base, at, shape, strides):
    return torch.as_strided(base, shape, strides, at)


def test_outputs_apart_from_queries():
    """out shares no memory with q, by whatever offset, and its rows none with one another; parts of one projection's
    rows do not."""
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    for dtype in (torch.float16, torch.float32):
        flat = torch.zeros(20000, dtype=dtype)
        q = flat[:5 * 384].view(5, 6, 64)
        n = len(c.log)
        for out in (flat[384:6 * 384].view(5, 6, 64),                           # a row on
                    flat[64:5 * 384 + 64].view(5, 6, 64),                       # a head on
                    flat[4 * 384:9 * 384].view(5, 6, 64),                       # the last row
                    _view(flat, 384, (5, 6, 64), (768, 64, 1)),                 # between rows that lie apart, and on others
                    _view(flat, 0, (5, 6, 64), (64, 320, 1)),                   # heads first
                    _view(flat, 10000, (5, 6, 64), (64, 64, 1)),                # rows on heads
                    _view(flat, 10000, (5, 6, 64), (320, 64, 1)), _view(flat, 10000, (5, 6, 64), (64, 256, 1)),
                    _view(flat, 10000, (5, 6, 64), (384, 32, 1)), _view(flat, 10000, (5, 6, 64), (0, 64, 1))):
            with pytest.raises(ValueError, match='out'):
                c.attend(q, table, starts, lengths, out=out)
        assert len(c.log) == n
        for out in (flat[5 * 384:10 * 384].view(5, 6, 64), _view(flat, 5 * 384, (5, 6, 64), (64, 320, 1))):
            assert c.attend(q, table, starts, lengths, out=out) is out
        wide = torch.zeros(5, 18, 64, dtype=dtype)
        for a, b in ((0, 6), (6, 0), (0, 12), (12, 0), (6, 12), (3, 10)):
            c.attend(wide[:, a:a + 6], table, starts, lengths, out=wide[:, b:b + 6])
            heads_first = torch.zeros(18, 5, 64, dtype=dtype).transpose(0, 1)
            c.attend(heads_first[:, a:a + 6], table, starts, lengths, out=heads_first[:, b:b + 6])
            by_head = torch.zeros(6, 18, 64, dtype=dtype).transpose(0, 1)       # 5 of 18 rows a head
            c.attend(by_head[a:a + 5], table, starts, lengths, out=by_head[b:b + 5])
        halves = torch.zeros(5, 6, 128, dtype=dtype)
        for t in (halves, halves.reshape(6, 5, 128).transpose(0, 1)):
            c.attend(t[..., :64], table, starts, lengths, out=t[..., 64:])
            c.attend(t[..., 64:], table, starts, lengths, out=t[..., :64])
            with pytest.raises(ValueError, match='out'):
                c.attend(t[..., :64], table, starts, lengths, out=t[..., 32:96])
        for a, b in ((0, 5), (5, 0), (3, 8), (6, 6)):
            with pytest.raises(ValueError, match='out'):
                c.attend(wide[:, a:a + 6], table, starts, lengths, out=wide[:, b:b + 6])
        one = torch.zeros(1, 12, 64, dtype=dtype)
        args = table, _ints(0, 0, 1), lengths
        c.attend(one[:, :6], *args, out=one[:, 6:])
        with pytest.raises(ValueError, match='out'):
            c.attend(one[:, :6], *args, out=one[:, 5:11])


def test_weights_apart():
    """The new weights are the old ones' own memory, place by place, or none of it; an eviction's none of it."""
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    q = _rows(5, 6)
    flat = torch.zeros(8000)
    w = flat[:6 * 200].view(2, 3, 200)
    for at, S in ((4, 200), (1000, 200), (1199, 192), (0, 192), (0, 201)):
        with pytest.raises(ValueError, match='weight_out'):
            c.attend(q, table, starts, lengths, weight=w, weight_out=flat[at:at + 6 * S].view(2, 3, S))
        with pytest.raises(ValueError, match='weight_out'):
            c.attend(q, table, starts, lengths, weight=flat[at:at + 6 * S].view(2, 3, S), weight_out=w)
    assert not c.log
    for at, S in ((0, 200), (1200, 200), (1300, 192)):
        c.attend(q, table, starts, lengths, weight=w, weight_out=flat[at:at + 6 * S].view(2, 3, S))
    one = _Dry(8, 1)
    one.attend(_rows(2, 2), table[:1], _ints(0, 2), lengths[:1], weight=flat[:200].view(1, 1, 200),
               weight_out=flat[:192].view(1, 1, 192))
    to = torch.ones(2, 1, dtype=torch.int32)
    n = len(c.log)
    for at in (0, 64, 1199):
        with pytest.raises(ValueError, match='weight_out'):
            c.evict(w[None], table, lengths, 5, to, weight_out=flat[at:at + 6 * 64].view(1, 2, 3, 64))
    assert len(c.log) == n
    c.evict(w[None], table, lengths, 5, to, weight_out=flat[1200:1200 + 6 * 64].view(1, 2, 3, 64))


def test_an_error_during_check_is_kept():
    """check() reads and clears the word in one step: what a call of another thread raises next is the next check's."""
    import ctypes
    c = _Dry(8, 3)
    c._wait = lambda: None

    class Device(_Recorder):
        def __getattr__(self, name):
            record = super().__getattr__(name)

            def launch(grid, block, stream, err, took):
                record(grid, block, stream, err, took)
                word = ctypes.c_int.from_address(err)
                ctypes.c_int.from_address(took).value = word.value
                word.value = next_word
            return launch
    c._kind = {c.dtype: Device(c.log)}
    c.err.fill_(1)
    next_word = 4
    with pytest.raises(RuntimeError, match='page id'):
        c.check()
    next_word = 0
    with pytest.raises(RuntimeError, match='length'):
        c.check()
    c.check()
    assert [e[0] for e in c.log] == ['pg_take'] * 3


def test_gradients_are_refused():
    """Nothing here has a backward pass: a tensor whose gradient is being recorded is refused, not answered without."""
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    q, g = _rows(5, 3), _rows(5, 3).requires_grad_()
    w, gw = torch.zeros(2, 3, 192), torch.zeros(2, 3, 192).requires_grad_()
    to = torch.ones(2, 1, dtype=torch.int32)
    calls = (lambda: c.append(g, q, table, starts, lengths), lambda: c.append(q, g, table, starts, lengths),
             lambda: c.attend(g, table, starts, lengths), lambda: c.attend(q, table, starts, lengths, out=g),
             lambda: c.attend(g * 2, table, starts, lengths), lambda: c.attend(q, table, starts, lengths, weight=gw),
             lambda: c.attend(q, table, starts, lengths, weight=w, weight_out=gw),
             lambda: c.evict(gw[None], table, lengths, 5, to))
    for call in calls:
        with pytest.raises(ValueError, match='gradient'):
            call()
    assert not c.log
    with torch.no_grad():
        for call in calls:
            call()
    c.attend(g.detach(), table, starts, lengths)


def test_extend_on_the_models_device():
    """A cache of another device is refused; the model's launches are made with its device the current one."""
    from vesta.gpt2 import VestaGPT2
    c = _Dry(8, 3)
    within = []
    c._enter = lambda: (within.append(1), (0, 'back'))[1]
    c._leave = lambda back: within.append(back)

    class Pass:
        def run(self, *a):
            return list(within)
    m = object.__new__(VestaGPT2)
    m.L, m.H, m.E, m.D, m._pf, m._paged = 1, 3, 64, 192, Pass(), Pass()
    table, starts, lengths = _batch()
    batch = _ints(*[0] * 5), _ints(*[0] * 5), table, starts, lengths
    weights = dict(fcw=torch.zeros(1, 192, 768, dtype=torch.float16))
    m.W = dict(wte=torch.zeros(5, 192, dtype=torch.float16, device='meta'), **weights)
    with pytest.raises(ValueError, match='device'):
        m.extend(c, *batch)
    assert not within
    m.W = dict(wte=torch.zeros(5, 192, dtype=torch.float16), **weights)
    assert m.extend(c, *batch) == [1] and within == [1, 'back']


def test_a_lost_plane_shows():
    """The GPU tests' rows of fp32 queries: right with three planes of queries and weights, off with fewer of either, or
    with weights that are made larger by their exponents."""
    import paged_planes as pp
    for base in pp.BASES:
        x = pp.gaps(400, 1, base)
        out, bound, *_ = pp.answer(x, base)
        wrong = ((3, 2), (1, 3), (3, 1)) + (((2, 3),) if base == 512.0 else ((3, 3, 14),))
        for planes in ((3, 3), *wrong):
            off = ((pp.emulate(x, base, *planes) - out).abs() > bound).sum()
            assert off == 0 if planes == (3, 3) else off > 40, (base, planes, int(off))
    # weights received: the exponent without the query's third plane is 2^-14 less
    x = pp.gaps(400, 1, 512.0)
    _, _, _, w, rel = pp.answer(x, 512.0)
    less = torch.exp2(-(512.0 - pp.cut(512.0 - x, 2))) / (1 + torch.exp2(-x))
    assert ((less - w).abs() > 1.5 * rel * w).all()


def test_tangents_are_refused():
    """Nothing here has a forward-mode derivative either: a tensor with a tangent is refused, in whatever mode of
    recording; one without is taken inside a level too."""
    import torch.autograd.forward_ad as forward
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    q, w, to = _rows(5, 3), torch.zeros(2, 3, 192), torch.ones(2, 1, dtype=torch.int32)
    with forward.dual_level():
        d, dw = (forward.make_dual(t, torch.ones_like(t)) for t in (q, w))
        for call in (lambda: c.append(d, q, table, starts, lengths), lambda: c.append(q, d, table, starts, lengths),
                     lambda: c.attend(d, table, starts, lengths), lambda: c.attend(q, table, starts, lengths, out=d),
                     lambda: c.attend(q, table, starts, lengths, weight=dw),
                     lambda: c.attend(q, table, starts, lengths, weight=w, weight_out=dw),
                     lambda: c.evict(dw[None], table, lengths, 5, to)):
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(ValueError, match='tangent'):
                    call()
        assert not c.log
        c.attend(d.detach(), table, starts, lengths)
        c.append(q, q, table, starts, lengths)
        assert c.log
