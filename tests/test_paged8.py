"""CPU tests of the 8-bit cache's calls (vesta/paged8.py): what is refused, and that every launch asked for covers what
its kernel indexes. The launches are recorded, not made."""
import pytest
import torch

import held8
from vesta import paged, paged8
from vesta.paged8 import PagedCache8


class _Recorder:
    def __init__(self, log):
        self.log = log

    def __getattr__(self, name):
        def launch(grid, block, stream, *vals):
            assert len(vals) == len(paged8.SIGNATURES[name]), name
            paged.struct.pack('@' + ''.join(paged._CODES[c] for c in paged8.SIGNATURES[name]), *vals)
            self.log.append((name, grid, block, vals))
        return launch


class _Dry(PagedCache8):
    """A cache on the CPU whose launches go into ``log``."""

    def __init__(self, *a, dtype='f16', form='i8', **kw):
        kw = {**dict(width=64, layers=1, page=64), **kw}
        self.form = form
        self._shape(*a, kw['width'], kw['layers'], kw['page'], dtype)
        self._allocate(torch.device('cpu'))
        self.log = []
        self._kind = {self.dtype: _Recorder(self.log)}
        if dtype == 'f16':
            self._kind[torch.float32] = _Recorder(self.log)

    def _enter(self):
        return 0, None


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _batch(B=2, N=3, M=5):
    return torch.zeros(B, N, dtype=torch.int32), _ints(*[0] * B, M), _ints(*[M] * B)


def _rows(M, H, E=64, dtype=torch.float16):
    return torch.zeros(M, H, E, dtype=dtype)


@pytest.mark.parametrize('bad', [dict(pages=0), dict(heads=0), dict(page=48), dict(width=80), dict(dtype='f32'),
                                 dict(form='i4'), dict(form=None), dict(dtype='i8'), dict(pages=1 << 20, page=64, heads=32),
                                 dict(pages=1 << 25)])
def test_shapes_refused(bad):
    with pytest.raises(ValueError):
        PagedCache8(**{**dict(pages=4, heads=2), **bad})


def test_no_gpu_raises():
    if torch.cuda.is_available():
        pytest.skip('a GPU is present')
    with pytest.raises(RuntimeError, match='no GPU'):
        PagedCache8(4, 2)


@pytest.mark.parametrize('form,held', [('i8', torch.int8), ('e4m3', torch.float8_e4m3fn)])
@pytest.mark.parametrize('dtype', ('f16', 'bf16'))
@pytest.mark.parametrize('width', (64, 128))
def test_layout(form, held, dtype, width):
    c = _Dry(8, 3, width=width, layers=2, page=16, dtype=dtype, form=form)
    for t, s in ((c.keys, c.kscales), (c.vals, c.vscales)):
        assert t.shape == (2, 8, 3, 16, width) and t.dtype == held and not t.view(torch.uint8).any()
        assert s.shape == (2, 8, 3, 16, width // 32) and s.dtype == torch.uint8
        assert (s == held8.LOW[form, dtype] + held8.BIAS[form]).all()        # zeros as appended ones are held
    table, starts, lengths = _batch()
    k = _rows(5, 3, width, c.dtype)
    for layer in (0, 1):
        c.append(k, k, table, starts, lengths, layer)
        name, grid, block, vals = c.log[-1]
        assert name == 'pg_append16' and grid * block >= 64 * 3 * -(-5 * width // 1024)
        assert vals[6:10] == tuple(t[layer].data_ptr() for t in (c.keys, c.vals, c.kscales, c.vscales))
    c.append(k.float(), k.float(), table, starts, lengths)
    assert c.log[-1][0] == 'pg_append32'
    c.attend(k, table, starts, lengths, 1)
    assert c.log[-1][3][3:7] == tuple(t[1].data_ptr() for t in (c.keys, c.vals, c.kscales, c.vscales))


def test_append_refusals():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    k = _rows(5, 3)
    for args, err in (((k.double(), k, table, starts, lengths), TypeError),
                      ((k.bfloat16(), k, table, starts, lengths), TypeError),
                      ((k, k.float(), table, starts, lengths), TypeError),
                      ((k, _rows(4, 3), table, starts, lengths), ValueError),
                      ((_rows(5, 2), _rows(5, 2), table, starts, lengths), ValueError),
                      ((k, k, table.long(), starts, lengths), TypeError),
                      ((k, k, table, starts[:2], lengths), ValueError),
                      ((k, k, table, None, lengths), TypeError),
                      ((k, k, table, starts, lengths, 1), ValueError)):
        with pytest.raises(err):
            c.append(*args)
        with pytest.raises(err):
            c.read(*args)
    with pytest.raises(ValueError):
        c.append(k.clone().requires_grad_(), k, table, starts, lengths)
    assert not c.log


def test_read():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    both = torch.zeros(5, 7, 64, dtype=torch.float16)
    k, v = both[:, :3], both[:, 4:]
    assert c.read(k, v, table, starts, lengths) == (k, v)
    name, grid, block, vals = c.log[-1]
    assert name == 'pg_read16' and grid * block >= 64 * 3 and vals[2:6] == (7 * 64, 64, 7 * 64, 64)
    c.read(k.float(), v.float(), table, starts, lengths)
    assert c.log[-1][0] == 'pg_read32'
    n = len(c.log)
    one = torch.zeros(1, 3, 64, dtype=torch.float16)
    for bad in ((k, k), (both[:, :3], both[:, 2:5]), (one.expand(5, 3, 64), v), (k, one.expand(5, 3, 64)),
                (k, v[:, :, ::2]), (k.clone().requires_grad_(), v)):
        with pytest.raises(ValueError):
            c.read(*bad, table, starts, lengths)
    assert len(c.log) == n


def test_attend_refusals():
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    q = _rows(5, 6)
    for kw, err in ((dict(q=_rows(5, 4)), ValueError), (dict(q=q.bfloat16()), TypeError), (dict(scale=0.0), ValueError),
                    (dict(most=0), ValueError), (dict(out=q), ValueError), (dict(out=q.float()), TypeError),
                    (dict(table=None), TypeError), (dict(weight=torch.zeros(2, 3, 192)), TypeError),
                    (dict(q=q.clone().requires_grad_()), ValueError)):
        with pytest.raises(err):
            c.attend(**{**dict(q=q, table=table, starts=starts, lengths=lengths), **kw})
    with pytest.raises(ValueError, match='evicts nothing'):
        c.evict(torch.zeros(1, 2, 3, 192), table, lengths, 4, table)
    assert not c.log
    with pytest.raises(TypeError):
        _Dry(8, 3, dtype='bf16').attend(q.float(), table, starts, lengths)


def test_nothing_to_do():
    """No tokens, no sequences, no pages in the table: no launch that would read what is not there."""
    c = _Dry(8, 3)
    for B, M, N in ((2, 0, 3), (0, 0, 3), (0, 4, 3)):
        table = torch.zeros(B, N, dtype=torch.int32)
        starts, lengths = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        c.append(_rows(M, 3), _rows(M, 3), table, starts, lengths)
        c.read(_rows(M, 3), _rows(M, 3), table, starts, lengths)
        assert not c.log
    c.read(_rows(4, 3), _rows(4, 3), torch.zeros(2, 0, dtype=torch.int32), _ints(0, 2, 4), _ints(0, 0))
    assert [e[0] for e in c.log] == ['pg_read16']        # (its rows become zeros)


@pytest.mark.parametrize('form', paged8.FORMS)
def test_definition(form):
    """The definition that the GPU's tests hold the kernels to: elements of a value each, rounded to nearest, ties to even."""
    x = torch.tensor([127.0] + [0.5, 1.5, 2.5, -0.5, -2.5] + [0.0] * 26)
    code, byte = held8.hold(x, form, 'f16')
    assert held8.values(code, byte, form)[0] == (127.0 if form == 'i8' else 128.0)
    if form == 'i8':
        assert held8.values(code, byte, form)[1:6].tolist() == [0.0, 2.0, 2.0, 0.0, -2.0] and byte.tolist() == [133]
        assert held8.hold(x * 1.0040, form, 'f16')[1].tolist() == [134]      # 127.508: the next power
    all_codes = torch.arange(256, dtype=torch.uint8)
    bias = torch.full((8,), held8.BIAS[form], dtype=torch.uint8)
    v = held8.values(all_codes, bias, form)
    held = all_codes.view(torch.int8 if form == 'i8' else torch.float8_e4m3fn).float()
    assert torch.equal(v.nan_to_num(999.0), held.double().nan_to_num(999.0))
    y = torch.randn(1000, 32, generator=torch.Generator().manual_seed(2))
    code, byte = held8.hold(y, form, 'f16')
    if form == 'e4m3':                                   # torch's rounding of the scaled values
        want = (y.double() / held8.power2(byte.long() - 127)).float().to(torch.float8_e4m3fn).view(torch.uint8)
        assert torch.equal(code, want)


def test_tangents_refused():
    """Tensors with a forward-mode tangent are refused as ones whose gradient is recorded are."""
    import torch.autograd.forward_ad as fwd
    c = _Dry(8, 3)
    table, starts, lengths = _batch()
    k = _rows(5, 3)
    with fwd.dual_level():
        d = fwd.make_dual(k, torch.ones_like(k))
        for call in (lambda: c.append(d, k, table, starts, lengths), lambda: c.append(k, d, table, starts, lengths),
                     lambda: c.read(k, d, table, starts, lengths), lambda: c.attend(d, table, starts, lengths),
                     lambda: c.attend(k, table, starts, lengths, out=d)):
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(ValueError, match='tangent'):
                    call()
        assert not c.log
        c.append(k, k, table, starts, lengths)
        assert len(c.log) == 1


class _Named(_Recorder):
    """As on a device, where a kernel's launcher is the same object each time."""

    def __getattr__(self, name):
        launch = super().__getattr__(name)
        setattr(self, name, launch)
        return launch


def _named(*a, **kw):
    c = _Dry(*a, **kw)
    c._kind = {dtype: _Named(c.log) for dtype in c._kind}
    return c


@pytest.mark.parametrize('heads', (3, 8, 12, 16))
@pytest.mark.parametrize('width', (64, 128))
@pytest.mark.parametrize('M', (1, 7, 64, 1001))
def test_waves_of_append_and_read(heads, width, M):
    """Eight heads of 128 in 16 bits are appended together, other rows a head at a time, and the waves are as many as
    the kernels index."""
    c = _named(40, heads, width=width)
    table, starts, lengths = _batch(2, 20, M)
    for dtype in (torch.float16, torch.float32):
        k = _rows(M, heads, width, dtype)
        c.append(k, k, table, starts, lengths)
        together = width == 128 and heads % 8 == 0 and dtype == torch.float16
        name, grid, block, _ = c.log[-1]
        assert name == ('pg_append16x8' if together else 'pg_append16' if dtype == torch.float16 else 'pg_append32')
        waves = M * heads // 8 if together else -(-M // (1024 // width)) * heads
        assert block == 256 and 4 * grid >= waves > 4 * (grid - 1)
        c.read(k, k.clone(), table, starts, lengths)
        name, grid, block, _ = c.log[-1]
        size = k.element_size()
        waves = -(-M // (1024 // (width * size))) * heads
        assert name == f'pg_read{8 * size}' and block == 256 and 4 * grid >= waves > 4 * (grid - 1)


@pytest.mark.parametrize('layers,pages,N', [(1, 300, 100), (3, 300, 100), (1, 150, 100)])
def test_rule_of_rows_past_the_cache(layers, pages, N, monkeypatch):
    """Long decodes whose tables have room for more of all layers' rows than the rule says are loaded past the caches,
    by any type of queries; a chunk whose rows are read again is not."""
    c = _named(pages, 3, layers=layers)
    table, starts, lengths = torch.zeros(2, N, dtype=torch.int32), _ints(0, 1, 2), _ints(1, 1)
    size = 2 * layers * min(2 * N, pages) * 64 * 3 * 64
    for dtype in (torch.float16, torch.float32):
        q = _rows(2, 3, dtype=dtype)
        for past, name in ((size, 'pg_attn'), (size - 1, 'pg_attn_past')):
            monkeypatch.setattr(paged8, 'ATTEND_PAST', past)
            c.log.clear()
            c.attend(q, table, starts, lengths, most=1)
            assert c.log[0][0] == name
        c.log.clear()
        c.attend(_rows(34, 3, dtype=dtype), table, _ints(0, 17, 34), lengths, most=17)
        assert c.log[0][0] == 'pg_attn'
