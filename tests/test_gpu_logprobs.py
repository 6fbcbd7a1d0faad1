"""Log probabilities on the GPU (vesta/logprobs.py) against plain PyTorch in 64 bits: odd vocabularies and pitches, bans,
ties, NaNs, one row and many, parts of rows and whole ones."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('no GPU')


LAYOUTS = {                                                # kernel, threads, parts of a row
    'rule': None, 'a wave': ('lp_rows64', 64, 1), 'a block of 256': ('lp_rows256', 256, 1),
    'a block of 512': ('lp_rows512', 512, 1), 'a block of 1024': ('lp_rows1024', 1024, 1),
    '3 blocks': ('lp_rows256', 256, 3), '64 blocks': ('lp_rows1024', 1024, 64), 'parts of 2': ('lp_part2', 256, 0),
    'parts of 4': ('lp_part4', 256, 0), 'parts of 8': ('lp_part8', 256, 0)}


@pytest.fixture(params=LAYOUTS)
def layout(request, monkeypatch):
    """Rows as the rule has them, or by one kernel, whole or in parts."""
    from vesta import logprobs as lp
    if request.param != 'rule':
        name, threads, parts = LAYOUTS[request.param]

        def fixed(M, V, size, top):
            if parts == 0 and V < 16 // size:              # less than a load
                return 'lp_rows64', 64, 1, V
            each = -(-V // parts) if parts else 256 * int(name[-1]) * 16 // size
            if parts == 0 and V > each:                    # (parts of the same size, of whole loads)
                each = -(-V // -(-V // each) // (16 // size)) * (16 // size)
            return name, threads, -(-V // each), each

        monkeypatch.setattr(lp, '_layout', fixed)


def _gen(*seed):
    return torch.Generator(device='cuda').manual_seed(sum(1009 ** i * int(s) for i, s in enumerate(seed)) % (1 << 31))


def _check(x, given, top):
    """The call's results for rows x.

    A term e^(x - m) is off by 2^-22 of itself from the exponential and by the rounding of x - m times log2 e, two half
    steps of |x - m| log2 e: its share of S by that times itself, of which the sum is bounded with the terms; a chain of
    additions is V / 256 (a thread's) and 32 of lanes, waves and parts; log S and the differences are rounded once each."""
    from vesta.logprobs import logprobs
    got = logprobs(x, given, top=top)
    M, V = x.shape
    x = x.double()
    m = x.amax(1, keepdim=True)
    d = x - torch.where(m == -math.inf, 0.0, m)
    e = torch.where(x == -math.inf, 0.0, torch.exp(d))
    S = e.sum(1, keepdim=True)
    none = S == 0
    u = 2.0 ** -24
    log_s = torch.where(none, 0.0, torch.log(S))
    fin = torch.where(x == -math.inf, 0.0, d)
    T = (e * fin).sum(1, keepdim=True)
    H = torch.where(none, 0.0, log_s - T / S)
    chain = (V / 256 + 32) * u
    ds = ((e * (4 * u + 4 * u * fin.abs())).sum(1, keepdim=True) / S).nan_to_num(0) + chain          # relative, of S
    dt = ((e * (4 * u + 4 * u * fin.abs()) * fin.abs()).sum(1, keepdim=True) / S).nan_to_num(0) \
        + (T / S).abs().nan_to_num(0) * (chain + ds + 4 * u)
    err = ds + 4 * u * (log_s.abs() + 1)
    lp = d - log_s

    def close(a, want, bound):
        a = a.double()
        same = (a == want) | (a.isnan() & want.isnan())
        bad = ~(torch.where(same, 0.0, (a - want).abs() - bound) <= 0)
        assert not bad.any(), (int(bad.sum()), a[bad][0].item(), want[bad][0].item(), bound.expand_as(want)[bad][0].item())

    close(got.entropy, H.squeeze(1), (err + dt).squeeze(1))
    if given is None:
        assert got.given is None
    else:
        g = given.view(M, -1).long()
        inside = (g >= 0) & (g < V)
        want = torch.where(inside, lp.gather(1, g.clamp(0, V - 1)), math.nan).view(given.shape)
        bound = err + 4 * u * want.view(M, -1).abs().nan_to_num(0, 0, 0)
        assert got.given.shape == given.shape
        close(got.given, want, bound.view(given.shape))
    if top == 0:
        assert got.top is None and got.ids is None
        return got
    order = torch.sort(torch.where(x.isnan(), math.inf, x), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.ids.long(), order)
    want = lp.gather(1, order)
    close(got.top, want, err + 4 * u * want.abs().nan_to_num(0, 0, 0))
    return got


VOCABS = (1, 2, 3, 7, 64, 65, 255, 1000, 1023, 4097, 50257)


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', VOCABS)
def test_rows(layout, kind, V):
    gen = _gen(V, len(kind))
    x = torch.randn(5, V, generator=gen, device='cuda').mul_(3)
    x[1] *= 8
    x[2] /= 100
    x = x.to(DT[kind])
    given = torch.randint(V, (5,), generator=gen, device='cuda')
    for top in sorted({0, 1, min(V, 5), min(V, 20), min(V, 64)}):
        _check(x, given, top)
    _check(x, torch.randint(-1, V + 2, (5, 3), generator=gen, device='cuda', dtype=torch.int32), 1)
    _check(x, None, 1)


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (3, 100, 1000, 4097, 50257))
@pytest.mark.parametrize('share', (0.0, 0.0005, 0.2))
def test_bans(layout, kind, V, share):
    """Rows of which little or nothing is allowed: the rest follows by id."""
    gen = _gen(V, 7)
    x = torch.randn(6, V, generator=gen, device='cuda').mul_(2).to(DT[kind])
    x.masked_fill_(torch.rand(6, V, generator=gen, device='cuda') >= share, -math.inf)
    x[0, V // 2] = 1.0                                     # one allowed
    x[1, 0] = -3.0
    x[2] = -math.inf
    x[3, V - 1] = torch.finfo(DT[kind]).min                # the type's lowest value beside -inf
    x[4] = torch.finfo(DT[kind]).min
    x[4, V // 3] = 0.0
    given = torch.stack((torch.full((6,), V // 2, device='cuda'), torch.zeros(6, dtype=torch.long, device='cuda')), 1)
    got = _check(x, given, min(V, 20))
    assert got.entropy[2] == 0 and (got.given[2] == -math.inf).all() and (got.top[2] == -math.inf).all()


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (5, 300, 50257))
def test_ties(layout, kind, V):
    """Equal logits, signed zeros among them: the lowest ids first, however many."""
    x = torch.zeros(5, V, device='cuda', dtype=DT[kind])
    x[0, ::2] = -0.0
    x[1] = torch.arange(V, device='cuda').remainder(3).to(x.dtype)
    x[2, :V // 2] = 1.0
    x[3] = -torch.arange(V, device='cuda').div(200, rounding_mode='floor').to(x.dtype)
    x[4] = torch.arange(V, device='cuda').div(2000, rounding_mode='floor').to(x.dtype)
    _check(x, torch.zeros(5, dtype=torch.long, device='cuda'), min(V, 64))
    _check(x, None, 1)


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (4, 1000, 50257))
def test_not_finite(layout, kind, V):
    """A NaN or +inf makes its own row NaN and no other, its ids are in order."""
    from vesta.logprobs import logprobs
    x = torch.randn(5, V, generator=_gen(V), device='cuda').to(DT[kind])
    x[1, V // 2] = math.nan
    x[2, V - 1] = math.inf
    x[3, 1] = math.nan
    x[3, 2] = math.inf
    x[3, 3] = -math.inf
    given = torch.zeros(5, dtype=torch.int32, device='cuda')
    got = logprobs(x, given, top=3)
    for t in (got.given, got.entropy, got.top):
        assert t[1:4].isnan().all() and t[[0, 4]].isfinite().all()
    assert got.ids[1, 0] == V // 2 and got.ids[2, 0] == V - 1 and got.ids[3, :2].tolist() == [1, 2]
    rest = torch.sort(x[1].nan_to_num(math.inf), descending=True, stable=True).indices[:3]
    assert got.ids[1].tolist() == rest.tolist()
    _check(x[[0, 4]], given[:2], 3)


def test_pitches_and_offsets(layout):
    """Rows inside a wider tensor, at any alignment, of which nothing beside them is read as theirs."""
    for kind in DT:
        wide = torch.full((6, 1100), math.nan, device='cuda', dtype=DT[kind])
        for at in range(9):
            x = wide[:, at:at + 1003]
            x.copy_(torch.randn(6, 1003, generator=_gen(at), device='cuda'))
            _check(x, torch.arange(6, device='cuda') * 200, 7)
            wide.fill_(math.nan)
        x = torch.randn(1, 700, generator=_gen(1), device='cuda').to(DT[kind])
        _check(x.expand(4, 700), torch.arange(4, device='cuda'), 3)


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('M,V', [(1, 200001), (3, 1 << 20), (300, 9001), (2000, 513)])
def test_sizes(kind, M, V):
    gen = _gen(M, V)
    x = torch.randn(M, V, generator=gen, device='cuda').mul_(4).to(DT[kind])
    given = torch.randint(V, (M, 2), generator=gen, device='cuda')
    for top in (0, 10):
        _check(x, given, top)


def test_nearly_certain():
    """Rows of one token far above the rest: log probabilities near 0 and small entropies."""
    x = torch.zeros(40, 3001, device='cuda')
    x[:, 77] = torch.arange(40, device='cuda') * 1.0
    _check(x, torch.full((40,), 77, device='cuda'), 2)


def test_a_large_offset():
    """Rows past 2^31 elements."""
    V = 300007
    x = torch.zeros(7300, V, device='cuda', dtype=torch.float16)                    # 2.19e9 elements
    x[-3:] = torch.randn(3, V, generator=_gen(9), device='cuda').half()
    from vesta.logprobs import logprobs
    given = torch.arange(7300, device='cuda')
    got = logprobs(x, given, top=5)
    last = _check(x[-3:], given[-3:], 5)
    assert torch.equal(got.ids[-3:], last.ids)
    assert (got.top[-3:] - last.top).abs().max() < 1e-5
    assert (got.given[0] + math.log(V)).abs() < 1e-4 and got.ids[0].tolist() == [0, 1, 2, 3, 4]


def test_very_many_rows():
    """More rows than a launch has waves: in several launches."""
    from vesta.logprobs import logprobs
    M = (1 << 26) + 7
    x = torch.zeros(M, 2, device='cuda', dtype=torch.float16)
    x[-1, 1] = 3.0
    given = torch.ones(M, dtype=torch.int32, device='cuda')
    got = logprobs(x, given, top=1)
    assert (got.given[:-1] + math.log(2)).abs().max() < 1e-6 and (got.entropy[:-1] - math.log(2)).abs().max() < 1e-6
    assert not got.ids[:-1].any() and got.ids[-1, 0] == 1
    _check(x[-9:], given[-9:], 1)
    assert (got.given[-1] + math.log1p(math.exp(-3))).abs() < 1e-6


def test_empty():
    from vesta.logprobs import logprobs
    got = logprobs(torch.zeros(0, 9, device='cuda'), torch.zeros(0, dtype=torch.int32, device='cuda'), top=2)
    assert got.given.shape == (0,) and got.entropy.shape == (0,) and got.top.shape == (0, 2)
    got = logprobs(torch.zeros(4, 9, device='cuda'), torch.zeros(4, 0, dtype=torch.int64, device='cuda'))
    assert got.given.shape == (4, 0) and got.entropy.shape == (4,)


def test_gradients_refused():
    from vesta.logprobs import logprobs
    x = torch.zeros(2, 9, device='cuda', requires_grad=True)
    with pytest.raises(ValueError, match='gradient'):
        logprobs(x)
    with torch.no_grad():
        logprobs(x)


def test_streams_and_graphs(layout):
    """Two captured calls replay on new contents, eager calls of another stream beside them."""
    from vesta.logprobs import logprobs
    x = torch.randn(3, 5001, device='cuda')
    given = torch.zeros(3, dtype=torch.int32, device='cuda')
    logprobs(x, given, top=4)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = logprobs(x, given, top=4)
        graphs.append((g, got))
    side = torch.cuda.Stream()
    for n in range(4):
        x.normal_()
        given.random_(0, 5001)
        want = logprobs(x, given, top=4)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            eager = logprobs(x, given, top=4)
        torch.cuda.synchronize()
        for got in (eager, *(got for _, got in graphs)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (1, 2, 5, 64, 1000, 4097, 50257))
def test_nans_from_the_first_id(layout, kind, V):
    """NaNs of either sign come first, above +inf, by the lowest id: at id 0, every third, the whole row."""
    from vesta.logprobs import logprobs
    x = torch.randn(7, V, generator=_gen(V, 5), device='cuda').to(DT[kind])
    x[0, 0] = math.nan
    x[1] = math.nan
    x[2, ::3] = math.nan
    x[3, 0] = math.inf
    x[3, V - 1] = math.nan
    x[4] = math.inf
    bits = x[5].view(torch.int32 if kind == 'f32' else torch.int16)
    bits.fill_(-1)                                         # the NaN of all ones
    given = torch.zeros(7, dtype=torch.int64, device='cuda')
    rank = torch.where(x.isnan(), 2.0, torch.where(x == math.inf, 1.0, torch.atan(x.double()) / 2))
    for top in sorted({1, min(V, 3), min(V, 64)}):
        got = logprobs(x, given, top=top)
        assert torch.equal(got.ids.long(), torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :top])
        for t in (got.given, got.entropy, got.top):
            assert t[:6].isnan().all() and t[6].isfinite().all()
        _check(x[6:], given[6:], top)


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (70, 1000, 5000, 50257))
def test_masks_of_a_value(layout, kind, V):
    """Rows whose masked tokens have a finite value: fewer allowed than are asked for, or as many; the rest by id."""
    from vesta.logprobs import logprobs
    gen = _gen(V, 11)
    allowed = (0, 1, 3, 19, 30, 64, 65, 500)
    for value in (-1e4, torch.finfo(DT[kind]).min, 7.0):
        x = torch.full((len(allowed), V), value, device='cuda').to(DT[kind])
        for row, n in zip(x, allowed):
            ids = torch.randperm(V, generator=gen, device='cuda')[:n]
            row[ids] = torch.randn(len(ids), generator=gen, device='cuda').mul_(3).to(row.dtype)
        given = torch.randint(V, (len(x),), generator=gen, device='cuda')
        for top in (1, 2, 5, 20, 64):
            _check(x, given, top)
        x[:, V // 2] = math.nan                            # (the same order behind a NaN)
        order = torch.sort(torch.where(x.isnan(), math.inf, x), dim=1, descending=True, stable=True).indices
        for top in (1, 2, 5, 64):
            assert torch.equal(logprobs(x, given, top=top).ids.long(), order[:, :top])


@pytest.mark.parametrize('kind', DT)
@pytest.mark.parametrize('V', (2048, 50176, 131072))       # (64 parts of 2 loads in fp32: as many as are joined)
def test_large_ones_in_few_places(layout, kind, V):
    """The largest logits where one thread of each wave has them, or two: more than a row's list holds."""
    vec = 4 if kind == 'f32' else 8
    x = torch.randn(4, V, generator=_gen(V, 3), device='cuda')
    load = torch.arange(V, device='cuda') // vec % 64
    x[0, load == 5] += 40
    x[1, load == 63] += 40
    x[2, (load == 0) | (load == 31)] += 40
    x[2, V // 3] = 50
    x[3] = torch.where(load == 9, 40.0, -1e4)
    x = x.to(DT[kind])
    for top in (1, 3, 20, 64):
        _check(x, None, top)


def _us(call):
    """The least of some calls' GPU times."""
    call()
    best = math.inf
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


@pytest.mark.parametrize('M,V,kind,top', [(2000, 50257, 'bf16', 64), (200, 128001, 'bf16', 20), (400, 50257, 'f32', 20)])
def test_reads_of_a_row(M, V, kind, top):
    """Ties, masks of a finite value and NaNs take a few readings of a row, not one for each alternative."""
    from vesta.logprobs import logprobs
    x = torch.randn(M, V, generator=_gen(M), device='cuda').to(DT[kind])
    plain = _us(lambda: logprobs(x, top=top))
    masked = torch.full_like(x, -1e4)
    masked[:, 100:103] = x[:, 100:103]
    flat, nan = torch.zeros_like(x), x.clone()
    nan[:, 5] = math.nan
    for y in (masked, flat, nan):
        assert _us(lambda: logprobs(y, top=top)) < 8 * plain
