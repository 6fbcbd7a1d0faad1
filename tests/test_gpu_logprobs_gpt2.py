"""GPT-2's log probabilities (``VestaGPT2.logprobs``, ``extend`` with ``given`` and ``top``), over a cache of 16 bits and of 8:
a text scored in ragged chunks and single tokens is what the model's own logits say of it. Logits agree within the bar
all engines are held to (2e-2); a log probability is a difference of two such."""
import pytest
import torch

import held8
from test_gpu_paged_gpt2 import BAR, D, H, L, V, Server, _ints, _prompt, _same, alone, hf  # noqa: F401

pytestmark = pytest.mark.gpu


class Scorer(Server):
    """A server that also hands out the log probabilities."""

    def __init__(self, model, seqs, cache=None, **kw):
        super().__init__(model, seqs, **kw)
        self.cache = cache or self.cache

    def score(self, chunks, given, **kw):
        extend, got = self.m.extend, []

        class Model:
            @staticmethod
            def extend(*a, **k):
                out = extend(*a, given=given, **kw, **k)
                got.append(out[2])
                return out[:2]

        self.m = Model
        try:
            return (*self.feed(chunks), got[0])
        finally:
            self.m = type('M', (), dict(extend=staticmethod(extend)))


def _each(m, text):
    """The model's own logits after each token of a text."""
    m.reset()
    out = []
    for t in text:
        m.x.fill_(t)
        m.step()
        out.append(m.logits()[0].clone())
    return torch.stack(out)


def _check(got, rows, given, top):
    """Results of the rows whose logits are ``rows`` up to BAR."""
    lp = torch.log_softmax(rows.double(), -1)
    assert (got.given.double() - lp.gather(1, given.long())).abs().max().item() < 2 * BAR
    # a weight is off by a factor of e^(2 BAR) at most, the entropy by 2 BAR (of H + log p's mean size)
    H0 = -(lp.exp() * lp).sum(-1)
    assert ((got.entropy.double() - H0).abs() < 2 * BAR * (2 * H0 + 1)).all()
    assert got.top.shape == got.ids.shape == (len(rows), top)
    assert (got.top[:, :-1] >= got.top[:, 1:]).all()
    assert (got.top.double() - lp.gather(1, got.ids.long())).abs().max().item() < 2 * BAR
    assert (lp.topk(top).values - got.top.double()).abs().max().item() < 2 * BAR


def test_a_text_in_chunks(hf, alone):  # noqa: F811
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    texts = [_prompt(90, 4), _prompt(33, 5)]
    rows = [_each(alone, t) for t in texts]
    s = Scorer(m, 2)
    for first, end in ((0, 20), (20, 21), (21, 33)):
        chunks = [t[first:end] for t in texts]
        nexts = [(t + [0])[first + 1:end + 1] for t in texts]
        given = _ints([[n, 7] for c in nexts for n in c])
        logits, tok, got = s.score(chunks, given, top=5)
        want = torch.cat([r[first:end] for r in rows])
        _check(got, want, given, 5)
        for b in range(2):
            _same(logits[b], tok[b], rows[b][end - 1], rows[b][end - 1].argmax())
    logits, tok, got = s.score([texts[0][33:], []], _ints(texts[0][34:] + [1]), top=1)
    _check(got._replace(given=got.given[:, None]), rows[0][33:], _ints(texts[0][34:] + [1])[:, None], 1)
    m.check()
    s.cache.check()


def test_many_rows(hf, alone, monkeypatch):  # noqa: F811
    """More rows than are scored at a time, also few at a time; only alternatives asked for."""
    from vesta import paged
    from vesta.gpt2 import VestaGPT2
    texts = [_prompt(60 + 3 * i, i) for i in range(9)]
    M = sum(map(len, texts))
    assert M > paged.SCORED
    first = None
    for scored in (paged.SCORED, 40, 1000):
        monkeypatch.setattr(paged, 'SCORED', scored)
        s = Scorer(VestaGPT2(hf, batch=1, tmax=32, engine='layered'), 9, pages=80)
        _, _, got = s.score(texts, None, top=3)
        assert got.given is None and got.entropy.shape == (M,)
        if first is None:
            first = got
            i0 = 0
            for b in (0, 1):
                rows = _each(alone, texts[b])
                lp = torch.log_softmax(rows.double(), -1)
                part = slice(i0, i0 + len(texts[b]))
                assert (got.top[part].double() - lp.gather(1, got.ids[part].long())).abs().max().item() < 2 * BAR
                i0 += len(texts[b])
        else:
            assert (got.entropy - first.entropy).abs().max().item() < BAR
            assert (got.top - first.top).abs().max().item() < BAR


def test_the_models_own_steps(hf):  # noqa: F811
    from vesta.gpt2 import VestaGPT2
    for engine in ('persistent', 'layered'):
        m = VestaGPT2(hf, batch=3, tmax=32, engine=engine)
        m.reset()
        m.x.copy_(_ints([5, 6, 7]))
        m.step()
        given = _ints([[1, 2], [3, V], [4, -1]])
        got = m.logprobs(given, top=4)
        lp = torch.log_softmax(m.logits().double(), -1)
        # the same logits: fp32 sums of 509 terms and a logarithm, 2^-24 times some tens
        assert (got.given[:, 0].double() - lp.gather(1, given[:, :1].long())[:, 0]).abs().max().item() < 1e-5
        assert got.given[1:, 1].isnan().all() and got.given[0, 1].isfinite()
        assert torch.equal(got.ids.long(), torch.sort(m.logits(), descending=True, stable=True).indices[:, :4])
        assert torch.equal(got.ids[:, 0], m.x)
        m = VestaGPT2(hf, batch=1, tmax=32, engine=engine)
        m.reset()
        m.prefill(_ints([[5, 6, 7]]))
        got = m.logprobs(top=1)
        assert got.given is None and got.entropy.shape == (1,) and torch.equal(got.ids[0], m.x)


@pytest.mark.parametrize('form', ('i8', 'e4m3'))
def test_over_a_cache_of_8_bits(hf, form):  # noqa: F811
    """Over rows held in 8 bits the model answers as over a 16-bit cache of the values that they stand for."""
    from vesta.gpt2 import VestaGPT2
    from vesta.paged import PagedCache
    from vesta.paged8 import PagedCache8

    class Rounded(PagedCache):
        def append(self, k, v, *a):
            super().append(*(held8.values(*held8.hold(t, form, 'f16'), form).to(t.dtype) for t in (k, v)), *a)

    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    caches = (PagedCache8(64, H, 64, layers=L, page=16, form=form), Rounded(64, H, 64, layers=L, page=16))
    servers = [Scorer(m, 3, cache) for cache in caches]
    texts = [_prompt(n, n) for n in (70, 1, 35)]
    results = [s.score(texts, _ints([t for c in texts for t in c]), top=3) for s in servers]
    for step in range(6):
        (l8, t8, p8), (l16, t16, p16) = results
        for b in range(3):
            _same(l8[b], t8[b], l16[b], t16[b])
        assert (p8.given - p16.given).abs().max().item() < 2 * BAR
        assert (p8.top - p16.top).abs().max().item() < 2 * BAR
        new = t16.tolist()
        results = [s.score([[t] for t in new], _ints(new), top=3, most=1) for s in servers]
    for s in servers:
        s.cache.check()
    m.check()


def test_a_captured_step(hf):  # noqa: F811
    """A decode step over an 8-bit cache with its log probabilities, captured and replayed."""
    from vesta.gpt2 import VestaGPT2
    from vesta.paged8 import PagedCache8
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    cache = PagedCache8(16, H, 64, layers=L, page=16)
    x, pos, given = _ints([1, 2]), _ints([0, 0]), _ints([3, 4])
    batch = (_ints([[0], [1]]), _ints([0, 1, 2]), _ints([1, 1]))

    def step():
        return m.extend(cache, x, pos, *batch, most=1, given=given, top=2)

    g = torch.cuda.CUDAGraph()
    m.extend(cache, x, pos, *batch, most=1)
    with pytest.raises(RuntimeError, match='before capturing'):
        with torch.cuda.graph(g):
            step()
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    Scorer(m, 1, room=16).score([_prompt(200, 1)], None, top=1)      # a larger call's buffers
    for n in range(3):
        x.copy_(_ints([10 + n, 20 + n]))
        given.copy_(_ints([30 + n, 40 + n]))
        want = [t.clone() for part in step() for t in (part if isinstance(part, tuple) else [part])]
        g.replay()
        torch.cuda.synchronize()
        flat = [t for part in got for t in (part if isinstance(part, tuple) else [part])]
        assert all(torch.equal(a, b) for a, b in zip(flat, want))
    m.check()
    cache.check()


def test_refusals(hf):  # noqa: F811
    from vesta.gpt2 import VestaGPT2
    from vesta.paged8 import PagedCache8
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    cache = PagedCache8(8, H, 64, layers=L, page=16)
    ok = dict(cache=cache, tokens=_ints([1, 2]), positions=_ints([0, 0]), table=_ints([[0], [1]]), starts=_ints([0, 1, 2]),
              lengths=_ints([1, 1]))
    assert len(m.extend(**ok)) == 2 and len(m.extend(**ok, given=_ints([1, 2]))) == 3 and len(m.extend(**ok, top=1)) == 3
    for kw, err in ((dict(cache=PagedCache8(8, H, 64, layers=L, page=16, dtype='bf16')), ValueError),
                    (dict(weight=torch.zeros(L, 2, H, 16, device='cuda')), ValueError), (dict(top=V + 1), ValueError),
                    (dict(top=65), ValueError), (dict(given=_ints([1])), ValueError), (dict(given=[1, 2]), TypeError),
                    (dict(given=_ints([1, 2]).float()), TypeError)):
        with pytest.raises(err):
            m.extend(**{**ok, **kw})
    with pytest.raises(ValueError):
        m.logprobs(top=V + 1)
    with pytest.raises(ValueError):
        m.logprobs(_ints([1, 2]))


@pytest.mark.parametrize('scored', (None, 40))
def test_given_of_many_rows(hf, alone, monkeypatch, scored):  # noqa: F811
    """Given tokens of more rows than are scored at a time: the first text's and the last one's, whose rows are scored
    last, against the model's own logits; one a row and two."""
    from vesta import paged
    from vesta.gpt2 import VestaGPT2
    if scored:
        monkeypatch.setattr(paged, 'SCORED', scored)
    texts = [_prompt(60 + 3 * i, i) for i in range(9)]
    M, last = sum(map(len, texts)), len(texts[-1])
    assert M > paged.SCORED and (M % paged.SCORED or M > 2 * paged.SCORED)
    given = _ints([[n, (7 * i + 3) % V] for i, n in enumerate(n for t in texts for n in t[1:] + [0])])
    rows = {0: (slice(0, len(texts[0])), _each(alone, texts[0])), 8: (slice(M - last, M), _each(alone, texts[8]))}
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    for ids in (given, given[:, 0].contiguous().long()):
        _, _, got = Scorer(m, 9, pages=80).score(texts, ids, top=2)
        for part, want in rows.values():
            g = ids.view(M, -1)[part]
            _check(type(got)(*(t[part].view(len(g), -1) if t is got.given else t[part] for t in got)), want, g, 2)
    m.check()
