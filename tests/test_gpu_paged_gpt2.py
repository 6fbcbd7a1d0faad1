"""GPT-2 over a paged cache (``VestaGPT2.extend``) against the model's own cache: each sequence of a ragged batch, fed in
chunks and single tokens, gives the tokens and logits it gives alone. Logits agree within the bar all engines are held
to (2e-2); a token may differ only where the two largest logits are nearer than twice that."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

L, D, H, V = 3, 192, 3, 509
BAR = 2e-2


@pytest.fixture(scope='module')
def hf():
    if not torch.cuda.is_available():
        pytest.skip('no GPU')
    from vesta.weights import GPT2Shape, RandomGPT2
    return RandomGPT2(GPT2Shape(L, D, H, 4 * D, vocab=V), 5)


@pytest.fixture(scope='module')
def alone(hf):
    from vesta.gpt2 import VestaGPT2
    return VestaGPT2(hf, batch=1, tmax=256, engine='layered')


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


class Server:
    """Sequences in the pages of one cache, fed a chunk each at a time."""

    def __init__(self, model, seqs, pages=64, page=16, room=16, weights=False):
        from vesta.paged import PagedCache
        self.m = model
        self.cache = PagedCache(pages, H, 64, layers=L, page=page, dtype='f16')
        self.page, self.free = page, list(range(pages))
        random.Random(3).shuffle(self.free)
        self.table = torch.full((seqs, room), -1, dtype=torch.int32, device='cuda')
        self.lens = [0] * seqs
        self.seen = [0] * seqs
        self.weight = torch.zeros(L, seqs, H, room * page, device='cuda') if weights else None

    def feed(self, chunks, **kw):
        for b, c in enumerate(chunks):
            for p in range(-(-self.lens[b] // self.page), -(-(self.lens[b] + len(c)) // self.page)):
                self.table[b, p] = self.free.pop()
            self.lens[b] += len(c)
        starts = [0]
        for c in chunks:
            starts.append(starts[-1] + len(c))
        positions = [p for b, c in enumerate(chunks) for p in range(self.seen[b], self.seen[b] + len(c))]
        self.seen = [s + len(c) for s, c in zip(self.seen, chunks)]
        logits, tok = self.m.extend(self.cache, _ints([t for c in chunks for t in c]), _ints(positions), self.table,
                                    _ints(starts), _ints(self.lens), weight=self.weight, **kw)
        return logits.clone(), tok.clone()


def _same(got, tok, want, wtok):
    assert (got - want).abs().max().item() < BAR
    if int(tok) != int(wtok):
        top = want.topk(2).values
        assert (top[0] - top[1]).item() < 2 * BAR


def _prompt(n, seed):
    return torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _alone(m, prompt, steps):
    """The logits and tokens after a prompt and after each of ``steps`` greedy tokens."""
    m.reset()
    m.prefill(_ints([prompt]))
    out = [(m.logits()[0].clone(), int(m.x))]
    for _ in range(steps):
        m.step()
        out.append((m.logits()[0].clone(), int(m.x)))
    return out


@pytest.mark.parametrize('page', (1, 16, 64))
def test_ragged_prompts_and_steps(hf, alone, page):
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=2, tmax=32)               # its own cache is not used: any engine, any batch
    prompts = [_prompt(n, n) for n in (37, 1, 90, 5)]
    want = [_alone(alone, p, 5) for p in prompts]
    s = Server(m, 4, pages=256 if page == 1 else 64, page=page, room=128 // page)
    logits, tok = s.feed(prompts)
    for step in range(6):
        for b in range(4):
            _same(logits[b], tok[b], *want[b][step])
        if step < 5:
            logits, tok = s.feed([[want[b][step][1]] for b in range(4)], most=1)
    m.check()
    s.cache.check()


def test_chunks_mixed_with_steps(hf, alone):
    """A prompt in three chunks while another sequence decodes and a third waits."""
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    a, b, c = _prompt(70, 1), _prompt(9, 2), _prompt(20, 3)
    wa, wb, wc = _alone(alone, a, 1), _alone(alone, b, 3), _alone(alone, c, 1)
    s = Server(m, 3)
    logits, tok = s.feed([[], b, c])
    _same(logits[1], tok[1], *wb[0])
    _same(logits[2], tok[2], *wc[0])
    for i, part in enumerate((a[:33], a[33:50], a[50:])):
        logits, tok = s.feed([part, [wb[i][1]], []])
        _same(logits[1], tok[1], *wb[i + 1])
    _same(logits[0], tok[0], *wa[0])
    logits, tok = s.feed([[wa[0][1]], [], [wc[0][1]]])
    _same(logits[0], tok[0], *wa[1])
    _same(logits[2], tok[2], *wc[1])


def test_many_rows(hf, alone):
    """Enough rows for the tiled products and the LayerNorms of many rows, and more than 64 sequences."""
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    prompts = [_prompt(1 + 7 * i % 61, i) for i in range(66)]
    s = Server(m, 66, pages=400, room=6)
    logits, tok = s.feed(prompts)
    assert sum(map(len, prompts)) >= 1536
    for b in (0, 1, 17, 40, 65):
        _same(logits[b], tok[b], *_alone(alone, prompts[b], 0)[0])


def test_weights_and_eviction(hf, alone):
    """Every token gives each head's positions a weight of 1 in all; a cache evicted to fewer positions answers as the
    model's own cache holding those rows does."""
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    prompts = [_prompt(70, 1), _prompt(25, 2)]
    s = Server(m, 2, weights=True)
    s.feed(prompts)
    for t in range(3):
        s.feed([[7 + t], [11 + t]], most=1)
    total = s.weight.sum(-1)
    # each weight is off by 2^-22 and the rounding of its exponent (scores below 16: 2^-19) of itself at most
    assert (total - torch.tensor([73.0, 28.0], device='cuda')[:, None]).abs().max().item() < 73 * 2.0 ** -18
    to = _ints([[s.free.pop() for _ in range(3)] for _ in range(2)])
    before = [s.cache.keys.clone(), s.cache.vals.clone()]
    lengths, w, kept = s.cache.evict(s.weight, s.table, _ints(s.lens), 40, to, recent=8)
    assert lengths.tolist() == [40, 28] and (kept[:, 0, :, -8:] == torch.arange(65, 73, device='cuda')).all()
    old, s.lens = s.table.clone(), lengths.tolist()
    s.table = torch.cat((to, torch.full((2, 5), -1, dtype=torch.int32, device='cuda')), 1).contiguous()
    s.weight = torch.cat((w, torch.zeros(L, 2, H, 5 * 16, device='cuda')), -1).contiguous()
    logits, tok = s.feed([[5], [6]], most=1)
    for b, n in enumerate((40, 28)):
        alone.reset()
        at = kept[:, b, :, :n].long()                               # [layers, heads, n]
        layer = torch.arange(L, device='cuda')[:, None, None]
        head = torch.arange(H, device='cuda')[None, :, None]
        for own, pool in zip((alone.keys, alone.vals), before):
            rows = pool[layer, old[b].long()[at // 16], at % 16, head]
            own[0, :, :n] = rows.transpose(1, 2)
        alone.seek(n)
        # the model's own position of the token is the row it goes to: learned position n here too
        s2 = Server(m, 1)
        s2.cache, s2.table, s2.lens, s2.seen, s2.free = s.cache, s.table[b:b + 1].contiguous(), [n], [n], s.free
        alone.x.fill_(5 + b)
        alone.step()
        got, gtok = s2.feed([[5 + b]], most=1)
        _same(got[0], gtok[0], alone.logits()[0], int(alone.x))
    s.cache.check()


def test_a_captured_step(hf, alone):
    """A decode step captured in a graph, its inputs advanced on the device between the replays."""
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    prompts = [_prompt(12, 1), _prompt(30, 2)]
    want = [_alone(alone, p, 6) for p in prompts]
    s = Server(m, 2)
    _, tok = s.feed(prompts)
    for b in range(2):
        for p in range(-(-s.lens[b] // 16), 4):
            s.table[b, p] = s.free.pop()
    x, pos, lengths, starts = tok.clone(), _ints(s.lens), _ints(s.lens), _ints([0, 1, 2])

    def step():
        lengths.add_(1)
        logits, tok = m.extend(s.cache, x, pos, s.table, starts, lengths, most=1)
        x.copy_(tok)
        pos.add_(1)
        return logits

    logits = step()                                                 # buffers, and the first step
    for b in range(2):
        _same(logits[b], x[b], *want[b][1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        logits = step()
    for k in range(2, 7):
        g.replay()
        torch.cuda.synchronize()
        for b in range(2):
            if int(x[b]) != want[b][k][1]:
                _same(logits[b], x[b], *want[b][k])
                return                                              # a tie: what follows differs
            _same(logits[b], x[b], *want[b][k])
    m.check()
    s.cache.check()


def test_capture_needs_room(hf, alone):
    """Buffers are made before a capture, and a graph outlives a larger call's."""
    from vesta.gpt2 import VestaGPT2
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    s = Server(m, 2)
    args = (s.cache, _ints([1, 2]), _ints([0, 0]), _ints([[0], [1]]), _ints([0, 1, 2]), _ints([1, 1]))
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='before capturing'):
        with torch.cuda.graph(g):
            m.extend(*args)
    want = [t.clone() for t in m.extend(*args)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = m.extend(*args)
    prompt = _prompt(200, 1)
    big, _ = Server(m, 1, room=16).feed([prompt])
    _same(big[0], 0, _alone(alone, prompt, 0)[0][0], 0)
    for _ in range(3):
        got[0].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        m.extend(*args)


def test_refusals(hf):
    from vesta.gpt2 import VestaGPT2
    from vesta.paged import PagedCache
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    cache = PagedCache(8, H, 64, layers=L, page=16)
    ok = dict(cache=cache, tokens=_ints([1, 2]), positions=_ints([0, 0]), table=_ints([[0], [1]]), starts=_ints([0, 1, 2]),
              lengths=_ints([1, 1]))
    m.extend(**ok)
    for kw, err in ((dict(cache=PagedCache(8, H, 64, layers=L + 1, page=16)), ValueError),
                    (dict(cache=PagedCache(8, H, 64, layers=L, page=16, dtype='bf16')), ValueError),
                    (dict(cache=None), TypeError), (dict(tokens=_ints([1, 2]).long()), TypeError),
                    (dict(tokens=_ints([[1, 2]])), ValueError), (dict(positions=_ints([0])), ValueError),
                    (dict(positions=None), TypeError), (dict(tokens=_ints([]), positions=_ints([])), ValueError),
                    (dict(starts=_ints([0, 2])), ValueError),
                    (dict(weight=torch.zeros(L, 2, H, 8, device='cuda')), ValueError)):
        with pytest.raises(err):
            m.extend(**{**ok, **kw})
    # ids and positions outside their tables are clamped into them, as a prompt's are
    a, _ = m.extend(**{**ok, 'tokens': _ints([V + 5, -3]), 'positions': _ints([99999, -1])})
    a = a.clone()
    b, _ = m.extend(**{**ok, 'tokens': _ints([V - 1, 0]), 'positions': _ints([1023, 0])})
    assert torch.equal(a, b)


def test_positions_and_ids_outside_their_tables(hf):
    """A conversation past the learned positions and an id past the vocabulary are errors; what padded rows hold is not:
    a sequence of length 0 in a batch of fixed size, a row before a sequence's first, rows behind the last sequence."""
    from vesta.gpt2 import VestaGPT2
    from vesta.paged import PagedCache
    m = VestaGPT2(hf, batch=1, tmax=32, engine='layered')
    cache = PagedCache(8, H, 64, layers=L, page=16)
    table = _ints([[0], [1], [2]])
    ok = dict(tokens=[1, 2, 3, 4, 5, 6], positions=[0, 1023, 0, 0, 1, 0])
    batch = (table, _ints([0, 2, 3, 5]), _ints([2, 0, 1]))         # the second is padding, the third's first row too
    rows = (0, 1, 4)

    def call(tokens, positions):
        out, _ = m.extend(cache, _ints(tokens), _ints(positions), *batch)
        return out.clone()

    want = call(**ok)
    cache.check()
    for what, low, high, text in (('positions', 0, 1023, 'position'), ('tokens', 0, V - 1, 'token id')):
        for value in (-1, high + 1, -1 << 31, (1 << 31) - 1):
            for i in range(6):
                a = {**ok, what: list(ok[what])}
                a[what][i] = value
                got = call(**a)
                if i in rows:
                    with pytest.raises(RuntimeError, match=text):
                        cache.check()
                    a[what][i] = low if value < 0 else high
                    assert torch.equal(got[0::2], call(**a)[0::2])
                else:
                    assert torch.equal(got[0::2], want[0::2])
                cache.check()
    m.check()
