"""A key/value cache in pages that holds its rows in 8 bits.

    cache = PagedCache8(pages=512, heads=12, width=64, layers=12, page=64, dtype='f16', form='i8')
    cache.append(k, v, table, starts, lengths, layer)             # new tokens' rows, rounded to what is held
    out = cache.attend(q, table, starts, lengths, layer)          # their attention over all positions
    cache.read(k, v, table, starts, lengths, layer)               # the new tokens' rows as they are held
    cache.check()                                                 # raises if a call met a bad page (syncs)

Batches, pages, streams, errors and refusals are ``vesta.paged.PagedCache``'s, and
``VestaGPT2.extend`` takes either; long decodes, which are bound by the cache's
bytes, read half as many here.

Each 32 values of a row are 8-bit elements and one power of two, the byte layout
of the OCP microscaling formats. A block's power is the least with which its
largest value is below 127.5 ('i8') or 464 ('e4m3') steps of it; values are
rounded to nearest, a tie to even.

* ``form='i8'``: whole numbers of +-127; a value is off by at most 1/127 of its
  block's largest (1/255 where that is just below 127.5/128 of a power of two). A
  block with an infinity or a NaN is held as NaNs.
* ``form='e4m3'``: floats of 4 bits exponent and 3 bits fraction; a value is off by
  at most 1/16 of itself, or by 2^-17.8 of its block's largest where that is more. An
  infinity or NaN is held as a NaN.

This holds within the powers that there are, which are limited such that every
value is one of ``dtype``'s: over 'f16' steps of 2^-24 at least and sizes of 65024
('i8') or 57344 ('e4m3') at most, over 'bf16' steps of 2^-126 and sizes of 127 2^119
(8.4e37) or 448 2^119 (3.0e38); larger values are held as these. So what attention
multiplies is what the cache holds, in 16 bits ('f16': f16 or f32 queries; 'bf16':
bf16), its softmax weights rounded as over a 16-bit cache; under f16 and f32
queries the products of values below 2^-14 are right to 2^-38 absolutely, not
relatively.

No weights are counted and nothing is evicted here.
"""
from __future__ import annotations

from pathlib import Path

from .paged import BLOCK, KINDS, PAGED_SRC, ROWS, SIGNATURES as SIGNATURES16, PagedCache, _collides, _overlap, kernels_of, loaded
from .prefill import MEM_CACHE_BYTES, PRELUDE_SRC

FORM_SRC = Path(__file__).resolve().parent / 'hip' / 'form8.h'
PAGED8_SRC = Path(__file__).resolve().parent / 'hip' / 'paged8.hip'
FORMS = ('i8', 'e4m3')
SCALED = 32                            # values of a power
LEAST = {('i8', 'f16'): 109, ('i8', 'bf16'): 7, ('e4m3', 'f16'): 112, ('e4m3', 'bf16'): 10}    # bytes of the least powers

# Bytes of elements in all layers' pools that a token's pass may read from which pg_attn loads them past the memory-side
# cache, which cannot keep them until the next token's (through it / past it, 8 heads of 128: two of 209 MB 54.1 / 52.2 us,
# one of 426 100.4 / 95.5; what fits is better kept: one of 209 45.1 / 52.0, of 304 63.1 / 67.5, of 333 75.2 / 75.7). The
# bytes are those that the tables have room for: how many positions there are is known on the device only. A table much
# wider than its sequences are long loses what the cache would have kept (45.1 / 52.0).
ATTEND_PAST = MEM_CACHE_BYTES * 5 // 4
# Heads of 128 whose 16-bit rows a wave of append takes together, one position's, where it has a multiple of them: its
# place is found once, by scalar operations (12,900 rows of 8 heads, a head of eight rows / eight heads of one: 17.1 /
# 15.5 us, 28,800: 44.4 / 41.3; in fp32 67.5 / 67.1).
TOGETHER = 8

_ATTENTION = ('pg_attn', 'pg_attn2', 'pg_attn8', 'pg_wide', 'pg_wide8')
# the pools' two parameters are four here, with the powers'
SIGNATURES = {name: SIGNATURES16[name] for name in ('pg_join', 'pg_wide_join', 'pg_take', 'pg_input')}
SIGNATURES.update({name: SIGNATURES16[name][:5] + 'pp' + SIGNATURES16[name][5:] for name in _ATTENTION})
SIGNATURES['pg_attn_past'] = SIGNATURES['pg_attn']
SIGNATURES.update({name: 'ppllll' + 'pppp' + SIGNATURES16['pg_append16'][8:]
                   for name in ('pg_append16', 'pg_append32', 'pg_append16x8', 'pg_read16', 'pg_read32')})

_OWN = {'pg_read16', 'pg_read32', 'pg_attn_past'}              # beside kernels_of's


def paged8_source(width: int, kind: str, form: str) -> str:
    return (f'#define VBLOCK {BLOCK}\n#define PG_E {width}\n#define PG_KIND {KINDS.index(kind)}\n'
            f'#define PG_FORM {1 + FORMS.index(form)}\n'
            + '\n'.join(src.read_text() for src in (PRELUDE_SRC, FORM_SRC, PAGED_SRC, PAGED8_SRC)))


class PagedCache8(PagedCache):
    """As ``PagedCache``, with rows of ``form`` 'i8' or 'e4m3' that stand for
    values of ``dtype``. ``keys`` and ``vals`` are [layers, pages, heads, page,
    width] tensors of elements (int8 or float8_e4m3fn), ``kscales`` and
    ``vscales`` [layers, pages, heads, page, width / 32] bytes: a value is its
    element times 2^(byte - 127), 'i8' elements counting 64ths."""

    def __init__(self, pages, heads, width=64, layers=1, page=64, dtype='f16', form='i8', device=None):
        if form not in FORMS:
            raise ValueError(f'form {form!r}: one of {FORMS}')
        self.form = form
        super().__init__(pages, heads, width, layers, page, dtype, device)

    def _load(self, kind):
        return loaded(self.device.index, (self.width, kind, self.form),
                      lambda: paged8_source(self.width, kind, self.form),
                      {name: SIGNATURES[name] for name in kernels_of(self.width, kind) | _OWN | ({'pg_append16x8'} if self.width == 128 else set())
                       if name in SIGNATURES})

    def _shape(self, pages, heads, width, layers, page, dtype):
        super()._shape(pages, heads, width, layers, page, dtype)
        if self.pages * self.page * self.heads >= 1 << 31:
            raise ValueError(f'{pages} pages of {page} rows of {heads} heads: fewer than 2^31 a layer')

    def _allocate(self, device):
        import torch
        self.device = device
        self.dtype = torch.float16 if self._dt == 'f16' else torch.bfloat16
        shape = (self.layers, self.pages, self.heads, self.page)
        held = torch.int8 if self.form == 'i8' else torch.float8_e4m3fn
        self.keys, self.vals = (torch.zeros(shape + (self.width,), dtype=torch.uint8, device=device).view(held)
                                for _ in range(2))
        self.kscales, self.vscales = (torch.full(shape + (self.width // SCALED,), LEAST[self.form, self._dt],
                                                 dtype=torch.uint8, device=device) for _ in range(2))
        self._ready(self.keys, self.vals, self.kscales, self.vscales)

    def _blocks(self, M, rows, heads):
        """Blocks whose waves take so many of M rows of so many heads each."""
        waves = -(-M // rows) * (self.heads // heads)
        if waves >= 1 << 26:                 # (a launch has fewer than 2^32 threads)
            raise ValueError(f'k: {M} rows are too many for one call')
        return -(-waves // (BLOCK // 64))

    def _appending(self, kn, M, f32):
        heads = TOGETHER if self.width == 128 and not f32 and self.heads % TOGETHER == 0 else 1
        grid = self._blocks(M, 1024 // (self.width * heads), heads)
        return kn.pg_append32 if f32 else kn.pg_append16 if heads == 1 else kn.pg_append16x8, grid

    def _layout(self, kn, B, N, M, G, wide, most):
        attn, *rest = super()._layout(kn, B, N, M, G, wide, most)
        if attn is kn.pg_attn and most * G <= ROWS:              # (each row is read once)
            if 2 * self.layers * min(B * N, self.pages) * self.page * self.heads * self.width > ATTEND_PAST:
                attn = kn.pg_attn_past
        return attn, *rest

    def attend(self, q, table, starts, lengths, layer=0, scale=None, out=None, most=None):
        """As ``PagedCache.attend``, without weights: attention of the new
        tokens' queries ``q`` [M, G * heads, width] over what ``layer`` holds
        of their sequences."""
        return super().attend(q, table, starts, lengths, layer, scale, out, most=most)

    def read(self, k, v, table, starts, lengths, layer=0):
        """What ``layer`` holds of the new tokens' key and value rows (of
        whole sequences, where their starts count all their positions), as
        values into ``k``, ``v`` [M, heads, width]: of the cache's type or f32,
        in either exactly. A row of a position that a sequence does not have (a
        padded row's) becomes 0, rows behind the last sequence stay as they are.
        Returns (k, v)."""
        B, N, seqs = self._batch(table, lengths, starts)
        at = self._layer(layer)
        ks = self._rows('k', k, self._new, self.heads)
        vs = self._rows('v', v, (k.dtype,), like=k.shape)
        size, E, last = 4 if k.dtype is self._f32 else 2, self.width, [0, 0]
        for n, (name, t, (_, row, head)) in enumerate((('k', k, ks), ('v', v, vs))):
            last[n] = (k.shape[0] - 1) * row + (self.heads - 1) * head + E
            # (what most calls are is told by a line: the whole rules take 3 us more)
            if not (head >= E and row >= (self.heads - 1) * head + E) and _collides(t.shape, (row, head)):
                raise ValueError(f'{name}: rows that lie on one another (strides {t.stride()})')
        if ks[0] < vs[0] + size * last[1] and vs[0] < ks[0] + size * last[0] and _overlap(k.shape, size, ks, vs):
            raise ValueError('v: memory other than that of k')
        M = k.shape[0]
        if M == 0 or B == 0:
            return k, v
        kn = self._kind[self.dtype]
        grid = self._blocks(M, 1024 // (E * size), 1)
        stream, back = self._enter()
        try:
            (kn.pg_read32 if size == 4 else kn.pg_read16)(grid, BLOCK, stream, ks[0], vs[0], *ks[1:], *vs[1:], *at, *seqs,
                                                          B, M, self.heads, self._err)
        finally:
            self._leave(back)
        return k, v

    def evict(self, *args, **kwargs):
        raise ValueError('a cache in 8 bits counts no weights and evicts nothing')
