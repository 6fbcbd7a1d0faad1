"""A key/value cache in pages, for sequences of different lengths, and its operators.

    cache = PagedCache(pages=512, heads=12, width=64, layers=12, page=64, dtype='f16')
    cache.append(k, v, table, starts, lengths, layer)             # new tokens' rows into their pages
    out = cache.attend(q, table, starts, lengths, layer)          # their attention over all positions
    out, w = cache.attend(q, ..., layer, weight=w[layer])         # ... counting the weight each receives
    lengths, w, kept = cache.evict(w, table, lengths, keep, to)   # the positions of least weight go
    cache.check()                                                 # raises if a call met a bad page (syncs)

A batch is B sequences in the same three int32 device tensors throughout:

* ``table`` [B, N]: the pages of each sequence, position s in page
  ``table[b, s // page]``, slot ``s % page``. Entries past a sequence's length
  are not looked at. Which page is whose is the caller's: pages may be shared
  where only read (a common prompt), not where two sequences write.
* ``lengths`` [B]: each sequence's positions, its new tokens included.
* ``starts`` [B + 1]: sequence b's new tokens are rows ``starts[b]`` ..
  ``starts[b + 1] - 1`` of the call's tensors, any number of each, none too.
  Rows behind ``starts[B]`` are left as they are.

New token j of c is at position ``lengths[b] - c + j`` and attends to the
positions up to its own. A token at a negative position (a padded row: length
0 in a batch of fixed size) is not stored, its output is 0.

Everything stays on the device and on torch's current stream, so a call can be
captured in a HIP graph and replayed with other contents of its tensors.
Calls allocate their workspaces from torch's allocator, none is shared between
two calls, which may come from several threads and streams. Tensors are checked
on the host (``TypeError``, ``ValueError``); what lies in ``table``, ``starts``
and ``lengths`` is checked on the device, where an impossible value is replaced
by a possible one and raises an error word that ``check()`` reads: results, a
weight updated in place among them, are then invalid. Nothing is appended for a
sequence whose starts or length are impossible, so the cache's rows stay right.
Nothing here has a backward pass: a tensor whose gradient is being recorded, or
that has a forward-mode tangent, is refused (``ValueError``).

``vesta.paged8.PagedCache8`` is the same with rows held in 8 bits.

The decode cache of ``VestaGPT2`` [B, L, tmax, H, 64] (reference
``vesta/gpt2.py:31-33``) holds one position for all its rows; this one is for
programs whose rows come and go.
"""
from __future__ import annotations

import ctypes
import math
import operator
import struct
import threading
import types
from pathlib import Path

from .launch import compile_code, lib, ok, track, unload
from .prefill import (ARGMAX_SPLIT, BLOCK as PF_BLOCK, FEW_ROWS as MHEAD_ROWS, LNM_ROWS, MODE_GELU, MODE_PLAIN,
                      MODE_QKV, MODE_RESID, PRELUDE_SRC, Prefill, _i, _mtiles, _p)

PAGED_SRC = Path(__file__).resolve().parent / 'hip' / 'paged.hip'
BLOCK = 256
WIDTHS = (64, 128)
KINDS = ('f16', 'bf16', 'f32')         # kernels' queries: the cache's type, or f32 over an f16 cache
PAGE_MAX = 1 << 16
STEP = {64: 64, 128: 32}               # positions of a wave's step in pg_attn, by width
JOIN_BLOCK = 512
JOIN_BLOCKS = 512             # rows of a pg_join block: the fewest of 1, 4 and 16 with so many blocks (512 / 2048: 128
                              # tiles after up to 5000 49 / 62, 512 after up to 4000 163 / 173, 16 the same)

# How a call's work is laid out; us a call (GPU time) on both sides of each rule.
ROWS = 16                     # query rows of a pg_attn block; pg_wide's have 128
FEW_ROWS = 32                 # a sequence of up to so many rows (new tokens times heads of a group) is pg_attn's
# More are pg_wide's, by (width, whether the queries are f32), from so many of its tiles on, or from so many rows a
# sequence where the tables have more than so many positions. pg_attn / pg_wide, width 64, 16 bits: 8 x 64 after 900
# (96 tiles) 16.7 / 24.8, 8 x 128 after 500 20.1 / 17.9, 16 x 128 after 500 (192) 30.7 / 18.6, 1 x 64 after 8000 28.6 /
# 29.0, 1 x 256 56.4 / 31.5; width 128, four heads a group: 1 x 128 (32 tiles) 7.9 / 10.9, 2 x 128 after 500 (64) 20.9 /
# 23.8, 4 x 128 (128) 34.5 / 24.5, 4 x 16 after 900 21.7 / 27.1, 1 x 64 after 2000 29.3 / 27.9, 2 x 16 after 30000 99.8 /
# 56.5; f32, width 64: 16 x 128 after 900 53.7 / 55.3, 24 x 128 76.7 / 75.2, 32 x 768 321 / 178, 1 x 64 after 8000 25.7 /
# 33.5, 1 x 256 63.3 / 48.6; f32, width 128: even at best, so it is not made.
WIDE_FROM = {(64, False): (128, 64, 4096), (128, False): (64, 64, 1536), (64, True): (256, 256, 4096),
             (128, True): (1 << 30, 1 << 30, 0)}
# A tile's positions go to several blocks, and a second launch puts them together, where the tables have more than so
# many positions: SPLIT up to 48 tiles, as many times more as there are tiles up to SPLIT_MOST, from 256 tiles on SPLIT
# for each 256. One token, whole / in parts, sequences of one length: width 64, 12 tiles after 1500 15.0 / 16.5, 2000
# 17.8 / 17.0, 5000 33.7 / 17.0; 64 tiles after 2000 17.2 / 17.3, 3000 23.3 / 21.3; 128 after 3000 24.7 / 30.5, 5000 37.0
# / 39.1; 288 after 2000 36.3 / 40.0, 3000 50.9 / 50.0, 5000 98.5 / 81.0; width 128, 8 tiles after 700 11.9 / 13.7, 1000
# 14.8 / 13.9; 64 after 700 12.2 / 14.0, 2000 26.1 / 22.5; 128 after 2000 27.5 / 33.2, 3000 37.5 / 41.5, 5000 85.6 /
# 70.9; 192 after 3000 54.0 / 60.7, 5000 101 / 105; 512 after up to 900 31.5 / 36.1, up to 4000 142 / 125.
SPLIT, SPLIT_MOST = {64: 2048, 128: 1024}, {64: 5120, 128: 4096}
TARGET = 2048                 # parts in all, about (64 after up to 4000, 1024 / 1536 / 2048 / 4096: 132.2 / 127.4 / 125.5
                              # / 131.1; 2 after 100003: 159.6 / 160.8 / 158.6 / 163.5; in 8 bits, 1024 / 1536 / 2048:
                              # 8 after 30,000 103 / 105 / 98, 2 after 120,001 106 / 100 / 101) ...
PART_STEPS = 8                # ... each of at least so many steps: two a wave
# The same of pg_wide, where it has fewer tiles than fill the chip twice (two blocks a CU are resident).
WIDE_SPLIT, WIDE_TARGET, WIDE_PART_STEPS = 1024, 512, 8
# Width 128, 16 bits, a tile's positions in one block: pg_wide8 (256 rows a block) from so many rows a sequence,
# positions of the tables and tiles of 128 rows on (128 / 256 rows a block: 64 x 32 tokens of four heads after 900, 128
# rows a sequence, 56.9 / 69.8; 4 x 600 34.1 / 38.3; 8 x 128 after 500, 256 tiles, 26.7 / 30.1; 32 x 700 266.8 / 249.6; 16
# x 128 after 900, 512 tiles, 53.8 / 48.4; 2 x 8192 1254 / 1092; 4096 after 27001 2070 / 1810).
TWICE = 256, 768, 512
EIGHT_WAVES = 256             # pg_attn of up to so many tiles (a block a CU) in blocks of eight waves (one token after
                              # 700, four / eight waves: 11.1 / 10.4; 8 x 128, 864 tiles: 13.4 / 19.1) ...
TWO_WAVES = 8                 # ... and of more, where the tables have up to so many steps, of two (f32, four / two waves:
                              # 8 x 128 13.2 / 8.4, 64 tokens after 256 18.6 / 16.0, after 512 24.6 / 24.6; 64 after
                              # 600 of width 128, 19 steps, 22.4 / 23.5)
# Neighbouring blocks that go to one XCD, of pg_attn and of the kernels for many rows (64 x 1 after up to 4000, 16 heads
# of 64, in 4 / 8: 145 / 135; in 1 / 4 / 8 / 16: 4 x 1999 with weights 179 / 181 / 194 / 189, 8 x 128 after 500 21.7 /
# 17.5 / 17.4 / 17.2).
RUN, WIDE_RUN = 8, 4
SCORES_MAX = 1 << 27          # scores (512 MB) that pg_attn keeps for the weights' pass (32 tokens after up to 1000: 24;
                              # made again by pg_weigh: 37)
# Rows of a sequence up to which it does (kept / made again, 12 heads of 64: 8 x 1 after 900 18.6 / 23.4, 8 x 8 26.4 /
# 23.5, 8 x 128 178 / 58, 64 x 8 after 1000 56 / 79; 8 x 4 of 128: 32 x 1 34.3 / 47.0, 64 x 4, 16 rows, 77 / 83, 64 x 8
# 124 / 100).
SCORES_ROWS = 8
# Blocks of the kernels that make scores again, about, by slices of the rows (pg_weigh_wide, 4 x 1999, 512 / 1024 / 1536 /
# 2048 / 4096: 323 / 202 / 196 / 195 / 206; pg_weigh, fp32 of width 128, whole / in slices: 1 x 909 of six heads, two
# keyed, 228 / 51, 8 x 128 of 32/8 65 / 43).
WEIGH_BLOCKS = 2048
SELECT_FEW = 4096             # positions up to which pg_select has 256 threads, not 1024 (1152 times 1024: 13 / 38)
ERRORS = {1: 'a page id outside the pool', 2: 'starts that do not ascend, or lie past the rows',
          4: 'a length past its table', 8: 'a sequence with more new tokens than `most`',
          16: "a position past the model's learned ones", 32: 'a token id outside the vocabulary'}

# parameters of the kernels: p a pointer, l a 64-bit, i a 32-bit whole number, f an fp32
_SEQS = 'iipipp'                       # pages, shift, table, its columns, starts, lengths
SIGNATURES = {
    'pg_append16': 'ppllll' + 'pp' + _SEQS + 'iii' + 'p',
    'pg_append32': 'ppllll' + 'pp' + _SEQS + 'iii' + 'p',
    'pg_attn': 'pll' + 'pp' + _SEQS + 'iiii' + 'iiiiif' + 'pllpp' + 'plp',
    'pg_attn2': 'pll' + 'pp' + _SEQS + 'iiii' + 'iiiiif' + 'pllpp' + 'plp',
    'pg_attn8': 'pll' + 'pp' + _SEQS + 'iiii' + 'iiiiif' + 'pllpp' + 'plp',
    'pg_join': 'ppiiiiiiiiiippllp',
    'pg_wide': 'pll' + 'pp' + _SEQS + 'iiii' + 'iiiiif' + 'pllppp',
    'pg_wide8': 'pll' + 'pp' + _SEQS + 'iiii' + 'iiiiif' + 'pllppp',
    'pg_wide_join': 'ppiiiiiiiiiippllp',
    'pg_weigh': 'pll' + 'p' + _SEQS + 'iiii' + 'fppipiiiip',
    'pg_given': 'plppiiiippipii',
    'pg_weigh_wide': 'pll' + 'p' + _SEQS + 'iiii' + 'fppipiiiip',
    'pg_total': 'pippiiiipipii',
    'pg_select': 'pipiiiiippipp',
    'pg_move': 'ppiipipipiiiip',
    'pg_take': 'pp',
    'pg_input': 'pppiiippiiippp',
}


def kernels_of(width: int, kind: str) -> set:
    """The kernels of a module: those of many rows are not made for f32 queries of width 128."""
    without = set() if (width, kind) in ((128, 'f16'), (128, 'bf16')) else {'pg_wide8'}
    if (width, kind) == (128, 'f32'):
        without |= {'pg_weigh_wide', 'pg_wide', 'pg_wide_join'}
    return set(SIGNATURES) - without


_CODES = {'p': 'P', 'l': 'q', 'i': 'i', 'f': 'f'}


def paged_source(width: int, kind: str) -> str:
    return (f'#define VBLOCK {BLOCK}\n#define PG_E {width}\n#define PG_KIND {KINDS.index(kind)}\n'
            + PRELUDE_SRC.read_text() + '\n' + PAGED_SRC.read_text())


class _Launcher:
    """One kernel with a buffer for its arguments: filled and read by one call
    at a time."""

    def __init__(self, fn, name, signature):
        self.fn, self.name = fn, name
        self.lock = threading.Lock()
        codes = '@' + ''.join(_CODES[c] for c in signature)
        self.pack = struct.Struct(codes)
        self.buf = ctypes.create_string_buffer(self.pack.size)
        base = ctypes.addressof(self.buf)
        offs = [struct.calcsize(codes[:k + 1]) - struct.calcsize(codes[k]) for k in range(1, len(codes))]
        self.args = (ctypes.c_void_p * len(offs))(*[base + o for o in offs])
        self.launch = lib().vh_launch

    def __call__(self, grid, block, stream, *vals):
        with self.lock:
            self.pack.pack_into(self.buf, 0, *vals)
            status = self.launch(self.fn, grid, block, 0, stream, self.args)
        if status:
            ok(status, self.name)


class _Kernels:
    """A module's kernels, those of ``signatures``, loaded on one device."""

    def __init__(self, device, source, signatures):
        import torch
        self.mod = ctypes.c_void_p()
        with torch.cuda.device(device):
            ok(lib().vh_module_load(compile_code(source), ctypes.byref(self.mod)), 'module load')
            track(self)
            for name, signature in signatures.items():
                fn = ctypes.c_void_p()
                ok(lib().vh_module_get_function(self.mod, name.encode(), ctypes.byref(fn)), name)
                setattr(self, name, _Launcher(fn, name, signature))

    def close(self):
        if self.mod is not None and self.mod.value:
            mod, self.mod = self.mod, None
            unload(mod)


_ANY2 = (None, None)
_loaded = {}
_loaded_lock = threading.Lock()


def loaded(device, key, source, signatures):
    """The kernels known as ``key`` on a device, loaded where they are first asked for."""
    with _loaded_lock:
        if (device, key) not in _loaded:
            _loaded[device, key] = _Kernels(device, source(), signatures)
        return _loaded[device, key]


def _at(t):
    """A tensor's address, 0 for none."""
    return 0 if t is None else t.data_ptr()


def _grid2(shape, strides):
    """(size, stride) of a [rows, heads, width] tensor's two outer axes, the one of shorter stride first; an axis of one
    has no stride."""
    return sorted(((n, s if n > 1 else 0) for n, s in zip(shape[:2], strides)), key=lambda a: a[1])


def _collides(shape, strides):
    """Whether rows of a [rows, heads, width] tensor may lie on one another."""
    (n0, s0), (n1, s1) = _grid2(shape, strides)
    return n0 > 1 and s0 < shape[2] or n1 > 1 and s1 < (n0 - 1) * s0 + shape[2]


def _overlap(shape, size, a, b):
    """Whether two tensors of one shape and item size, (address, row stride, head stride) each, may share memory. They do
    not where one ends before the other, or where they are parts of one row (one head of heads-first rows), as the
    queries of a fused projection and its other columns, or of one head's."""
    ga, gb = _grid2(shape, a[1:]), _grid2(shape, b[1:])
    last = [sum((n - 1) * s for n, s in g) + shape[2] for g in (ga, gb)]
    apart = (b[0] - a[0]) // size
    if apart >= last[0] or -apart >= last[1] or not shape[0]:
        return False
    (inner, outer), E = (s for _, s in ga), shape[2]

    def between(pitch, fa, fb):          # what a and b cover of each `pitch`: fa from 0 on, fb from where b begins
        return fa <= apart % pitch <= pitch - fb
    if outer and gb[1][1] == outer and between(outer, *((g[0][0] - 1) * g[0][1] + E for g in (ga, gb))):
        return False
    return not (inner and ga == gb and outer % inner == 0 and between(inner, E, E))


def _dealt(n, run):
    """Blocks of a grid whose kernel deals n tasks to the device's eight XCDs in runs."""
    return 8 * run * -(-n // (8 * run))


class PagedCache:
    """``pages`` pages of ``page`` rows (a power of two) in each of ``layers``
    layers, for ``heads`` key heads of ``width`` 64 or 128. ``keys`` and
    ``vals`` are [layers, pages, page, heads, width] tensors of ``dtype``
    ('f16' or 'bf16'), zeroed."""

    def __init__(self, pages, heads, width=64, layers=1, page=64, dtype='f16', device=None):
        """``device``: a CUDA device or its index, the current one by default."""
        self._shape(pages, heads, width, layers, page, dtype)
        import torch
        if not torch.cuda.is_available():
            raise RuntimeError('no GPU: the paged cache needs a ROCm device')
        device = torch.device('cuda', device) if isinstance(device, int) else torch.device(device or 'cuda')
        if device.type != 'cuda':
            raise ValueError(f'device {device}: a CUDA device')
        self._allocate(torch.device('cuda', torch.cuda.current_device() if device.index is None else device.index))
        # torch.cuda's own, without the stream object around the handle
        self._current = torch._C._cuda_getDevice
        self._raw_stream = torch._C._cuda_getCurrentRawStream
        self._kind = {self.dtype: self._load(dtype)}
        if dtype == 'f16':
            self._kind[torch.float32] = self._load('f32')

    def _load(self, kind):
        return loaded(self.device.index, (self.width, kind), lambda: paged_source(self.width, kind),
                      {name: SIGNATURES[name] for name in kernels_of(self.width, kind)})

    def _shape(self, pages, heads, width, layers, page, dtype):
        pages, heads, width, layers, page = map(operator.index, (pages, heads, width, layers, page))
        if dtype not in ('f16', 'bf16'):
            raise ValueError(f"dtype {dtype!r}: the cache is 'f16' or 'bf16'")
        if width not in WIDTHS:
            raise ValueError(f'heads of {width}: their width is one of {WIDTHS}')
        if not (1 <= page <= PAGE_MAX and page & (page - 1) == 0):
            raise ValueError(f'pages of {page} rows: a power of two up to {PAGE_MAX}')
        if min(pages, heads, layers) < 1:
            raise ValueError(f'{pages} pages, {heads} heads, {layers} layers: one at least of each')
        if heads * width >= 1 << 31:
            raise ValueError(f'{heads} heads of {width}: rows of fewer than 2^31 values')
        if pages * page >= 1 << 31:
            raise ValueError(f'{pages} pages of {page} rows: fewer than 2^31 rows a layer')
        self.pages, self.heads, self.width, self.layers, self.page = pages, heads, width, layers, page
        self._shift = page.bit_length() - 1
        self._scale = 1.0 / math.sqrt(width)
        self._dt = dtype

    def _allocate(self, device):
        import torch
        self.device = device
        self.dtype = torch.float16 if self._dt == 'f16' else torch.bfloat16
        shape = (self.layers, self.pages, self.page, self.heads, self.width)
        self.keys = torch.zeros(shape, dtype=self.dtype, device=self.device)
        self.vals = torch.zeros(shape, dtype=self.dtype, device=self.device)
        self._ready(self.keys, self.vals)

    def _ready(self, *pools):
        """What every call needs (a call's checks cost about as much as its launch)."""
        import torch
        self._pools = [tuple(p[n].data_ptr() for p in pools) for n in range(self.layers)]      # each layer's
        self._index = self.keys.get_device()
        self._i32, self._f32, self._empty = torch.int32, torch.float32, torch.empty
        self._recording, self._forward = torch.is_grad_enabled, torch.autograd.forward_ad
        self._new = self.dtype, self._f32                          # types of new rows, and of queries
        self._queries = self._new if self._dt == 'f16' else (self.dtype,)
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._err = self.err.data_ptr()

    # ------------------------------------------------------------ checks
    def _ints(self, name, t, shape):
        try:
            fits = t.dtype is self._i32 and t.get_device() == self._index and t.is_contiguous()
            got = t.shape
        except AttributeError:
            fits = False
        if not fits:
            raise TypeError(f'{name}: need a contiguous int32 tensor on {self.device}')
        if got != shape and (shape[-1] is not None or len(got) != 2 or shape[0] not in (None, got[0])):
            raise ValueError(f'{name}: shape {tuple(got)}, need {tuple("any" if w is None else w for w in shape)}')
        return t.data_ptr()

    def _batch(self, table, lengths, starts=None, new=True):
        """B, N and the kernels' arguments for a batch (``new``: of new tokens, whose ``starts`` they need)."""
        at = self._ints('table', table, _ANY2)
        B, N = table.shape
        self._few('table', N)
        return B, N, (self.pages, self._shift, at, N, self._ints('starts', starts, (B + 1,)) if new else 0,
                      self._ints('lengths', lengths, (B,)))

    def _few(self, name, n):
        if n * self.page >= 1 << 31:
            raise ValueError(f'{name}: {n} pages of {self.page} rows a sequence, fewer than 2^31 rows are possible')

    def _rows(self, name, t, dtypes, heads=None, like=None):
        """New tokens' rows [M, heads, width]: any strides but the last, 16-byte aligned. Returns their address and
        strides."""
        try:
            fits = t.dtype in dtypes and t.get_device() == self._index
            shape = t.shape
        except AttributeError:
            fits = False
        if not fits:
            raise TypeError(f'{name}: need a tensor of {" or ".join(str(d)[6:] for d in dtypes)} on {self.device}')
        if len(shape) != 3 or shape[2] != self.width or (heads is not None and shape[1] != heads) \
                or (like is not None and shape != like):
            raise ValueError(f'{name}: shape {tuple(shape)}, need '
                             f'{tuple(like) if like is not None else ("rows", heads or "heads", self.width)}')
        if t.requires_grad and self._recording():
            self._no_gradient(name)
        if self._forward._current_level >= 0 and self._forward.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name}: no tangent is made of it; detach it')
        row, head, one = t.stride()
        at = t.data_ptr()
        if (one != 1 or (row | head) & (3 if t.dtype is self._f32 else 7) or at & 15) and t.numel():
            raise ValueError(f'{name}: rows of consecutive, 16-byte aligned values needed (strides {t.stride()})')
        return at, row, head

    @staticmethod
    def _no_gradient(name):
        raise ValueError(f'{name}: no gradient is made of it; detach it, or call under torch.no_grad()')

    def _layer(self, layer):
        layer = operator.index(layer)
        if not 0 <= layer < self.layers:
            raise ValueError(f'layer {layer} of {self.layers}')
        return self._pools[layer]

    def _enter(self):
        """The stream to launch on, with the cache's device the current one; and the device to go back to, or None."""
        if self._current() == self._index:
            return self._raw_stream(self._index), None
        import torch
        back = torch.cuda.current_device()
        torch.cuda.set_device(self._index)
        return self._raw_stream(self._index), back

    @staticmethod
    def _leave(back):
        if back is not None:
            import torch
            torch.cuda.set_device(back)

    def _appending(self, kn, M, f32):
        """The kernel that appends M rows and its blocks, of eight values a thread."""
        grid = -(-M * self.heads * (self.width // 8) // BLOCK)
        if grid >= 1 << 31:
            raise ValueError(f'k: {M} rows are too many for one call')
        return kn.pg_append32 if f32 else kn.pg_append16, grid

    # ------------------------------------------------------------ operators
    def append(self, k, v, table, starts, lengths, layer=0):
        """The new tokens' key and value rows ``k``, ``v`` [M, heads, width]
        into their pages of ``layer``. They are of the cache's type or f32
        (rounded to nearest). Rows of other sequences' slots stay as they are;
        a page that two of the new rows' sequences share gets either's."""
        B, N, seqs = self._batch(table, lengths, starts)
        at = self._layer(layer)
        k_at, *ks = self._rows('k', k, self._new, self.heads)
        v_at, *vs = self._rows('v', v, (k.dtype,), like=k.shape)
        M = k.shape[0]
        if M == 0 or B == 0 or N == 0:
            return
        launch, grid = self._appending(self._kind[self.dtype], M, k.dtype is self._f32)
        stream, back = self._enter()
        try:
            launch(grid, BLOCK, stream, k_at, v_at, *ks, *vs, *at, *seqs, B, M, self.heads, self._err)
        finally:
            self._leave(back)

    def attend(self, q, table, starts, lengths, layer=0, scale=None, out=None, weight=None, weight_out=None, most=None):
        """Attention of the new tokens' queries ``q`` [M, G * heads, width]
        (query heads G h .. G h + G - 1 read key head h) over their sequences'
        positions in ``layer``: softmax(``scale`` q . k), 1 / sqrt(width) by
        default, times the values. ``q`` is of the cache's type or, over an f16
        cache, f32; the result is of q's type: ``out`` [M, G * heads, width],
        made if not given (its memory none of q's, its rows apart from one
        another). A token that sees no position gets zeros.

        ``weight`` [B, heads, S] (f32, contiguous, S at least the table's
        positions): the softmax weight that each position has received so far.
        Then the call returns (out, weight_out), where weight_out [B, heads, S'] is
        weight plus what the new tokens give, over the query heads of the key
        head; the new positions start at 0, and past the lengths it is 0.
        ``weight_out`` may be given (memory of its own), ``weight`` itself is
        updated if it is not.

        ``most``: a bound of the new tokens of a sequence that the program
        knows (1 for a decode step); the work is laid out by it."""
        B, N, seqs = self._batch(table, lengths, starts)
        at = self._layer(layer)
        qs = self._rows('q', q, self._queries)
        M, Hq, _ = q.shape
        G, odd = divmod(Hq, self.heads)
        if Hq == 0 or odd:
            raise ValueError(f'q: {Hq} heads are not a multiple of the {self.heads} key heads')
        scale2 = 1.4426950408889634 * (self._scale if scale is None else float(scale))
        if not 2.0 ** -126 <= scale2 < 2.0 ** 127:
            raise ValueError(f'scale {scale}: positive and finite in 32 bits')
        if most is not None and (most := operator.index(most)) < 1:
            raise ValueError(f'most {most}: at least 1')
        if out is None:
            out = q.new_empty((M, Hq, self.width))
            to = out.data_ptr(), Hq * self.width, self.width
        else:
            to = self._rows('out', out, (q.dtype,), like=q.shape)
            q_at, q_row, q_head = qs
            o_at, o_row, o_head = to
            E, size = self.width, 4 if q.dtype is self._f32 else 2
            # (what most calls are is told by a line each: the whole rules take 3 us more)
            if not (o_head >= E and o_row >= (Hq - 1) * o_head + E) and _collides(q.shape, (o_row, o_head)):
                raise ValueError(f'out: rows that lie on one another (strides {out.stride()})')
            if q_at < o_at + size * ((M - 1) * o_row + (Hq - 1) * o_head + E) \
                    and o_at < q_at + size * ((M - 1) * q_row + (Hq - 1) * q_head + E) \
                    and _overlap(q.shape, size, qs, to):
                raise ValueError('out: memory other than that of q (which a second pass may read again)')
        S = So = 0
        if weight is not None:
            weight_out = weight if weight_out is None else weight_out
            S, So = (self._weights(n, w, (B, self.heads), N * self.page)
                     for n, w in (('weight', weight), ('weight_out', weight_out)))
            if weight_out is not weight and self._shared(weight, weight_out) and (
                    weight_out.data_ptr() != weight.data_ptr() or So != S and B * self.heads > 1):
                raise ValueError('weight_out: weight itself or other memory')
        elif weight_out is not None:
            raise ValueError('weight_out: no weight given')
        most = M if most is None else min(most, M)
        kn = self._kind[q.dtype]
        stream, back = self._enter()
        try:
            f32 = q.dtype is self._f32
            wide = self._wide(B, N, M, G, most, f32)
            lse = scores = pitch = target = 0
            floats = 0                   # of the one workspace: lse, scores, parts
            if weight is not None:
                pitch = -(-N * self.page // 64) * 64
                floats = -(-M * Hq // 4) * 4
                if not wide and most * G <= SCORES_ROWS and 0 < M * Hq * pitch <= SCORES_MAX:
                    scores = 4 * floats
                    floats += M * Hq * pitch
            if M and B:
                attn, block, rows, tiles, target, blocks, least, run = self._layout(kn, B, N, M, G, wide, most)
                ws = 4 * floats
                floats += blocks * rows * (self.width + 2) if target else 0
            if floats:
                held = self._floats(floats)
                base = held.data_ptr()
                lse = base if weight is not None else 0
                scores = scores and base + scores
            if M and B:
                to = (*to, lse)
                args = (_dealt(blocks, run), block, stream, *qs, *at, *seqs, B, M, self.heads, G, target, least, run,
                        blocks, most, scale2, *to, base + ws if target else 0)
                if wide:
                    attn(*args, self._err)
                else:
                    attn(*args, scores, pitch, self._err)
                if target:
                    cut = next((c for c in (1, 4) if tiles * rows // c <= JOIN_BLOCKS), 16)
                    (kn.pg_wide_join if wide else kn.pg_join)(
                        tiles * (rows // cut), JOIN_BLOCK, stream, *seqs[4:], B, N * self.page, M, self.heads, G, target,
                        least, run, blocks, cut, base + ws, *to)
            if weight is not None and B and So:
                self._receive(kn, stream, (*qs, at[0]), seqs, (B, M, G), most, wide, scale2, lse, scores,
                              pitch, (weight.data_ptr(), S, weight_out.data_ptr(), So))
        finally:
            self._leave(back)
        return out if weight is None else (out, weight_out)

    def _wide(self, B, N, M, G, most, f32):
        """Whether blocks of 128 rows make the call's (``WIDE_FROM``)."""
        tiles, rows, positions = WIDE_FROM[self.width, f32]
        return most * G > FEW_ROWS and (self.heads * max(B, M * G // 128) >= tiles
                                        or most * G >= rows and N * self.page > positions)

    def _layout(self, kn, B, N, M, G, wide, most):
        """The kernel and threads of a block, its rows, the tiles of so many rows there can be, the parts asked for (0:
        one a tile) and those there can be, the least steps of one, the blocks to an XCD in turn."""
        positions = N * self.page
        if wide:
            rows, aim, most_tiles, least, split = 128, WIDE_TARGET, 2 * WIDE_TARGET, WIDE_PART_STEPS, WIDE_SPLIT
        else:
            rows, aim, most_tiles, least, split = ROWS, TARGET, 16 * TARGET, PART_STEPS, SPLIT[self.width]
        tiles = self.heads * (B if most * G <= rows else M * G // rows + B)
        if tiles > 256:
            split = split * tiles // 256
        elif not wide:
            split = max(split, min(split * tiles // 48, SPLIT_MOST[self.width]))
        target = aim if tiles < most_tiles and positions > split else 0
        blocks = target + tiles + 64
        if blocks >= 1 << 28 or M * G >= 1 << 30:
            raise ValueError(f'q: {M} rows of {B} sequences are too many for one call')
        run = WIDE_RUN if wide else RUN
        if wide:
            attn, block = kn.pg_wide, BLOCK
            if self.width == 128 and target == 0 and all(n >= m for n, m in zip((most * G, positions, tiles), TWICE)):
                attn, block, rows = kn.pg_wide8, 2 * BLOCK, 256
                tiles = self.heads * (M * G // rows + B)
                blocks = tiles + 64
        elif target:
            attn, block = kn.pg_attn, BLOCK
        elif tiles <= EIGHT_WAVES:
            attn, block = kn.pg_attn8, 2 * BLOCK
        elif positions <= TWO_WAVES * STEP[self.width]:
            attn, block = kn.pg_attn2, BLOCK // 2
        else:
            attn, block = kn.pg_attn, BLOCK
        return attn, block, rows, tiles, target, blocks, least, run

    def _floats(self, n):
        """A workspace of a call."""
        return self._empty(n, dtype=self._f32, device=self.device)

    def _receive(self, kn, stream, keys, seqs, extents, most, wide, scale2, lse, scores, pitch, to):
        """The weights' pass after ``attend``'s: from the scores it left, or making them again."""
        B, M, G = extents
        bh, So, cap = B * self.heads, to[-1], seqs[3] * self.page
        if scores:
            blocks = -(-So // 1024)
            kn.pg_given(bh * blocks, BLOCK, stream, scores, pitch, *seqs[4:], cap, M, self.heads, G, lse, *to, blocks)
            return
        weigh, width, run = (kn.pg_weigh_wide, 256, WIDE_RUN) if wide else (kn.pg_weigh, 128, RUN)
        blocks = -(-So // width)
        slices = max(1, min(WEIGH_BLOCKS // (bh * blocks), most * G // width))
        part = None if slices == 1 else self._floats(slices * bh * So)
        weigh(_dealt(bh * blocks * slices, run), BLOCK, stream, *keys, *seqs, B, M, self.heads, G, scale2, lse, *to, blocks,
              run, slices, _at(part))
        if slices > 1:
            blocks = -(-So // 256)
            kn.pg_total(bh * blocks, BLOCK, stream, part.data_ptr(), slices, *seqs[4:], cap, B, M, self.heads, *to, blocks)

    def _weights(self, name, w, lead, least):
        try:
            fits = w.dtype is self._f32 and w.get_device() == self._index and w.is_contiguous()
            shape = w.shape
        except AttributeError:
            fits = False
        if not fits:
            raise TypeError(f'{name}: need a contiguous float32 tensor on {self.device}')
        if w.requires_grad and self._recording():
            self._no_gradient(name)
        if self._forward._current_level >= 0 and self._forward.unpack_dual(w).tangent is not None:
            raise ValueError(f'{name}: no tangent is made of it; detach it')
        if tuple(shape[:-1]) != lead or not least <= shape[-1] < 1 << 31:
            raise ValueError(f'{name}: shape {tuple(shape)}, need {lead} and {least} positions at least')
        return shape[-1]

    @staticmethod
    def _shared(a, b):
        """Whether two contiguous tensors of 4-byte items share memory."""
        at, to = a.data_ptr(), b.data_ptr()
        return at < to + 4 * b.numel() and to < at + 4 * a.numel()

    def evict(self, weight, table, lengths, keep, to, recent=0, weight_out=None):
        """Keep ``keep`` positions of each sequence (all where it has no more):
        its ``recent`` last ones and, of the others, those of largest
        ``weight`` [layers, B, heads, S] (f32, contiguous; a tie goes to the
        lowest position, NaN counts as the largest), chosen for each layer and
        head on its own. They go, in their order, into the pages ``to`` [B, N']
        (int32, N' pages of at least ``keep`` rows in all), which must be none
        of the pages that the call reads; ``table``'s pages stay as they are,
        for their owner to hand out again.

        Returns (lengths [B], weight_out [layers, B, heads, S'], kept [layers,
        B, heads, keep]): the new lengths, the kept positions' weights (0
        behind them) and which positions they were (-1 behind them)."""
        B, N, seqs = self._batch(table, lengths, new=False)
        to_at = self._ints('to', to, (B, None))
        No = to.shape[1]
        if to_at == seqs[2] and B and N:
            raise ValueError('to: pages other than those that are read')
        self._few('to', No)
        keep, recent = operator.index(keep), operator.index(recent)
        if keep < 1 or recent < 0:
            raise ValueError(f'keep {keep} of at least 1 position, recent {recent} of at least 0')
        if No * self.page < keep:
            raise ValueError(f'to: {No} pages of {self.page} rows cannot hold {keep} positions')
        lead = (self.layers, B, self.heads)
        S = self._weights('weight', weight, lead, N * self.page)
        if weight_out is None:
            weight_out = self._empty(lead + (No * self.page,), dtype=self._f32, device=self.device)
        So = self._weights('weight_out', weight_out, lead, No * self.page)
        if self._shared(weight, weight_out):
            raise ValueError('weight_out: memory other than that of weight')
        kept = self._empty(lead + (keep,), dtype=self._i32, device=self.device)
        new = self._empty(B, dtype=self._i32, device=self.device)
        if B == 0:
            return new, weight_out, kept
        kn = self._kind[self.dtype]
        blocks = -(-keep * self.heads * (self.width // 8) // BLOCK)
        if self.layers * B * max(blocks, self.heads) >= 1 << 31:
            raise ValueError(f'{self.layers} layers of {B} sequences are too many for one call')
        stream, back = self._enter()
        try:
            kn.pg_select(self.layers * B * self.heads, 256 if N * self.page <= SELECT_FEW else 1024, stream,
                         weight.data_ptr(), S, seqs[5], N * self.page, B, self.heads, keep, min(recent, keep),
                         kept.data_ptr(), weight_out.data_ptr(), So, new.data_ptr(), self._err)
            kn.pg_move(self.layers * B * blocks, BLOCK, stream, *self._pools[0], *seqs[:4], to_at, No, kept.data_ptr(), keep,
                       B, self.heads, blocks, self._err)
        finally:
            self._leave(back)
        return new, weight_out, kept

    def _wait(self):
        """For all the device's streams."""
        import torch
        torch.cuda.synchronize(self.device)

    def check(self):
        """Raise if an earlier call, on any stream, met a page, a length or
        starts that cannot be (waits for the device); the word is cleared in
        the same step, so that none raised meanwhile is lost. Not while a
        graph is captured."""
        self._wait()
        took = self._empty(1, dtype=self._i32, device=self.device)
        stream, back = self._enter()
        try:
            self._kind[self.dtype].pg_take(1, 64, stream, self._err, took.data_ptr())
        finally:
            self._leave(back)
        word = int(took.item())
        if word:
            why = ', '.join(text for bit, text in ERRORS.items() if word & bit)
            raise RuntimeError(f'paged cache: {why}; the results are invalid')


PLANS = 8                              # row counts whose launches a PagedPass keeps recorded
SCORED = 512                           # rows whose logits it makes at a time where all rows' log probabilities are asked
                                       # for: 103 MB of GPT-2's, which stay in the memory-side cache (24,576 rows, 256 /
                                       # 512 / 1024 / 4096 at a time: 7.8 / 6.7 / 7.1 / 6.9 ms)


class PagedPass(Prefill):
    """One pass of a GPT-2 over ragged new tokens and a paged cache
    (``VestaGPT2.extend``): the layered engine's products and LayerNorms
    (``base``, whose module and packed weights are used), with the cache's
    ``append`` and ``attend`` in the place of its attention. The qkv product
    writes its key and value rows where ``append`` takes them from: to a
    product's epilogue the staging rows are M caches of one position.
    Activation buffers grow to the largest call and are kept."""

    def __init__(self, model, base):
        import torch
        self.base, self.fn, self._own, self.err = base, base.fn, base._own, base.err
        self.layers = model.L
        self.m = types.SimpleNamespace(W=model.W, D=model.D, H=model.H, L=1, tmax=1, keys=None, vals=None,
                                       weight_bytes=model.weight_bytes,
                                       t=torch.zeros(1, dtype=torch.int32, device=self.err.device))
        self._ws, self._ws_at, self._graph, self._plan, self.mod = None, ctypes.c_void_p(), None, [], None
        self._held, self._buf, self._plans = (0, 0), None, {}
        self._scores, self._score_plans = None, {}
        self._outgrown = []              # buffers that a captured graph may hold

    def _room(self, M, B):
        """Buffers for M rows of B sequences (rows past M reach discarded outputs only)."""
        import torch
        if M <= self._held[0] and B <= self._held[1]:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f'extend: call once with at least {M} tokens of {B} sequences before capturing such a call')
        # (doubled at least, so that all that were outgrown are no more than the present ones)
        M, B = self._held = tuple(h if n <= h else 1 << (n - 1).bit_length() for n, h in zip((M, B), self._held))
        self._outgrown.append(self._buf)
        m, dev = self.m, self.err.device
        F, V = m.W['fcw'].shape[2], m.W['wte'].shape[0]
        f32, f16, i32 = (dict(dtype=t, device=dev) for t in (torch.float32, torch.float16, torch.int32))
        rows, last = 16 * _mtiles(M), 16 * _mtiles(B)
        self._buf = types.SimpleNamespace(
            tok=torch.zeros(M, **i32), wpe=torch.empty(M, m.D, **f16), Z=torch.empty(M, m.D, **f32),
            Q=torch.empty(M, m.D, **f32), O=torch.zeros(M, m.D, **f32), K=torch.empty(M, m.D, **f16),
            V=torch.empty(M, m.D, **f16), AF=torch.zeros(2 * rows * m.D, **f16), GF=torch.zeros(2 * rows * F, **f16),
            ZL=torch.empty(B, m.D, **f32), CF=torch.zeros(2 * last * m.D, **f16), logit=torch.empty(B, V, **f32),
            x=torch.zeros(B, **i32), next=torch.zeros(B, **f32), apv=torch.empty(B * ARGMAX_SPLIT, **f32),
            api=torch.empty(B * ARGMAX_SPLIT, **i32))
        self._plans, self._score_plans = {}, {}

    def _workspace(self, n):
        if self._ws is None or self._ws.numel() < n:
            self._outgrown.append(self._ws)
            n = 1 << (n - 1).bit_length()
        return super()._workspace(n)

    def _record(self, build):
        self._plan = []
        build()
        plan, self._plan = self._plan, []
        return plan

    def _norm(self, X, w, b, to, rows):
        D, mt = self.m.D, _mtiles(rows)
        if rows >= LNM_ROWS:
            self._launch('pf_lnm8' if D <= 1024 else 'pf_lnm16', -(-rows // 16),
                         [_p(X), _i(rows), _i(D), _p(w), _p(b), _p(to), _i(mt), _p(self.err)])
        else:
            self._launch('pf_ln', rows, [_p(X), _i(0), _i(1), _p(w), _p(b), _i(D), _p(to), _i(mt), _p(self.err)])

    def _launches(self, M, B):
        """The recorded launches of a pass of M rows: embedding; each layer's qkv product; each layer's rest; head."""
        key = (M, B)
        if key in self._plans:
            return self._plans[key]
        while len(self._plans) >= PLANS:
            del self._plans[next(iter(self._plans))]
        m, b, W, err = self.m, self._buf, self.m.W, self.err
        D, F, V, mt = m.D, W['fcw'].shape[2], W['wte'].shape[0], _mtiles(M)

        def embed():                     # (the positions' rows are gathered: row m's is row m)
            self._launch('pf_embed_ln', M, [_p(b.tok), _i(M), _p(m.t), _p(W['wte']), _p(b.wpe), _p(b.Z), _i(D), _i(V),
                                            _i(M), _p(W['ln1w'][0]), _p(W['ln1b'][0]), _p(b.AF), _i(mt), _p(err)])

        def qkv(layer):                  # row i of layer l is row i + l to the epilogue
            m.keys, m.vals = (ctypes.c_void_p(t.data_ptr() - 2 * layer * D) for t in (b.K, b.V))
            self._product(b.AF, D, 'qkvw', layer, 3 * D, MODE_QKV, bias=W['qkvb'][layer], out=b.Q, ldo=D, M=M, P=1)

        def rest(layer):
            self._launch('pf_frag_rows', -(-M * (D // 8) // PF_BLOCK), [_p(b.O), _i(M), _i(D), _p(b.AF), _i(mt), _p(err)])
            ln2 = W['ln2w'][layer], W['ln2b'][layer], b.AF
            if not self._product(b.AF, D, 'ow', layer, D, MODE_RESID, bias=W['ob'][layer], out=b.Z, ldo=D, ln=ln2, M=M):
                self._norm(b.Z, *ln2, M)
            self._product(b.AF, D, 'fcw', layer, F, MODE_GELU, bias=W['fcb'][layer], F=b.GF, M=M)
            last = layer + 1 == self.layers
            ln1 = None if last else (W['ln1w'][layer + 1], W['ln1b'][layer + 1], b.AF)
            if not self._product(b.GF, F, 'pw', layer, D, MODE_RESID, bias=W['pb'][layer], out=b.Z, ldo=D, ln=ln1, M=M) \
                    and not last:
                self._norm(b.Z, *ln1, M)

        def head():
            self._norm(b.ZL, W['lnfw'], W['lnfb'], b.CF, B)
            if B <= MHEAD_ROWS:
                self._mhead(b.CF, D, V, b.logit, B)
            else:
                self._pgemm(b.CF, D, 'wte', None, V, MODE_PLAIN, out=b.logit, ldo=V, M=B)
            self._launch('pf_argmax_part', B * ARGMAX_SPLIT, [_p(b.logit), _i(V), _i(ARGMAX_SPLIT), _p(b.apv), _p(b.api)])
            self._launch('pf_argmax', B, [_p(b.apv), _p(b.api), _i(ARGMAX_SPLIT), _p(b.x), _p(b.next), _p(m.t), _i(0)])

        self._plans[key] = (self._record(embed), [self._record(lambda n=n: qkv(n)) for n in range(self.layers)],
                            [self._record(lambda n=n: rest(n)) for n in range(self.layers)], self._record(head))
        return self._plans[key]

    def _score_room(self, M):
        """Buffers for the logits of M rows, SCORED at a time."""
        import torch
        from . import logprobs
        rows = min(SCORED, M)
        if self._scores is not None and self._scores[1].shape[0] >= rows:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f'extend: call once with the log probabilities of {M} tokens before capturing such a call')
        W, dev = self.m.W['wte'], self.err.device
        logprobs.load(dev.index, torch.float32)
        rows = min(SCORED, 1 << (rows - 1).bit_length())
        self._outgrown.append(self._scores)
        self._scores = (torch.zeros(2 * 16 * _mtiles(rows) * self.m.D, dtype=torch.float16, device=dev),
                        torch.empty(rows, W.shape[0], dtype=torch.float32, device=dev))
        self._score_plans = {}

    def _score(self, M, given, top):
        """The log probabilities of all M rows (``vesta.logprobs``), their logits made SCORED rows at a time."""
        from . import logprobs
        m, b, W = self.m, self._buf, self.m.W
        D, V, dev = m.D, W['wte'].shape[0], self.err.device
        frag, logits = self._scores
        if M not in self._score_plans:
            while len(self._score_plans) >= PLANS:
                del self._score_plans[next(iter(self._score_plans))]

            def product(first, n):
                self._norm(b.Z[first:first + n], W['lnfw'], W['lnfb'], frag, n)
                if n <= MHEAD_ROWS:
                    self._mhead(frag, D, V, logits, n)
                else:
                    self._pgemm(frag, D, 'wte', None, V, MODE_PLAIN, out=logits, ldo=V, M=n)

            self._score_plans[M] = [(first, n, self._record(lambda first=first, n=n: product(first, n)))
                                    for first in range(0, M, SCORED) for n in (min(SCORED, M - first),)]
        got = logprobs.empty(given, top, M, dev)
        for first, n, plan in self._score_plans[M]:
            self._replay(plan)
            part = slice(first, first + n)
            logprobs.fill(logprobs.LogProbs(*(None if t is None else t[part] for t in got)), logits[:n],
                          None if given is None else given[part], top)
        return got

    def run(self, cache, tokens, positions, table, starts, lengths, weight=None, most=None, given=None, top=0):
        """The new tokens' pass; returns the logits of each sequence's last
        row and the largest's id, which the next call overwrites, and, of
        ``given`` tokens or ``top`` alternatives, all rows' log probabilities."""
        import torch
        M, B, H = tokens.shape[0], table.shape[0], self.m.H
        scored = given is not None or top
        self._room(M, B)
        if scored:
            self._score_room(M)
        embed, qkv, rest, head = self._launches(M, B)
        b = self._buf
        wpe = self.m.W['wpe']
        stream, back = cache._enter()
        try:
            cache._kind[cache.dtype].pg_input(
                -(-M * (self.m.D // 8) // BLOCK), BLOCK, stream, tokens.data_ptr(), positions.data_ptr(), wpe.data_ptr(),
                wpe.shape[0], self.m.D, self.m.W['wte'].shape[0], starts.data_ptr(), lengths.data_ptr(), B, M,
                table.shape[1] * cache.page, b.tok.data_ptr(), b.wpe.data_ptr(), cache._err)
        finally:
            cache._leave(back)
        q, o, k, v = (t[:M].view(M, H, -1) for t in (b.Q, b.O, b.K, b.V))
        self._replay(embed)
        for layer in range(self.layers):
            self._replay(qkv[layer])
            cache.append(k, v, table, starts, lengths, layer)
            cache.attend(q, table, starts, lengths, layer, out=o, most=most,
                         **({} if weight is None else dict(weight=weight[layer])))
            self._replay(rest[layer])
        torch.index_select(b.Z, 0, (starts[1:] - 1).clamp(0, M - 1), out=b.ZL[:B])
        self._replay(head)
        out = b.logit[:B], b.x[:B]
        return (*out, self._score(M, given, top)) if scored else out
