"""Log probabilities of given tokens, entropies and the most likely tokens.

    got = logprobs(logits, given, top=5)
    got.given      # [M] or [M, C]: each row's log probability of its given tokens
    got.entropy    # [M]: of the row's distribution, in nats
    got.top        # [M, 5]: the largest log probabilities, in order
    got.ids        # [M, 5]: whose they are (int32); of equal ones the lowest id first

``logits`` are rows [M, V] of f32, f16 or bf16 with any pitch, ``given`` int32
or int64 ids [M] or [M, C] on the same device (None: none). What tells how well
a model, or a cache held in fewer bits, predicts a text (``VestaGPT2.extend``
with ``given``), and what a server answers with beside its tokens.

Rows are read once, in one launch (two for few long rows), on torch's current
stream; nothing is read back, so a call can be captured in a HIP graph (after a
first one of its type of logits). Sums are fp32. With alternatives asked for, a
row is read two or three times more where over a thousand of its tokens tie for
the last of them (a mask of a finite value that leaves fewer than are asked
for, a flat row), or one is NaN or +inf; bans of -inf do not need that. Only where
more than a thousand large ones lie in the same places of each 64 loads of 16
bytes is it read once for each alternative.

A banned token (-inf) has the log probability -inf; a row that bans all has -inf
throughout and the entropy 0. A NaN or +inf in a row makes its results NaN (ids
are of its order then, NaN the largest). A given id outside the vocabulary has
the log probability NaN. There is no backward pass, no forward-mode one either:
logits whose gradient is being recorded, or that have a tangent, are refused.

The reference's programs end in the largest logit's id (reference
``vesta/programs/gpt2.vst:78-82``).
"""
from __future__ import annotations

import functools
import operator
from collections import namedtuple
from pathlib import Path

from .paged import loaded
from .prefill import PRELUDE_SRC

LOGPROBS_SRC = Path(__file__).resolve().parent / 'hip' / 'logprobs.hip'
KINDS = ('f32', 'f16', 'bf16')
TOP = 64                               # alternatives at most
JOIN_FEW = 256                         # of a row's parts together, up to which lp_join takes them

SIGNATURES = {
    **{f'lp_rows{n}': 'pli' + 'piiiii' + 'ppppp' for n in (64, 256, 512, 1024)},
    **{f'lp_part{n}': 'pliiii' + 'p' for n in (2, 4, 8)},
    **{name: 'pli' + 'piiii' + 'ppppp' for name in ('lp_join', 'lp_join_many')},
}

LogProbs = namedtuple('LogProbs', 'given entropy top ids')


def logprobs_source(kind: str) -> str:
    return f'#define VBLOCK 256\n#define LP_KIND {KINDS.index(kind)}\n' + PRELUDE_SRC.read_text() + '\n' + LOGPROBS_SRC.read_text()


# How rows are laid out; us a call (GPU time), f32 logits if not said, k alternatives, on both sides of each rule.
# Rows of up to so many bytes are a wave's (20,000 x 1000, a wave / 256 threads: 19 / 47; 30 x 1000, k 5: 4.5 / 4.7; 100 x
# 3000: 3.9 / 3.3; 1000 x 3000, k 5: 8.0 / 6.9) ...
WAVE_BYTES = 8 << 10
# ... of up to so many a block's of 256 threads (256 / 512: 16 x 20,000, k 5: 6.4 / 6.5; 3000 x 16,000 31.2 / 31.4, k 5 34.0 /
# 39.3; 5000 x 30,000 bf16 57 / 63, k 5 74 / 91; 8192 x 50,257 283 / 270, k 5 286 / 280) ...
BLOCK_BYTES = 128 << 10
# ... of more a block's of 1024 threads for up to so many rows, a CU each, of 512 for more (1024 / 512: 8 x 50,257, k 5: 9.1 /
# 9.1; 200: 10.9 / 12.9; 512: 24.4 / 22.8; 8192: 323 / 279; 200 x 128,001 bf16, k 20: 20.6 / 25.4).
CU_ROWS = 256
# Rows of more than so many bytes are dealt to blocks whose elements stay in registers (lp_part), and a second launch joins
# them: it takes 5 us of the host's more, and for short rows saves less (whole / in parts; 8 x 50,257 7.0 / 4.9, k 5 9.1 /
# 7.2, one call after another from Python 13.5 / 18.6). A captured call, which does without the host, is laid out alike ...
PART_BYTES = 240 << 10
# ... for up to so many rows (64 x 128,001 bf16, k 20: 19.1 / 13.5; 100: 19.9 / 18.4; 200: 20.6 / 26.6) ...
PARTS_ROWS = 64
# ... or so many with no alternatives (200 x 128,001 bf16 13.4 / 13.9; 300: 23.4 / 18.1) ...
PARTS_ROWS_NO_TOP = 384
# ... in the smallest parts (2, 4 or 8 loads a thread) with which there are up to so many, and up to JOIN_FEW alternatives
# of a row (8 x 50,257, k 5, parts of 2 / 4 / 8 loads: 7.2 / 7.2 / 7.9; 64: 10.1 / 9.3 / 8.8; 8 x 128,001 bf16, k 20: 13.3 / 11.3 /
# 11.0).
PARTS = 512
# A row past 64 of the largest parts goes to blocks that loop over 64 parts (1 x 2,000,000: 7.0, whole 145).
MOST_PARTS = 64


@functools.lru_cache(maxsize=256)
def _layout(M, V, size, top):
    """The kernel of a row or its parts, its threads, how many parts and the elements of one."""
    row = V * size
    if row <= BLOCK_BYTES:
        threads = 64 if row <= WAVE_BYTES else 256
        return f'lp_rows{threads}', threads, 1, V
    vec = 16 // size
    if row > PART_BYTES and M <= (PARTS_ROWS if top else PARTS_ROWS_NO_TOP):
        for loads in (2, 4, 8):
            parts = -(-V // (256 * loads * vec))
            if M * parts <= PARTS and parts * top <= JOIN_FEW or loads == (8 if top else 4):
                break
        if parts <= MOST_PARTS:
            return f'lp_part{loads}', 256, parts, -(-V // (parts * vec)) * vec
        if M <= PARTS_ROWS:
            each = -(-V // MOST_PARTS)
            return 'lp_rows512', 512, -(-V // each), each
    threads = 1024 if M <= CU_ROWS else 512
    return f'lp_rows{threads}', threads, 1, V


_known = {}                            # kernels by (device index, type of logits)


def load(index, dtype):
    """The kernels of a type of logits on a device, loaded by the first call (which a capture cannot be)."""
    import torch
    kind = {torch.float32: 'f32', torch.float16: 'f16', torch.bfloat16: 'bf16'}[dtype]

    def source():
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f'logprobs: call once with {kind} logits before capturing such a call')
        return logprobs_source(kind)

    _known[index, dtype] = loaded(index, ('logprobs', kind), source, SIGNATURES)
    return _known[index, dtype]


def logprobs(logits, given=None, top=0):
    """``LogProbs(given, entropy, top, ids)`` of rows of logits [M, V]: see
    above. ``given`` is None where none is given, ``top`` and ``ids`` are None
    for ``top=0``; ``top`` is at most 64 and V."""
    import torch
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda
            and logits.dtype in (torch.float32, torch.float16, torch.bfloat16)):
        raise TypeError('logits: need a device tensor of float32, float16 or bfloat16')
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError('logits: no gradient is made of them; detach them, or call under torch.no_grad()')
    forward = torch.autograd.forward_ad
    if forward._current_level >= 0 and forward.unpack_dual(logits).tangent is not None:      # (the first: 0.3 us less)
        raise ValueError('logits: no tangent is made of them; detach them')
    shape = logits.shape
    if len(shape) != 2 or not 1 <= shape[1] < 1 << 30:
        raise ValueError(f'logits: shape {tuple(shape)}, need rows of 1 to 2^30 logits')
    M, V = shape
    if V > 1 and logits.stride(1) != 1:
        raise ValueError(f'logits: rows of consecutive values needed (strides {logits.stride()})')
    top = check(given, top, M, V, logits.device)
    got = empty(given, top, M, logits.device)
    fill(got, logits, given, top)
    return got


def check(given, top, M, V, device):
    """``top`` as a whole number, if it and ``given`` are what a call of M rows of V logits takes."""
    import torch
    top = operator.index(top)
    if not 0 <= top <= min(TOP, V):
        raise ValueError(f'top {top}: from 0 to {min(TOP, V)}')
    if given is not None:
        if not (isinstance(given, torch.Tensor) and given.dtype in (torch.int32, torch.int64) and given.device == device
                and given.is_contiguous()):
            raise TypeError(f'given: need a contiguous int32 or int64 tensor on {device}')
        shape = given.shape
        if len(shape) not in (1, 2) or shape[0] != M:
            raise ValueError(f'given: shape {tuple(shape)}, need ({M},) or ({M}, any)')
    return top


def empty(given, top, M, device):
    """Room for the results of M rows."""
    import torch
    new, f32 = torch.empty, torch.float32
    return LogProbs(None if given is None else new(given.shape, dtype=f32, device=device),
                    new(M, dtype=f32, device=device),
                    new((M, top), dtype=f32, device=device) if top else None,
                    new((M, top), dtype=torch.int32, device=device) if top else None)


def fill(got, logits, given, top):
    """The launches of a call whose arguments have been checked."""
    import torch
    M, V = logits.shape
    if M == 0:
        return
    index = logits.get_device()
    C = 0 if given is None else given.numel() // M
    name, threads, parts, each = _layout(M, V, logits.element_size(), top)
    if M * parts * threads >= 1 << 32:       # more threads than a launch can have: half the rows at a time
        for rows in (slice(0, M // 2), slice(M // 2, M)):
            fill(LogProbs(*(None if t is None else t[rows] for t in got)), logits[rows],
                 None if given is None else given[rows], top)
        return
    kn = _known.get((index, logits.dtype)) or load(index, logits.dtype)
    row = (logits.data_ptr(), logits.stride(0) if M > 1 else V, V, given.data_ptr() if C else 0,
           int(C > 0 and given.dtype is torch.int64), C, top, parts)
    in_parts = name.startswith('lp_part')
    back = torch._C._cuda_getDevice()
    if back != index:
        torch.cuda.set_device(index)
    try:
        stream = torch._C._cuda_getCurrentRawStream(index)
        ws = torch.empty(M * parts * (2 + top), dtype=torch.int64, device=logits.device) if in_parts or parts > 1 else None
        to = (got.given.data_ptr() if C else 0, got.entropy.data_ptr(), got.top.data_ptr() if top else 0,
              got.ids.data_ptr() if top else 0, 0 if ws is None else ws.data_ptr())
        if in_parts:
            getattr(kn, name)(M * parts, threads, stream, *row[:3], top, parts, each, to[-1])
        else:
            getattr(kn, name)(M * parts, threads, stream, *row, each, *to)
        if ws is not None:
            (kn.lp_join if parts * top <= JOIN_FEW else kn.lp_join_many)(M, 64, stream, *row, *to)
    finally:
        if back != index:
            torch.cuda.set_device(back)
