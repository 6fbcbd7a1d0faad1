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
stream; nothing is read back, so a call can be captured in a HIP graph. Sums
are fp32. A banned token (-inf) has the log probability -inf; a row that bans
all has -inf throughout and the entropy 0. A NaN or +inf in a row makes its
results NaN (ids are of its order then, NaN the largest). A given id outside
the vocabulary has the log probability NaN. There is no backward pass: logits
whose gradient is being recorded are refused.

The reference's programs end in the largest logit's id (reference
``vesta/programs/gpt2.vst:78-82``).
"""
from __future__ import annotations

import operator
from collections import namedtuple
from pathlib import Path

from .paged import loaded
from .prefill import PRELUDE_SRC

LOGPROBS_SRC = Path(__file__).resolve().parent / 'hip' / 'logprobs.hip'
KINDS = ('f32', 'f16', 'bf16')
TOP = 64                               # alternatives at most

SIGNATURES = {
    **{f'lp_rows{n}': 'pli' + 'piiiii' + 'ppppp' for n in (256, 512, 1024)},
    'lp_join': 'pli' + 'piiii' + 'ppppp',
}

LogProbs = namedtuple('LogProbs', 'given entropy top ids')


def logprobs_source(kind: str) -> str:
    return f'#define VBLOCK 256\n#define LP_KIND {KINDS.index(kind)}\n' + PRELUDE_SRC.read_text() + '\n' + LOGPROBS_SRC.read_text()


def _layout(M, V, size):
    """The threads of a block, the parts of a row and the elements of one."""
    return 1024, 1, V


def _kernels(device, kind):
    return loaded(device, ('logprobs', kind), lambda: logprobs_source(kind), SIGNATURES)


def logprobs(logits, given=None, top=0):
    """``LogProbs(given, entropy, top, ids)`` of rows of logits [M, V]: see
    above. ``given`` is None where none is given, ``top`` and ``ids`` are None
    for ``top=0``; ``top`` is at most 64 and V."""
    import torch
    kinds = {torch.float32: 'f32', torch.float16: 'f16', torch.bfloat16: 'bf16'}
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in kinds):
        raise TypeError('logits: need a device tensor of float32, float16 or bfloat16')
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError('logits: no gradient is made of them; detach them, or call under torch.no_grad()')
    if logits.dim() != 2 or not 1 <= logits.shape[1] < 1 << 30:
        raise ValueError(f'logits: shape {tuple(logits.shape)}, need rows of 1 to 2^30 logits')
    M, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        raise ValueError(f'logits: rows of consecutive values needed (strides {logits.stride()})')
    top = operator.index(top)
    if not 0 <= top <= min(TOP, V):
        raise ValueError(f'top {top}: from 0 to {min(TOP, V)}')
    if given is not None:
        if not (isinstance(given, torch.Tensor) and given.dtype in (torch.int32, torch.int64)
                and given.device == logits.device and given.is_contiguous()):
            raise TypeError(f'given: need a contiguous int32 or int64 tensor on {logits.device}')
        if given.dim() not in (1, 2) or given.shape[0] != M:
            raise ValueError(f'given: shape {tuple(given.shape)}, need ({M},) or ({M}, any)')
    return _run(logits, kinds[logits.dtype], given, top)


def _run(logits, kind, given, top):
    import torch
    M, V = logits.shape
    dev, size = logits.device, logits.element_size()
    f32 = dict(dtype=torch.float32, device=dev)
    entropy = torch.empty(M, **f32)
    out = None if given is None else torch.empty(given.shape, **f32)
    best = torch.empty((M, top), **f32) if top else None
    ids = torch.empty((M, top), dtype=torch.int32, device=dev) if top else None
    got = LogProbs(out, entropy, best, ids)
    if M == 0:
        return got
    C = 0 if given is None or given.numel() == 0 else given.numel() // M
    threads, parts, each = _layout(M, V, size)
    if M * parts >= 1 << 31:
        raise ValueError(f'logits: {M} rows are too many for one call')
    index = dev.index
    kn = _kernels(index, kind)
    ws = torch.empty(M * parts * (2 + top), dtype=torch.int64, device=dev) if parts > 1 else None
    row = (logits.data_ptr(), logits.stride(0) if M > 1 else V, V, given.data_ptr() if C else 0,
           int(C > 0 and given.dtype == torch.int64), C, top, parts)
    to = (out.data_ptr() if C else 0, entropy.data_ptr(), best.data_ptr() if top else 0, ids.data_ptr() if top else 0,
          ws.data_ptr() if parts > 1 else 0)
    back = torch.cuda.current_device()
    if back != index:
        torch.cuda.set_device(index)
    try:
        stream = torch._C._cuda_getCurrentRawStream(index)
        getattr(kn, f'lp_rows{threads}')(M * parts, threads, stream, *row, each, *to)
        if parts > 1:
            kn.lp_join(M, 256, stream, *row, *to)
    finally:
        if back != index:
            torch.cuda.set_device(back)
    return got
