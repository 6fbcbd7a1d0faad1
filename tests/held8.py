"""What a cache in 8 bits holds (vesta/paged8.py), from its definition, in 64 bits: by tables and searches, not by the
bits that the kernels work on."""
import torch

LOW = {('i8', 'f16'): -24, ('i8', 'bf16'): -126, ('e4m3', 'f16'): -15, ('e4m3', 'bf16'): -117}
HIGH = {('i8', 'f16'): 9, ('i8', 'bf16'): 119, ('e4m3', 'f16'): 7, ('e4m3', 'bf16'): 119}
BIAS = {'i8': 133, 'e4m3': 127}
# the values of the codes 0 .. 126 of an e4m3 float without its sign; 127 is a NaN
E4M3 = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def power2(p):
    """2^p exactly, p a whole-number tensor."""
    return ((p.long() + 1023) << 52).view(torch.float64)


def hold(x, form, dtype):
    """Codes [.., width] (uint8) and powers' bytes [.., width / 32] of x [.., width]."""
    x = x.double().unflatten(-1, (-1, 32))
    finite = x.isfinite()
    largest = torch.where(finite, x.abs(), 0.0).amax(-1, keepdim=True)
    low, high = LOW[form, dtype], HIGH[form, dtype]
    edges = (127.5 if form == 'i8' else 464.0) * power2(torch.arange(low, high, device=x.device))
    p = low + (largest >= edges).sum(-1, keepdim=True)
    y = x / power2(p)
    if form == 'i8':
        code = torch.round(y.nan_to_num(0.0, 0.0, 0.0)).clamp(-127, 127).long() & 255
        byte = torch.where(finite.all(-1), p.squeeze(-1) + 133, 255)
    else:
        table = torch.tensor(E4M3, dtype=torch.float64, device=x.device)
        up = torch.searchsorted(table, y.abs().nan_to_num(0.0, 0.0, 0.0)).clamp(1, 126)
        over, under = table[up] - y.abs(), y.abs() - table[up - 1]
        code = torch.where((over < under) | ((over == under) & (up % 2 == 0)), up, up - 1)
        code = torch.where(finite, code + 128 * torch.signbit(x), 127)
        byte = p.squeeze(-1) + 127
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def values(code, byte, form):
    """What codes (uint8) and bytes stand for, in 64 bits."""
    c = code.long()
    if form == 'i8':
        x = torch.where(c > 127, c - 256, c).double()
        x = torch.where((byte == 255).repeat_interleave(32, -1), torch.nan, x)
    else:
        table = torch.tensor(E4M3 + [float('nan')], dtype=torch.float64, device=code.device)
        x = table[c & 127] * torch.where(c > 127, -1.0, 1.0)
    return x * power2(byte.long() - BIAS[form]).repeat_interleave(32, -1)
