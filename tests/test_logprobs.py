"""CPU tests of ``vesta.logprobs.logprobs``: what is refused."""
import pytest
import torch

from vesta import logprobs as lp


class _Device(torch.Tensor):
    """A tensor on the CPU that says it is a device's."""
    is_cuda = True


def _on(t):
    return t.as_subclass(_Device)


def test_needs_a_device_tensor():
    for bad in (torch.zeros(2, 8), None, [[0.0]], _on(torch.zeros(2, 8, dtype=torch.float64)),
                _on(torch.zeros(2, 8, dtype=torch.int32))):
        with pytest.raises(TypeError, match='logits'):
            lp.logprobs(bad)


@pytest.mark.parametrize('logits', [torch.zeros(8), torch.zeros(2, 2, 8), torch.zeros(2, 0), torch.zeros(8, 2).t(),
                                    torch.zeros(2, 16)[:, ::2], torch.zeros(2, 8, requires_grad=True)])
def test_shapes_and_strides(logits):
    with pytest.raises(ValueError, match='logits'):
        lp.logprobs(_on(logits))


def test_other_arguments():
    x = _on(torch.zeros(3, 8))
    for top in (-1, 9, 65):
        with pytest.raises(ValueError, match='top'):
            lp.logprobs(x, top=top)
    with pytest.raises(TypeError):
        lp.logprobs(x, top=1.5)
    for given in ([0, 1, 2], torch.zeros(3), torch.zeros(3, dtype=torch.int16), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(TypeError, match='given'):
            lp.logprobs(x, given)
    for shape in ((), (2,), (4, 1), (3, 1, 1)):
        with pytest.raises(ValueError, match='given'):
            lp.logprobs(x, torch.zeros(shape, dtype=torch.int64))


@pytest.mark.parametrize('size', (2, 4))
@pytest.mark.parametrize('M,V', [(1, 1), (1, 50257), (8, 50257), (1, 1 << 20), (3, 200000), (4096, 50257), (100000, 3), (64, 128001)])
def test_layout(M, V, size):
    """The parts of a row cover it, none is empty, and the joining kernel's limit holds."""
    threads, parts, each = lp._layout(M, V, size)
    assert threads in (256, 512, 1024) and 1 <= parts <= 64
    assert parts * each >= V > (parts - 1) * each
