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
@pytest.mark.parametrize('top', (0, 5, 20, 64))
@pytest.mark.parametrize('M', (1, 8, 64, 65, 256, 300, 4096, 100000))
@pytest.mark.parametrize('V', (1, 3, 1000, 5001, 32768, 32769, 50257, 128001, 200000, 1 << 19, (1 << 19) + 1, (1 << 30) - 1))
def test_layout(M, V, size, top):
    """The parts of a row cover it, none is empty, and the kernels' limits hold."""
    name, threads, parts, each = lp._layout(M, V, size, top)
    assert name in lp.SIGNATURES and 1 <= parts <= 64
    assert parts * each >= V > (parts - 1) * each
    if name.startswith('lp_part'):
        assert threads == 256 and each <= 256 * int(name[7:]) * (16 // size) and V >= 16 // size and each % (16 // size) == 0
    else:
        assert name == f'lp_rows{threads}'


def test_tangents_refused():
    """Forward-mode derivatives are not made either, and not dropped without a word; outside a level nothing has one."""
    import torch.autograd.forward_ad as fwd
    x = torch.zeros(3, 8)
    with fwd.dual_level():
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(ValueError, match='logits'):
                lp.logprobs(_on(fwd.make_dual(x, torch.ones_like(x))))
        with pytest.raises(ValueError, match='top'):       # (no tangent: on to the next check)
            lp.logprobs(_on(x), top=9)
