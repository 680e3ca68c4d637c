"""newton_schulz's host side: which out= is written where it lies, and options past fp32."""
import pytest
import torch

import mi_adamw
from mi_adamw import _lib
from mi_adamw.muon import NS_COEFFICIENTS, _options, _overlap


def test_overlap():
    buffer = torch.zeros(4000)

    def at(start, stride, shape=(3, 5, 7)):
        return buffer.as_strided(shape, stride, start)

    x = at(100, (35, 7, 1))
    assert not _overlap(x, x) and not _overlap(x, at(100, (35, 7, 1)))
    for out in (at(101, (35, 7, 1)), at(135, (35, 7, 1)), at(65, (35, 7, 1)), at(100, (40, 7, 1)),
                at(204, (35, 7, 1)), at(0, (50, 7, 1)), at(100, (35, 1, 5))):
        assert _overlap(x, out) and _overlap(out, x)
    for out in (at(205, (35, 7, 1)), at(1000, (35, 7, 1)), torch.zeros(3, 5, 7)):
        assert not _overlap(x, out) and not _overlap(out, x)
    # a batch that repeats one matrix, and one matrix, which is read before any of it is written
    assert _overlap(at(100, (0, 7, 1)), at(100, (35, 7, 1)))
    assert not _overlap(x[:1], at(101, (35, 7, 1), (1, 5, 7)))


@pytest.mark.parametrize("eps", [1e39, -1e39, 3.5e38])
def test_an_eps_past_fp32_is_named(eps):
    """The kernels hold eps in fp32."""
    with pytest.raises(ValueError, match="eps"):
        _options(NS_COEFFICIENTS, eps, 5, _lib.NS_HALF)
    with pytest.raises(ValueError, match="eps"):
        mi_adamw.Muon([torch.nn.Parameter(torch.zeros(3, 4))], eps=eps)
    _options(NS_COEFFICIENTS, 3.4e38, 5, _lib.NS_HALF)
