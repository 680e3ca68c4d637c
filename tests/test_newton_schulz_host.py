"""Which out= of newton_schulz is written where it lies, decided on the host."""
import torch

from mi_adamw.muon import _overlap


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
