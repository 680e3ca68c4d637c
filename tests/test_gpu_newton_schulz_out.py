"""newton_schulz's out=: autograd sees the write, memory that out shares with x, and large batches."""
import pytest
import torch

import mi_adamw

pytestmark = pytest.mark.gpu

DEV = "cuda"
SINGLE = 199 * 3 * 2.0 ** -23            # derived in test_gpu_newton_schulz.py


def normal(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


@pytest.mark.parametrize("shape", [(20, 30), (200, 300), (3, 20, 30)])
@pytest.mark.parametrize("layout", ["itself", "dense", "columns dense", "strided"])
def test_out_is_seen_by_autograd(shape, layout):
    x = normal(*shape)
    if layout == "itself":
        out = x
    elif layout == "dense":
        out = torch.empty_like(x)
    elif layout == "columns dense":
        out = torch.empty_like(x.mT.contiguous()).mT
    else:
        out = torch.empty(*shape, 2, device=DEV)[..., 0]
    w = torch.ones_like(x, requires_grad=True)
    product = (w * out).sum()               # saves out for w's gradient
    version = out._version
    mi_adamw.newton_schulz(x, out=out)
    assert out._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_x_alone_is_not_written():
    x = normal(40, 50)
    version = x._version
    mi_adamw.newton_schulz(x)
    assert x._version == version
    with torch.inference_mode():            # tensors without a version
        y = torch.empty_like(x)
        mi_adamw.newton_schulz(x, out=y)
    assert torch.equal(y, mi_adamw.newton_schulz(x))


@pytest.mark.parametrize("rows,cols", [(40, 60), (150, 200)])
@pytest.mark.parametrize("ahead", [False, True])
def test_out_among_the_batch(rows, cols, ahead, monkeypatch):
    """out begins a matrix, or a row, before or behind x in the same memory."""
    from mi_adamw import muon
    monkeypatch.setattr(muon, "_WORKSPACE", 3 * 192 * 256 * 12)    # a few matrices at once
    for shift in (rows * cols, cols):
        n = 9
        store = normal((n + 1) * rows * cols)
        early, late = (store[s:s + n * rows * cols].view(n, rows, cols) for s in (0, shift))
        x, out = (early, late) if ahead else (late, early)
        want = torch.stack([mi_adamw.newton_schulz(m) for m in x.clone()])
        assert mi_adamw.newton_schulz(x, out=out) is out
        assert ((out - want).norm() <= 2 * SINGLE * want.norm()).item()


def test_more_matrices_than_a_launch_takes():
    for rows, cols in ((1, 1), (2, 3)):
        x = normal(2 ** 23 + 5, rows, cols)
        got = mi_adamw.newton_schulz(x)
        for at in (0, 2 ** 23 - 2, 2 ** 23 - 1, 2 ** 23 + 4):
            want = mi_adamw.newton_schulz(x[at])
            assert ((got[at] - want).norm() <= 2 * SINGLE * want.norm()).item()
        assert torch.isfinite(got).all()
    # as many, of more 64 x 64 blocks
    x = normal(2 ** 21, 1, 1).expand(-1, 1, 320)
    assert torch.isfinite(mi_adamw.newton_schulz(x)).all()
