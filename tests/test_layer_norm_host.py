"""layer_norm's Python path on the CPU, its launches stubbed."""
import gc

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

from mi_adamw import norm


@pytest.fixture
def launches(monkeypatch):
    made = []
    monkeypatch.setattr(norm, "_call", lambda fn, args, device, what: made.append((what, args)))
    return made


@pytest.mark.parametrize("residual", [False, True])
def test_a_forward_without_its_backward_ends(launches, residual):
    """What the outputs' node saves holds neither the node nor the outputs."""
    x = torch.randn(6, 16, requires_grad=True)
    r = torch.randn(6, 32)[:, ::2].requires_grad_(True) if residual else None
    w, b = (torch.randn(16, requires_grad=True) for _ in "wb")
    out = norm._LayerNorm.apply(x, r, w, b, 1e-5, torch.float32)
    outs = out if residual else (out,)
    ends = [StorageWeakRef(t.untyped_storage()) for t in outs]
    assert len(launches) == 1 and not any(e.expired() for e in ends)
    del out, outs
    gc.collect()
    assert all(e.expired() for e in ends)


@pytest.mark.parametrize("residual", [False, True])
def test_the_backward_reads_what_was_normalised(launches, residual):
    x = torch.randn(2, 3, 16, requires_grad=True)
    r = torch.randn(2, 3, 16, requires_grad=True) if residual else None
    w = torch.randn(16, requires_grad=True)
    out = norm._LayerNorm.apply(x, r, w, None, 1e-5, torch.float32)
    y, s = out if residual else (out, x)
    y.sum().backward()
    (_, forward), (_, args) = launches
    assert args.x == s.data_ptr() == (forward.sum if residual else forward.x)
    assert (args.rows, args.hidden, args.x_row) == (6, 16, 16)
    assert (args.mean, args.rstd) == (forward.mean, forward.rstd)


def test_a_changed_sum_is_noticed(launches):
    x, r = (torch.randn(6, 16, requires_grad=True) for _ in "xr")
    y, s = norm._LayerNorm.apply(x, r, None, None, 1e-5, torch.float32)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
