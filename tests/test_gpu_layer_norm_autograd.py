"""layer_norm among autograd's other parts: errors keep their types through the native call,
activation checkpoints, saved-tensor hooks, forward-mode derivatives."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.utils.checkpoint import checkpoint

import mi_adamw

pytestmark = pytest.mark.gpu

DEV = "cuda"


def normal(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


def leaves(rows=24, hidden=96):
    return [t.requires_grad_(True) for t in (normal(rows, hidden), normal(rows, hidden, seed=1),
                                             normal(hidden, seed=2), normal(hidden, seed=3))]


def norm(x, r, w, b):
    return mi_adamw.layer_norm(x, w, b, residual=r)


def grads(f, ts):
    y, s = f(*ts)
    return torch.autograd.grad((y.square().sum() + (s * s.detach().cos()).sum()), ts)


@pytest.mark.parametrize("early_stop", [True, False])
@pytest.mark.parametrize("strided", [False, True])
def test_activation_checkpoint(early_stop, strided):
    """The recomputation ends, by an exception from within the norm's own saving of tensors, as soon
    as everything is there again."""
    from torch.utils.checkpoint import set_checkpoint_early_stop
    ts = leaves()
    if strided:
        ts[1] = normal(24, 192)[:, ::2].detach().requires_grad_(True)
    want = grads(norm, ts)
    with set_checkpoint_early_stop(early_stop):
        got = grads(lambda *a: checkpoint(norm, *a, use_reentrant=False), ts)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_an_error_in_a_hook_keeps_its_type():
    class Mine(Exception):
        pass

    def refuse(t):
        raise Mine("no")

    ts = leaves()
    with pytest.raises(Mine):
        with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t):
            norm(*ts)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
        y, s = norm(*ts)
    with pytest.raises(Mine):
        (y.sum() + s.sum()).backward()


@pytest.mark.parametrize("when", ["forward", "backward"])
def test_out_of_memory_keeps_its_type(when):
    x = torch.zeros(1 << 18, 1 << 10, device=DEV, requires_grad=True)        # 1 GiB
    w = torch.ones(1 << 10, device=DEV)
    if when == "backward":
        y = mi_adamw.layer_norm(x, w, out_dtype=torch.bfloat16)
        dy = torch.zeros_like(y)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    room = torch.cuda.memory_reserved() + (256 << 20)
    torch.cuda.set_per_process_memory_fraction(room / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            if when == "forward":
                mi_adamw.layer_norm(x, w)
            else:
                torch.autograd.grad(y, x, dy)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


@pytest.mark.parametrize("when", ["forward", "backward"])
def test_a_refusal_of_the_library_is_its_own_error(when):
    import ctypes
    from mi_adamw import _lib
    lib = _lib.load()
    own = [ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _lib.NORM_BINDINGS]
    refuse = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)(
        lambda args, stream: _lib.E_INVALID)
    at = ctypes.cast(refuse, ctypes.c_void_p).value
    ts = leaves()
    y, s = norm(*ts)
    try:
        _lib._host.bind_layer_norm(at, own[1], at, own[3], _lib.MiAdamwError)
        with pytest.raises(mi_adamw.MiAdamwError, match="invalid argument"):
            norm(*ts) if when == "forward" else (y.sum() + s.sum()).backward()
    finally:
        _lib._host.bind_layer_norm(*own, _lib.MiAdamwError)
    norm(*ts)[0].sum().backward()


@pytest.mark.parametrize("strided", [False, True])
def test_saved_tensors_that_come_back_in_another_layout(strided):
    """A hook gives back the same values, at strides of its own."""
    ts = leaves()
    if strided:
        ts[0] = normal(24, 192)[:, ::2].detach().requires_grad_(True)
    want = grads(norm, ts)

    def pack(t):
        return t.dim(), t.t().contiguous() if t.dim() == 2 else torch.stack([t, t], 1)

    def unpack(packed):
        dim, t = packed
        return t.t() if dim == 2 else t[:, 0]

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y, s = norm(*ts)
    got = torch.autograd.grad((y.square().sum() + (s * s.detach().cos()).sum()), ts)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("mode", ["no gradient", "gradient", "no_grad"])
@pytest.mark.parametrize("strided", [False, True])
def test_forward_mode_derivatives_are_refused(which, mode, strided):
    ts = [t.detach() for t in leaves()]
    if strided:
        ts[0] = normal(24, 192)[:, ::2]
    if mode == "gradient":
        ts = [t.requires_grad_(True) for t in ts]
    norm(*ts)
    with fwAD.dual_level(), torch.set_grad_enabled(mode != "no_grad"):
        norm(*ts)
        ts[which] = fwAD.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            norm(*ts)


def test_newton_schulz_refuses_forward_mode():
    x = normal(20, 30)
    with fwAD.dual_level():
        y = mi_adamw.newton_schulz(x)
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mi_adamw.newton_schulz(dual)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mi_adamw.newton_schulz(x, out=fwAD.make_dual(y, torch.ones_like(y)))


def test_function_transforms_are_refused():
    """torch.func's wrappers have no memory of their own: an error, not a wrong number."""
    x, w = normal(4, 16), normal(16)
    for f in (lambda a: torch.func.jvp(lambda t: mi_adamw.layer_norm(t, w), (a,), (a,)),
              lambda a: torch.func.vmap(lambda t: mi_adamw.layer_norm(t, w))(a),
              lambda a: torch.func.grad(lambda t: mi_adamw.layer_norm(t, w).sum())(a),
              lambda a: torch.func.jvp(mi_adamw.newton_schulz, (a,), (a,))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(x)


@pytest.mark.parametrize("strided", [False, True])
def test_an_eps_past_fp32_is_refused(strided):
    x, w = normal(4, 64), normal(64)
    x = x[:, ::2] if strided else x[:, :32].contiguous()
    with pytest.raises(ValueError, match="eps"):
        mi_adamw.layer_norm(x, w[:32], None, 1e39)
    assert torch.isfinite(mi_adamw.layer_norm(x, w[:32], None, 3.4e38)).all()
