"""newton_schulz, layer_norm and Muon called from torch.compile'd functions: they run as they are,
between the graphs.  A trace refuses them."""
import pytest
import torch

import mi_adamw

pytestmark = pytest.mark.gpu

DEV = "cuda"


def normal(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


def compiled(f):
    torch._dynamo.reset()
    return torch.compile(f, backend="eager")


@pytest.mark.parametrize("options", [{}, dict(precision="half", steps=3)])
def test_newton_schulz(options):
    x = normal(150, 200)

    def f(t):
        return 2 * mi_adamw.newton_schulz(t + 1, **options)

    assert torch.equal(compiled(f)(x), f(x))


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_layer_norm(strided, residual, grad):
    x = normal(12, 128)[:, ::2] if strided else normal(12, 64)
    ts = [x.detach(), normal(12, 64, seed=1), normal(64, seed=2), normal(64, seed=3)]
    ts = [t.requires_grad_(grad) for t in ts]

    def f(x, r, w, b):
        x = torch.as_strided(x, x.shape, x.stride()) if strided else x * 2
        out = mi_adamw.layer_norm(x, w, b, residual=r if residual else None)
        return out[0] + 3 * out[1] if residual else out * 3

    want, got = f(*ts), compiled(f)(*ts)
    assert torch.equal(want, got)
    if grad:
        used = ts if residual else [ts[0], *ts[2:]]
        for a, b in zip(torch.autograd.grad(got.square().sum(), used),
                        torch.autograd.grad(want.square().sum(), used)):
            assert torch.equal(a, b)


def test_module_and_step():
    def run(wrap):
        torch.manual_seed(0)
        model = torch.nn.Sequential(torch.nn.Linear(64, 96, bias=False), mi_adamw.LayerNorm(96),
                                    torch.nn.Linear(96, 64, bias=False)).to(DEV)
        opt = mi_adamw.Muon([p for p in model.parameters() if p.dim() == 2], lr=0.02)
        f, x = wrap(model), normal(8, 64)
        for _ in range(3):
            opt.zero_grad()
            f(x).square().mean().backward()
            opt.step()
        return [p.detach() for p in model.parameters()]

    assert all(torch.equal(a, b) for a, b in zip(run(compiled), run(lambda m: m)))


@pytest.mark.parametrize("strided", [False, True])
def test_tracing_is_refused(strided):
    """A trace would record the outputs' allocation and none of the launches."""
    x, w = normal(4, 64), normal(32)
    x = x[:, ::2] if strided else x[:, :32].contiguous()
    for f in (lambda t: mi_adamw.layer_norm(t, w), mi_adamw.newton_schulz):
        with pytest.raises(NotImplementedError, match="torch.jit.trace"):
            torch.jit.trace(f, x, check_trace=False)
