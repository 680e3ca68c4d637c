"""newton_schulz in half precision on matrices of low rank, whose weight lies in few rows or falls
off steeply from row to row, against the iteration in 64 bits.

Tolerance, relative in the 2-norm.  Within the rows and columns that the matrix has, a step adds
three roundings of 11 bits (of X, of S and of P off its diagonal), each times |b s^2 + c s^4| < 3 and
with nothing to average them where two rows carry everything: rms 3 * 2^-11 / sqrt(3), over five
steps 3 sqrt(5) 2^-11.  Directions outside take a share only from X's rounding times the mean of
P's diagonal: with r singular values of size s = 1 / sqrt(r) at the start, the step in which they
reach 1 adds 2.8 r / m of it and the steps left multiply by a^4 / sqrt(r):
a^4 2.8 sqrt(r) / m 2^-11 / sqrt(3).
"""
import math

import pytest
import torch

import mi_adamw
from mi_adamw.muon import NS_COEFFICIENTS

pytestmark = pytest.mark.gpu

DEV = "cuda"
A, B, C = NS_COEFFICIENTS


def limit(rank, m):
    inside = 3 * math.sqrt(5)
    outside = A ** 4 * 2.8 * math.sqrt(rank) / m / math.sqrt(3)
    return (inside + outside) * 2.0 ** -11


def exact(x):
    x = x.double()
    x = x / x.square().sum().sqrt()
    for _ in range(5):
        s = x @ x.t()
        x = A * x + (B * s + C * (s @ s)) @ x
    return x


def normal(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


def error(got, x):
    """Rows and columns of zeros stay zeros: the 64-bit iteration is run without them."""
    rows, cols = x.ne(0).any(1), x.ne(0).any(0)
    assert not got[~rows].any() and not got[:, ~cols].any()
    want = exact(x[rows][:, cols])
    return ((got[rows][:, cols].double() - want).norm() / want.norm()).item()


def few_rows(m, n, rows, rank, seed):
    x = torch.zeros(m, n, device=DEV)
    g = torch.Generator().manual_seed(seed)
    x[torch.randperm(m, generator=g)[:rows].to(DEV)] = (
        normal(rows, rank, seed=seed) @ normal(rank, n, seed=seed + 50))
    return x


@pytest.mark.parametrize("rows,rank", [(2, 1), (3, 1), (8, 1), (8, 2), (32, 1), (32, 8)])
@pytest.mark.parametrize("m,n", [(256, 384), (130, 700), (768, 768)])
@pytest.mark.parametrize("tall", [False, True])
def test_few_rows(rows, rank, m, n, tall):
    for seed in range(3):
        x = few_rows(m, n, rows, rank, seed)
        x = x.t().contiguous() if tall else x
        assert error(mi_adamw.newton_schulz(x, precision="half"), x) <= limit(rank, m)


@pytest.mark.parametrize("rank", [1, 4, 32, 256])
@pytest.mark.parametrize("spread", [1.0, 2.0, 3.0])
def test_rows_of_falling_size(rank, spread):
    x = (normal(256, 1, seed=7) * spread).exp() * (normal(256, rank) @ normal(rank, 384, seed=1))
    assert error(mi_adamw.newton_schulz(x, precision="half"), x) <= limit(rank, 256)


@pytest.mark.parametrize("rank", [1, 4, 16, 64, 128])
def test_dense_of_low_rank(rank):
    x = normal(256, rank) @ normal(rank, 384, seed=1)
    assert error(mi_adamw.newton_schulz(x, precision="half"), x) <= limit(rank, 256)


@pytest.mark.parametrize("batch,m,n", [(12, 768, 3072), (1, 2048, 8192), (1, 4100, 5000),
                                       (1, 16500, 16500)])
def test_few_rows_at_larger_tiles(batch, m, n):
    x = few_rows(m, n, 3, 1, 5)
    got = mi_adamw.newton_schulz(x if batch == 1 else x.expand(batch, m, n), precision="half")
    for y in (got if batch > 1 else [got]):
        assert error(y, x) <= limit(1, m)


def test_muon():
    """A step from zero weights without momentum is minus lr times the orthogonalised gradient."""
    shapes = [(768, 768), (300, 200), (150, 600)]
    params = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in shapes]
    for k, p in enumerate(params):
        p.grad = few_rows(*p.shape, 3, 1, k)
    mi_adamw.Muon(params, lr=1.0, momentum=0.0, nesterov=False, weight_decay=0.0).step()
    for p in params:
        got = -p.detach() / math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        assert error(got, p.grad) <= limit(1, min(p.shape)) + 2.0 ** -22
