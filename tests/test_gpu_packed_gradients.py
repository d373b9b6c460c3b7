"""GPU: gradients of packed attention where the gradient that arrives is small or large, or the sequences are long, against float64 as a
multiple of what rounding the exact results leaves."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def gradients(n, count, heads, key_heads, dim, dtype, size, keys=1.0, values=1.0):
    """``((got, exact, rounded), ...)`` of dq, dk and dv, float64; ``size`` of dout."""
    import sparse
    scale = dim ** -0.5
    q, k, v, dout = (x.to(dtype).cuda() for x in (normal(1, count * n, heads, dim), keys * normal(2, count * n, key_heads, dim),
                                                  values * normal(3, count * n, key_heads, dim), size * normal(4, count * n, heads, dim)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    offsets = torch.arange(0, count * n + 1, n, dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(sparse.packed_attention(*leaves, offsets, scale), leaves, dout)
    exact = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in leaves]
    hidden = ~torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for b in range(count):
        at = slice(b * n, b * n + n)
        for h in range(heads):
            g = h // (heads // key_heads)
            qd, kd, vd, dd = q[at, h].detach().double(), k[at, g].detach().double(), v[at, g].detach().double(), dout[at, h].double()
            p = (scale * qd @ kd.t()).masked_fill(hidden, -math.inf).softmax(-1)
            ds = scale * p * (dd @ vd.t() - (dd * (p @ vd)).sum(-1, keepdim=True))
            exact[0][at, h] = ds @ kd
            exact[1][at, g] += ds.t() @ qd
            exact[2][at, g] += p.t() @ dd
    return [(x.double(), e, e.to(dtype).double()) for x, e in zip(got, exact)]


def check(which, *args, **kw):
    """Roundings of the same relative size, of what is multiplied and of the result, give sqrt(2) of the result's alone, in any unit."""
    got, exact, rounded = gradients(*args, **kw)[which]
    assert torch.isfinite(got).all()
    assert (got - exact).norm() <= 1.1 * math.sqrt(2) * (rounded - exact).norm()


SIZES = [(40, 20, 4, 2), (700, 1, 4, 2), (4096, 1, 2, 1)]


@pytest.mark.parametrize("size", [1.0, 1e-1, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,count,heads,key_heads", SIZES)
def test_dq_of_small_gradients(n, count, heads, key_heads, dim, size):
    """dS of long sequences and small gradients lies below fp16's normal values."""
    check(0, n, count, heads, key_heads, dim, torch.float16, size)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [33, 700])
def test_dq_where_ds_is_beyond_the_type(n, dim):
    """A dS above 65504, and a dq below it."""
    check(0, n, 2, 2, 1, dim, torch.float16, 2000.0, keys=2.0 ** -9, values=60.0)
