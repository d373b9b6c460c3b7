"""GPU: gradients of packed attention where the gradient that arrives is small or large, or the sequences are long, against float64 as a
multiple of what rounding the exact results leaves."""
import math

import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def gradients(n, count, heads, key_heads, dim, dtype, size, queries=1.0, keys=1.0, values=1.0):
    """``((got, exact, rounded), ...)`` of dq, dk and dv, float64; ``size`` of dout."""
    import sparse
    scale = dim ** -0.5
    q, k, v, dout = (x.to(dtype).cuda() for x in (queries * normal(1, count * n, heads, dim), keys * normal(2, count * n, key_heads, dim),
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


@pytest.mark.parametrize("size", [1.0, 1e-1, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,count,heads,key_heads", SIZES)
def test_dk_of_small_gradients(n, count, heads, key_heads, dim, size):
    check(1, n, count, heads, key_heads, dim, torch.float16, size)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [33, 700])
def test_dk_where_ds_is_beyond_the_type(n, dim):
    check(1, n, 2, 2, 1, dim, torch.float16, 2000.0, queries=2.0 ** -9, values=60.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_long_sequences_in_bf16(dim):
    """Many tiles of both walks, sequences of a length that is no multiple of a tile."""
    for which in range(3):
        check(which, 2979, 2, 2, 1, dim, torch.bfloat16, 1.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_with_gradients_unlike_its_neighbours(dim):
    """Each key has a power of two of its own: one whose value row is 2^-12 of the others' keeps all bits of its dS, one whose row
    grows along the queries that see it is lifted less as it goes."""
    import sparse
    n = 600
    q, k, v, dout = (x.half().cuda() for x in (normal(1, n, 1, dim), normal(2, n, 1, dim), normal(3, n, 1, dim), 1e-3 * normal(4, n, 1, dim)))
    dout *= torch.exp2(torch.linspace(0, 12, n, device="cuda"))[:, None, None].half()       # later queries count for more
    v[::7] *= 2.0 ** -12
    offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dk = torch.autograd.grad(sparse.packed_attention(*leaves, offsets, dim ** -0.5), leaves, dout)[1][:, 0].double()
    want, bound = po.rows(*(to_np(t[:, 0]) for t in (q, k, v)), np.tril(np.ones((n, n), dtype=bool)), dim ** -0.5, "float16", to_np(dout[:, 0]),
                          lifted=True)["dk"]
    off = np.abs(dk.cpu().numpy() - want)
    assert (off <= bound).all()                 # every rounding at its worst: a key near the end has few queries, which may round alike


@pytest.mark.parametrize("n,count,heads,key_heads", SIZES[1:])
@pytest.mark.parametrize("dim", [64, 128])
def test_dk_of_tiny_ds_and_large_queries(dim, n, count, heads, key_heads):
    """dS of 1e-9 makes a dk of 1e-4.  Every other tile of keys begins with queries that do not see it: they say nothing of its dS."""
    check(1, n, count, heads, key_heads, dim, torch.float16, 1e-6, queries=2.0 ** 13, keys=2.0 ** -13)


@pytest.mark.parametrize("n,count,heads,key_heads", SIZES[1:])
@pytest.mark.parametrize("dim", [64, 128])
def test_dq_of_tiny_ds_and_large_keys(dim, n, count, heads, key_heads):
    check(0, n, count, heads, key_heads, dim, torch.float16, 1e-6, queries=2.0 ** -13, keys=2.0 ** 13)
