"""GPU: how packed attention, the cache and attention over it are called: refusals, other routes to the same launch, copies of a
cache, calls at once, and what autograd may ask of them."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def normal(seed, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def packed_call(**changed):
    import sparse
    given = dict(q=normal(1, 9, 4, 64), k=normal(2, 9, 2, 64), v=normal(3, 9, 2, 64), offsets=int32([0, 4, 9]), scale=0.125)
    return sparse.packed_attention(**{**given, **changed})


@pytest.mark.parametrize("changed,error,needle", [
    (dict(q=lambda: normal(1, 9, 4, 64).float()), TypeError, "float16 or all bfloat16"),
    (dict(v=lambda: normal(1, 9, 2, 64, dtype=torch.bfloat16)), TypeError, "float16 or all bfloat16"),
    (dict(k=lambda: normal(1, 9, 2, 64).cpu()), ValueError, "same GPU"),
    (dict(q=lambda: normal(1, 1, 9, 4, 64)), ValueError, "3 dimensions"),
    (dict(q=lambda: normal(1, 9, 4, 80)), ValueError, "head dim"),
    (dict(k=lambda: normal(1, 8, 2, 64)), ValueError, "belong together"),
    (dict(q=lambda: normal(1, 9, 3, 64)), ValueError, "cannot share"),
    (dict(offsets=lambda: int32([0, 9]).long()), ValueError, "int32"),
    (dict(offsets=lambda: int32([[0, 9]])), ValueError, "int32"),
    (dict(offsets=lambda: int32([0, 9]).cpu()), ValueError, "GPU of the operands"),
    (dict(offsets=lambda: int32([0, 0, 9, 9])[::2]), ValueError, "contiguous"),
    (dict(offsets=lambda: int32([])), ValueError, "one entry more"),
])
def test_packed_refusals(changed, error, needle):
    with pytest.raises(error, match=needle):
        packed_call(**{name: make() for name, make in changed.items()})


def new_cache(held=torch.int8, pages=6, page=32):
    import sparse
    cache = sparse.KeyValueCache(pages, 2, 64, dtype=held, page=page)
    dtype = torch.float16 if held.itemsize == 1 else held
    rows = [normal(i, pages * page, 2, 64, dtype=dtype) for i in (5, 6)]
    cache.write(*rows, torch.arange(pages * page, dtype=torch.int32, device="cuda"))
    return cache


def cached_call(cache=None, **changed):
    import sparse
    given = dict(q=normal(1, 2, 3, 4, 64), k=normal(2, 2, 3, 2, 64), v=normal(3, 2, 3, 2, 64), cache=cache or new_cache(),
                 pages=int32([[0, 3, 1], [5, 2, 0]]), lengths=int32([70, 33]), tree=None, scale=0.125)
    return sparse.cached_attention(**{**given, **changed})


@pytest.mark.parametrize("changed,error,needle", [
    (dict(q=lambda: normal(1, 2, 3, 4, 64).float()), TypeError, "float16 or all bfloat16"),
    (dict(q=lambda: normal(1, 6, 4, 64)), ValueError, "4 dimensions"),
    (dict(k=lambda: normal(1, 2, 3, 4, 64)), ValueError, "belong together"),
    (dict(k=lambda: normal(1, 2, 3, 1, 64), v=lambda: normal(1, 2, 3, 1, 64)), ValueError, "does not fit a cache"),
    (dict(pages=lambda: int32([0, 3])), ValueError, "pages must be"),
    (dict(pages=lambda: int32(3)), ValueError, "pages must be"),
    (dict(pages=lambda: int32([[0, 3, 1]])), ValueError, "2 sequences"),
    (dict(pages=lambda: int32([[0, 3, 1], [5, 2, 0]]).long()), ValueError, "pages must be"),
    (dict(lengths=lambda: int32([70, 33]).cpu()), ValueError, "GPU of the operands"),
    (dict(lengths=lambda: int32([70, 33, 1])), ValueError, "lengths"),
    (dict(tree=lambda: torch.ones(3, 3, device="cuda")), ValueError, "tree must be bool"),
    (dict(tree=lambda: torch.ones(2, 2, dtype=torch.bool, device="cuda")), ValueError, "tree must be bool"),
    (dict(tree=lambda: torch.ones(3, 3, 3, dtype=torch.bool, device="cuda")), ValueError, "tree must be bool"),
    (dict(tree=lambda: torch.ones(3, 3, dtype=torch.bool)), ValueError, "tree must be bool"),
    (dict(tree=lambda: [[True] * 3] * 3), ValueError, "tree must be bool"),
    (dict(q=lambda: normal(1, 1, 1025, 2, 64), k=lambda: normal(1, 1, 1025, 2, 64), v=lambda: normal(1, 1, 1025, 2, 64),
          pages=lambda: int32([[0]]), lengths=lambda: int32([1])), ValueError, "at most 1024"),
    (dict(cache=lambda: new_cache(torch.bfloat16)), TypeError, "attended to in that type"),
])
def test_cached_refusals(changed, error, needle):
    with pytest.raises(error, match=needle):
        cached_call(**{name: make() for name, make in changed.items()})


def test_cache_refusals():
    cache, rows = new_cache(), normal(1, 4, 2, 64)
    for args, error, needle in (
            ((rows.float(), rows, int32([0, 1, 2, 3])), TypeError, "float16 or both bfloat16"),
            ((rows, rows.bfloat16(), int32([0, 1, 2, 3])), TypeError, "float16 or both bfloat16"),
            ((rows[:, :1], rows[:, :1], int32([0, 1, 2, 3])), ValueError, r"must be \[tokens, 2, 64\]"),
            ((rows, rows[:3], int32([0, 1, 2, 3])), ValueError, "must be"),
            ((rows, rows.cpu(), int32([0, 1, 2, 3])), ValueError, "cache's GPU"),
            ((rows, rows, int32([0, 1, 2])), ValueError, "4 rows and 3 slots"),
            ((rows, rows, int32([0, 1, 2, 3]).long()), ValueError, "slots must be"),
            ((rows, rows, [0, 1, 2, 3]), ValueError, "slots must be")):
        with pytest.raises(error, match=needle):
            cache.write(*args)
    for args, error, needle in (((int32([0]), torch.float64), TypeError, "read as"), ((int32([[0]]), torch.float16), ValueError, "slots must be"),
                                ((int32([0]).cpu(), torch.float16), ValueError, "GPU of the operands")):
        with pytest.raises(error, match=needle):
            cache.read(*args)
    with pytest.raises(TypeError, match="takes rows of that type"):
        new_cache(torch.bfloat16).write(rows, rows, int32([0, 1, 2, 3]))
    with pytest.raises(AttributeError):
        cache.keys = rows


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn, torch.float16])
@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_a_copy_of_a_cache_is_its_own(how, held):
    cache = new_cache(held)
    other = copy.deepcopy(cache) if how == "deepcopy" else pickle.loads(pickle.dumps(cache))
    want = cached_call(cache)
    assert torch.equal(cached_call(other), want)
    slots = torch.arange(192, dtype=torch.int32, device="cuda")
    other.write(*(torch.zeros(192, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2)), slots)
    assert torch.equal(cached_call(cache), want)
    assert not other.read(slots, torch.float32)[0].any() and cache.read(slots, torch.float32)[0].any()


def test_the_route_without_native_host_code_makes_the_same_launch():
    import sparse
    cache, number = new_cache(), np.float64(0.125)             # a scale of another type is looked at in Python
    tree = torch.rand(2, 3, 3, generator=torch.Generator().manual_seed(1)).cuda() < 0.5
    for kw in (dict(), dict(tree=tree), dict(tree=tree[0])):
        assert torch.equal(cached_call(cache, **kw), cached_call(cache, scale=number, **kw))
    spread = normal(8, 3, 3, 2, 64).transpose(1, 2)[1:]        # strides out of order
    assert torch.equal(cached_call(cache, k=spread.transpose(1, 2)), cached_call(cache, k=spread.transpose(1, 2).contiguous()))
    leaves = [normal(i, 9, h, 64).requires_grad_() for i, h in ((1, 4), (2, 2), (3, 2))]
    dout = normal(4, 9, 4, 64)
    runs = []
    for scale in (0.125, number):
        out = sparse.packed_attention(*leaves, int32([0, 4, 9]), scale)
        runs.append((out.detach(),) + torch.autograd.grad(out, leaves, dout))
        assert out.grad_fn is not None
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    with torch.no_grad():
        assert all(torch.equal(packed_call(scale=s), runs[0][0]) for s in (0.125, number))


def test_gradients_are_not_differentiable_again():
    q = normal(1, 9, 4, 64).requires_grad_()
    for scale in (0.125, np.float64(0.125)):
        out = packed_call(q=q, scale=scale)
        grad, = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.float().sum().backward()


def test_an_operand_changed_in_place_is_noticed():
    q = normal(1, 9, 4, 64).requires_grad_()
    k = normal(2, 9, 2, 64)
    for scale in (0.125, np.float64(0.125)):
        out = packed_call(q=q, k=k, scale=scale)
        k.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwad
    with fwad.dual_level():
        q = fwad.make_dual(normal(1, 9, 4, 64), normal(2, 9, 4, 64))
        with pytest.raises((RuntimeError, NotImplementedError)):
            packed_call(q=q)
    packed_call()


def test_calls_at_once_on_two_streams():
    """Chunks of long sequences go through workspaces: every call has its own."""
    import sparse
    cache = new_cache(pages=64)
    pages = torch.stack([torch.randperm(64, generator=torch.Generator().manual_seed(i)) for i in range(2)]).int().cuda()
    calls = [dict(cache=cache, pages=pages, lengths=int32(lengths), q=normal(i, 2, 3, 4, 64)) for i, lengths in enumerate(([2048, 900], [17, 2000]))]
    want = [cached_call(**kw) for kw in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(cached_call(**calls[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_a_page_may_belong_to_several_sequences_and_come_twice():
    """Shared prefixes: what is seen is what the table says, each time that it says it."""
    cache = new_cache(torch.float16)
    twice = cached_call(cache, pages=int32([[2, 2, 1], [2, 2, 1]]), lengths=int32([64, 64]))
    spread = new_cache(torch.float16)
    for name in ("keys", "values"):
        getattr(spread, name)[4].copy_(getattr(cache, name)[2])
    assert torch.equal(twice, cached_call(spread, pages=int32([[2, 4, 1], [4, 2, 0]]), lengths=int32([64, 64])))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,count", [(700, 1), (40, 20)])
def test_gradients_lose_no_more_than_the_rounding_of_ds(n, count, dim, dtype):
    """Error of dq and dk against float64, as a multiple of what rounding the exact ones would leave.  Two roundings of the same relative
    size, of dS and of the result, give sqrt(2); delta from a rounded result would move all of a row of dS alike (measured: 1.6)."""
    import sparse
    heads, key_heads, scale = 4, 2, dim ** -0.5
    q, k, v = (normal(i, count * n, h, dim, dtype=dtype).requires_grad_() for i, h in ((1, heads), (2, key_heads), (3, key_heads)))
    dout = normal(4, count * n, heads, dim, dtype=dtype)
    offsets = torch.arange(0, count * n + 1, n, dtype=torch.int32, device="cuda")
    dq, dk = torch.autograd.grad(sparse.packed_attention(q, k, v, offsets, scale), (q, k), dout)
    # [count, heads, n, dim]
    apart = lambda t: t.detach().cpu().double().view(count, n, -1, dim).transpose(1, 2)
    qd, kd, vd, dd = (apart(t) for t in (q, k, v, dout))
    kd, vd = (t.repeat_interleave(heads // key_heads, 1) for t in (kd, vd))
    s = (scale * qd @ kd.transpose(2, 3).contiguous()).masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -math.inf)
    p = s.softmax(-1)
    ds = scale * p * (dd @ vd.transpose(2, 3).contiguous() - (dd * (p @ vd)).sum(-1, keepdim=True))
    exact_q = ds @ kd
    exact_k = (ds.transpose(2, 3).contiguous() @ qd).view(count, key_heads, -1, n, dim).sum(2)
    for got, exact in ((dq, exact_q), (dk, exact_k)):
        rounded = exact.to(dtype).double()
        assert (apart(got) - exact).norm() <= 1.1 * math.sqrt(2) * (rounded - exact).norm()


def test_calls_without_gradients_refuse_operands_that_autograd_follows():
    """A result without history would cut a training loop off from them without a word."""
    import torch.autograd.forward_ad as fwad
    cache, rows, slots = new_cache(), normal(1, 4, 2, 64), int32([0, 1, 2, 3])
    shapes = dict(q=(2, 3, 4, 64), k=(2, 3, 2, 64), v=(2, 3, 2, 64))
    for name, shape in shapes.items():
        leaf = normal(1, *shape).requires_grad_()
        for operand in (leaf, leaf * 1, (leaf * 1).transpose(0, 1).contiguous().transpose(0, 1)):
            with pytest.raises(RuntimeError, match="cached_attention is not differentiable"):
                cached_call(cache, **{name: operand})
        with torch.no_grad():
            want = cached_call(cache, **{name: leaf})
        assert torch.equal(cached_call(cache, **{name: leaf.detach()}), want) and not want.requires_grad
        with fwad.dual_level():
            with pytest.raises(RuntimeError, match="not differentiable"):
                cached_call(cache, **{name: fwad.make_dual(leaf.detach(), leaf.detach().clone())})
    before = cache.read(slots, torch.float32)
    leaf = (2 * rows).requires_grad_()
    for k, v in ((leaf, rows), (rows, leaf), (leaf * 1, rows)):
        with pytest.raises(RuntimeError, match="write is not differentiable"):
            cache.write(k, v, slots)
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="not differentiable"):
            cache.write(fwad.make_dual(rows, 2 * rows), rows, slots)
    assert all(torch.equal(a, b) for a, b in zip(before, cache.read(slots, torch.float32)))
    with torch.no_grad():
        cache.write(leaf, rows, slots)
    assert not torch.equal(before[0], cache.read(slots, torch.float32)[0])


def test_saved_tensors_that_hooks_give_back():
    """As they were after a stay on the host, in another layout: the same gradients; as something else: refused before any launch."""
    leaves = [normal(i, 9, h, 64).requires_grad_() for i, h in ((1, 4), (2, 2), (3, 2))]
    dout = normal(4, 9, 4, 64)

    def grads(pack, unpack, scale):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = packed_call(q=leaves[0], k=leaves[1], v=leaves[2], scale=scale)
        return torch.autograd.grad(out, leaves, dout)

    spread = lambda t: torch.stack([t, t], -1)[..., 0] if t.dtype != torch.int32 else t        # every other value
    for scale in (0.125, np.float64(0.125)):
        want = grads(lambda t: t, lambda t: t, scale)
        for pack, unpack in ((lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, spread)):
            assert all(torch.equal(a, b) for a, b in zip(grads(pack, unpack, scale), want))
        for at in range(7):                                    # one of the saved tensors
            for change in (lambda t: t.cpu(), lambda t: t[:-1] if t.dtype != torch.int32 else t[None], lambda t: t.to(torch.float64)):
                count = iter(range(7))
                with pytest.raises((ValueError, TypeError)):
                    grads(lambda t: (next(count), t), lambda x: change(x[1]) if x[0] == at else x[1], scale)
