"""GPU: ``packed_attention`` against the float64 oracle, within bounds that count roundings (oracle/packed_oracle.py)."""
import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def kind_of(dtype):
    return str(dtype).replace("torch.", "")


def offsets_of(lengths, first=0):
    return torch.tensor(np.cumsum([first] + list(lengths)), dtype=torch.int32, device="cuda")


def operands(seed, tokens, heads, key_heads, dim, dtype, grads=True):
    g = torch.Generator().manual_seed(seed)
    shapes = [(tokens, heads, dim), (tokens, key_heads, dim), (tokens, key_heads, dim)]
    made = [torch.randn(s, generator=g).to(dtype).cuda() for s in shapes]
    if grads:
        made = [t.requires_grad_(True) for t in made]
        made.append(torch.randn(shapes[0], generator=g).to(dtype).cuda())
    return made


def compare(got, want, what):
    value, bound = want
    off = np.abs(to_np(got) - value)
    worst = off - bound
    assert np.isfinite(to_np(got)).all(), what
    assert (worst <= 0).all(), f"{what}: {off.max()} where {bound.flat[worst.argmax()]} is allowed at {np.unravel_index(worst.argmax(), off.shape)}"


def run(lengths, heads, key_heads, dim, dtype, causal=True, scale=None, first=0, behind=0, seed=1):
    import sparse
    tokens = first + sum(lengths) + behind
    scale = dim ** -0.5 if scale is None else scale
    q, k, v, dout = operands(seed, tokens, heads, key_heads, dim, dtype)
    offsets = offsets_of(lengths, first)
    out = sparse.packed_attention(q, k, v, offsets, scale, causal)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    with torch.no_grad():
        assert torch.equal(sparse.packed_attention(q, k, v, offsets, scale, causal), out)
    want = po.packed(*(to_np(t) for t in (q, k, v)), to_np(offsets).astype(int), scale, causal, kind_of(dtype), to_np(dout))
    for got, name in zip((out,) + grads, ("out", "dq", "dk", "dv")):
        assert got.dtype == dtype
        compare(got, want[name], (name, lengths, heads, key_heads, dim, dtype, causal))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [2], [31, 32, 33], [63, 1, 64, 65, 0, 127], [128], [129, 0, 0, 200], [300, 5]])
def test_lengths(lengths, dim, dtype):
    run(lengths, 2, 2, dim, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (3, 1), (4, 2), (8, 1), (12, 4), (16, 16), (5, 5)])
def test_grouped_heads(heads, key_heads, dtype):
    run([70, 1, 140], heads, key_heads, 64, dtype)
    run([70, 1, 140], heads, key_heads, 128, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_every_token_sees_its_whole_sequence(dim, dtype):
    run([1, 40, 130, 64], 4, 2, dim, dtype, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(scale):
    run([130, 20], 2, 1, 64, torch.float16, scale=scale)
    run([130, 20], 2, 1, 128, torch.bfloat16, scale=scale, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    rng = np.random.RandomState(3)
    run(rng.randint(0, 9, 300).tolist(), 2, 1, 64, dtype)      # found by a search of more than one step
    run([1] * 65 + [0] * 70 + [3], 1, 1, 128, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first,behind", [(0, 1), (5, 0), (37, 200)])
def test_tokens_outside_every_sequence_are_not_read_and_give_zeros(first, behind, dtype):
    import sparse
    lengths, heads, key_heads, dim = [33, 0, 65], 4, 2, 128
    run(lengths, heads, key_heads, dim, dtype, first=first, behind=behind)
    tokens = first + sum(lengths) + behind
    q, k, v, dout = operands(2, tokens, heads, key_heads, dim, dtype)
    with torch.no_grad():
        for t in (q, k, v, dout):
            t[:first] = float("nan")
            t[tokens - behind:] = float("inf")
    out = sparse.packed_attention(q, k, v, offsets_of(lengths, first), 0.1)
    for t in (out,) + torch.autograd.grad(out, (q, k, v), dout):
        assert torch.isfinite(t).all()
        assert not t[:first].any() and not t[tokens - behind:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_value_that_is_no_number_reaches_only_tokens_that_see_it(where, bad, dim, dtype):
    """In the forward result: tokens before it, and other sequences, give what they give without it."""
    import sparse
    lengths, at = [50, 150, 9], 50 + 70
    q, k, v = operands(4, sum(lengths), 2, 1, dim, dtype, grads=False)
    clean = sparse.packed_attention(q, k, v, offsets_of(lengths), 0.1)
    {"k": k, "v": v}[where][at, 0, 5] = bad
    out = sparse.packed_attention(q, k, v, offsets_of(lengths), 0.1)
    sees = torch.zeros(sum(lengths), dtype=torch.bool)
    sees[at:50 + 150] = True
    assert torch.equal(out[~sees], clean[~sees])
    if where == "v":
        assert not torch.isfinite(out[sees][:, :, 5]).any()
        assert torch.equal(torch.cat([out[:, :, :5], out[:, :, 6:]], 2), torch.cat([clean[:, :, :5], clean[:, :, 6:]], 2))
    elif bad != bad:
        assert torch.isnan(out[sees]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["k", "v", "dout", "q"])
def test_a_value_that_is_no_number_reaches_only_gradients_that_depend_on_it(which, dtype):
    import sparse
    lengths, at, dim = [50, 150, 9], 50 + 70, 64
    q, k, v, dout = operands(5, sum(lengths), 2, 1, dim, dtype)

    def grads():
        out = sparse.packed_attention(q, k, v, offsets_of(lengths), 0.1)
        return torch.autograd.grad(out, (q, k, v), dout)

    clean = grads()
    with torch.no_grad():
        {"q": q, "k": k, "v": v, "dout": dout}[which][at] = float("nan")
    dq, dk, dv = grads()
    n = torch.arange(sum(lengths))
    inside = (n >= 50) & (n < 200)
    queries = (n == at) if which in ("q", "dout") else inside & (n >= at)          # whose own gradient it enters
    keys = inside & (n <= at) if which in ("q", "dout") else inside                # a query behind it sees every key before
    assert torch.equal(dq[~queries], clean[0][~queries])
    assert torch.equal(dk[~keys], clean[1][~keys])
    assert torch.equal(dv[~keys], clean[2][~keys])


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores of hundreds: the reference point of the exponentials has to move along a row."""
    import sparse
    lengths, dim = [260], 64
    q, k, v = operands(6, 260, 2, 2, dim, dtype, grads=False)
    k *= torch.linspace(0.5, 8, 260, device="cuda").to(dtype)[:, None, None]
    got = sparse.packed_attention(q, k, v, offsets_of(lengths), 1.0)
    compare(got, po.packed(*(to_np(t) for t in (q, k, v)), [0, 260], 1.0, True, kind_of(dtype))["out"], "out")


def test_slices_of_a_fused_projection_are_read_in_place():
    import sparse
    lengths, heads, key_heads, dim = [90, 41], 4, 2, 64
    g = torch.Generator().manual_seed(8)
    fused = torch.randn(131, (heads + 2 * key_heads) * dim, generator=g).half().cuda().requires_grad_(True)
    q, k, v = (t.view(131, -1, dim) for t in fused.split([heads * dim, key_heads * dim, key_heads * dim], 1))
    out = sparse.packed_attention(q, k, v, offsets_of(lengths), 0.125)
    apart = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    want = sparse.packed_attention(*apart, offsets_of(lengths), 0.125)
    assert torch.equal(out, want)
    dout = torch.randn(out.shape, generator=g).half().cuda()
    (got,) = torch.autograd.grad(out, fused, dout)
    want = torch.autograd.grad(want, apart, dout)
    assert torch.equal(got, torch.cat([t.reshape(131, -1) for t in want], 1))


def test_odd_strides_and_starts_are_copied():
    import sparse
    g = torch.Generator().manual_seed(9)
    flat = torch.randn(3 * 40 * 2 * 64 + 8, generator=g).half().cuda()
    odd = flat[1:1 + 40 * 2 * 64].view(40, 2, 64)                           # starts 2 bytes into its storage
    wide = torch.randn(40, 2, 67, generator=g).half().cuda()[:, :, :64]     # rows 67 values apart
    every = torch.randn(40, 2, 128, generator=g).half().cuda()[:, :, ::2]   # values 2 apart
    got = sparse.packed_attention(odd, wide, every, offsets_of([40]), 0.125)
    assert torch.equal(got, sparse.packed_attention(odd.clone(), wide.contiguous(), every.contiguous(), offsets_of([40]), 0.125))
    heads_first = torch.randn(2, 40, 64, generator=g).half().cuda().transpose(0, 1)
    got = sparse.packed_attention(heads_first, heads_first, heads_first, offsets_of([40]), 0.125)
    same = heads_first.contiguous()
    assert torch.equal(got, sparse.packed_attention(same, same, same, offsets_of([40]), 0.125))


def test_an_expanded_gradient_and_shared_leaf():
    import sparse
    x = torch.randn(70, 2, 64, generator=torch.Generator().manual_seed(10)).half().cuda().requires_grad_(True)
    out = sparse.packed_attention(x, x, x, offsets_of([70]), 0.125)
    (got,) = torch.autograd.grad(out.float().sum(), x)                      # the gradient of a sum is one value, expanded
    parts = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    out = sparse.packed_attention(*parts, offsets_of([70]), 0.125)
    want = torch.autograd.grad(out, parts, torch.ones_like(out))
    assert torch.allclose(got.float(), sum(t.float() for t in want), rtol=2 ** -9, atol=2 ** -12)


def test_gradient_of_queries_alone():
    import sparse
    q, k, v, dout = operands(11, 130, 4, 2, 128, torch.bfloat16)
    offsets = offsets_of([130])
    want = torch.autograd.grad(sparse.packed_attention(q, k, v, offsets, 0.1), (q, k, v), dout)
    (dq,) = torch.autograd.grad(sparse.packed_attention(q, k.detach(), v.detach(), offsets, 0.1), q, dout)
    assert torch.equal(dq, want[0])
    (dk,) = torch.autograd.grad(sparse.packed_attention(q.detach(), k, v.detach(), offsets, 0.1), k, dout)
    assert torch.equal(dk, want[1])


def test_gradients_against_differences():
    """The directional derivative of a random projection of the result, by central differences of the float64 oracle at the
    operands, against the gradients: off by at most their bounds and by what a step of 2^-8 leaves (third order)."""
    import sparse
    lengths, dim = [37, 20], 64
    q, k, v, dout = operands(12, 57, 2, 1, dim, torch.float16)
    out = sparse.packed_attention(q, k, v, offsets_of(lengths), 0.125)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    base, g = [to_np(t) for t in (q, k, v)], to_np(dout)
    want = po.packed(*base, [0, 37, 57], 0.125, True, "float16", g)
    rng = np.random.RandomState(0)
    for i, name in enumerate(("dq", "dk", "dv")):
        direction = rng.choice([-1.0, 1.0], base[i].shape)

        def value(step):
            moved = [b + step * direction if j == i else b for j, b in enumerate(base)]
            return (po.packed(*moved, [0, 37, 57], 0.125, True, "float16")["out"][0] * g).sum()

        h = 2.0 ** -8
        slope, coarse = (value(h) - value(-h)) / (2 * h), (value(2 * h) - value(-2 * h)) / (4 * h)
        allowed = want[name][1].sum() + 2 * abs(slope - coarse) + 1e-9
        assert abs((to_np(grads[i]) * direction).sum() - slope) <= allowed, name


def test_empty_batches():
    import sparse
    none = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    out = sparse.packed_attention(none, none, none, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 2, 64)
    out.sum().backward()
    q, k, v, dout = operands(13, 20, 2, 2, 64, torch.float16)
    for offsets in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((4,), 7, dtype=torch.int32, device="cuda")):
        out = sparse.packed_attention(q, k, v, offsets)
        assert not out.any()
        for t in torch.autograd.grad(out, (q, k, v), dout):
            assert not t.any()


def test_offsets_that_make_no_sense_stay_inside_the_operands():
    """They are taken as the nearer end of the tokens; a sequence that ends before it begins is empty."""
    import sparse
    q, k, v, dout = operands(14, 60, 2, 1, 64, torch.float16)
    for values, meant in (([0, 1000], [0, 60]), ([-5, 30, 10 ** 9], [0, 30, 60]), ([60, 0], [0, 0]),
                          ([-2 ** 31, 2 ** 31 - 1, 3], [0, 60, 60])):
        pair = []
        for o in (values, meant):
            out = sparse.packed_attention(q, k, v, torch.tensor(o, dtype=torch.int32, device="cuda"), 0.1)
            pair.append((out,) + torch.autograd.grad(out, (q, k, v), dout))
        torch.cuda.synchronize()
        if values != [60, 0] and values[-1] != 3:
            assert all(torch.equal(a, b) for a, b in zip(*pair))


def test_streams_and_graphs():
    import sparse
    lengths = [100, 3, 60]
    q, k, v, dout = operands(15, 200, 4, 2, 64, torch.bfloat16)
    offsets = offsets_of(lengths)
    want = sparse.packed_attention(q, k, v, offsets, 0.125)
    grads = torch.autograd.grad(want, (q, k, v), dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = sparse.packed_attention(q, k, v, offsets, 0.125)
        got = torch.autograd.grad(out, (q, k, v), dout)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, grads))

    # leaves of their own: a backward pass must not be captured while an eager graph of the same leaves lives
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse.packed_attention(*leaves, offsets, 0.125)
        got = torch.autograd.grad(out, leaves, dout)
    out = out.detach()
    for lengths in ([100, 3, 60], [1, 199, 0], [0, 0, 5]):        # the offsets are read at every replay
        offsets.copy_(offsets_of(lengths))
        for t in (out,) + got:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = sparse.packed_attention(q, k, v, offsets, 0.125)
        grads = torch.autograd.grad(want, (q, k, v), dout)
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, grads))


def test_the_same_bits_every_time():
    import sparse
    q, k, v, dout = operands(16, 700, 8, 2, 64, torch.float16)
    offsets = offsets_of([300, 1, 399])
    runs = []
    for _ in range(3):
        out = sparse.packed_attention(q, k, v, offsets, 0.125)
        runs.append((out,) + torch.autograd.grad(out, (q, k, v), dout))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_a_sequence_that_ends_before_it_begins_alone_gives_zeros():
    import sparse
    q, k, v, dout = operands(17, 60, 2, 1, 64, torch.float16)
    for values in ([60, 0], [2 ** 31 - 1, -2 ** 31], [40, 40], [60, 60, 0]):
        out = sparse.packed_attention(q, k, v, torch.tensor(values, dtype=torch.int32, device="cuda"), 0.1)
        for t in (out,) + torch.autograd.grad(out, (q, k, v), dout):
            assert not t.any(), values


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at", [3, 70, 390])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_an_infinite_key(bad, at, dim, dtype):
    """A query whose score of it is +inf has no softmax: NaN in its result, its dq and every gradient that it has a part in.  One whose score
    is -inf gives the key no weight: results and gradients as without it, but for dq's channel of the infinity, where 0 meets it.
    The rest against float64, as a multiple of what rounding the exact results leaves."""
    import math

    import sparse
    n, scale = 400, dim ** -0.5
    q, k, v, dout = operands(18, n, 1, 1, dim, dtype)
    with torch.no_grad():
        q[:, 0, 5] = q[:, 0, 5].abs() + 0.25
        q[300:, 0, 5] *= -1
        if at == 3:
            q[:60, 0, 5] *= -1
        k[at, 0, 5] = bad
    out = sparse.packed_attention(q, k, v, offsets_of([n]), scale)
    got = (out,) + torch.autograd.grad(out, (q, k, v), dout)
    qd, kd, vd, dd = (t[:, 0].detach().double() for t in (q, k, v, dout))
    seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    none = (seen[:, at] & (qd[:, 5] * bad > 0))               # queries without a softmax
    kd[at, 5] = 0
    s = (scale * qd @ kd.t()).masked_fill(~seen, -math.inf)
    s[:, at] = -math.inf                                      # of the others that see it
    p = s.softmax(-1)
    p[none] = 0
    ds = scale * p * (dd @ vd.t() - (dd * (p @ vd)).sum(-1, keepdim=True))
    below = torch.arange(n, device="cuda") <= (none.nonzero().max() if none.any() else -1)       # keys that a query of `none` sees
    for name, x, exact, lost in zip(("out", "dq", "dk", "dv"), got, (p @ vd, ds @ kd, ds.t() @ qd, p.t() @ dd), (none, none, below, below)):
        x = x[:, 0].detach()
        assert torch.isnan(x[lost]).all(), name
        keep = ~lost[:, None].expand_as(x)
        if name == "dq":
            keep = keep.clone()
            assert not torch.isfinite(x[seen[:, at], 5]).any(), name
            keep[seen[:, at], 5] = False
        assert torch.isfinite(x[keep]).all(), name
        off, rounded = (x.double() - exact)[keep].norm(), (exact.to(dtype).double() - exact)[keep].norm()
        assert off <= 1.1 * math.sqrt(2) * rounded + (0 if keep.any() else 1), (name, off, rounded)
