"""GPU: ``packed_linear_attention`` and ``linear_attention_step`` against the float64 oracle (oracle/linear_oracle.py).

Two tolerances.  Every value within the oracle's bound; and, for inputs of zero mean, the 2-norm of a result's error within ``unit`` of
the result's own: a result's rounding and that of the operand behind it (a weight, or the state) are independent and each is at most
``unit`` of its value, evenly distributed, so that its root mean square is at most unit / sqrt(3), and sqrt(2 / 3) < 1.  States in
fp32: 1e-6 (sums of up to 2000 terms whose roundings, 2^-24 each of the partial sum, are independent)."""
import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import linear_oracle as lo

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
NAMES = ("out", "last", "dq", "dk", "dv", "dfirst")


def kind_of(dtype):
    return str(dtype).replace("torch.", "")


def int32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def normal(seed, *shape, dtype=torch.float16, mul=1.0):
    return (mul * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def decays(heads, seed=0):
    """From a memory of a token and a half to one of thousands; the first head forgets nothing."""
    d = -torch.exp2(-0.5 - 11 * torch.rand(heads, generator=torch.Generator().manual_seed(seed)))
    d[0] = 0.0
    return d.cuda()


def inputs(lengths, heads, group, dim, dtype, states=True, seed=1, front=0, back=0, mul=1.0):
    tokens = front + sum(lengths) + back
    x = {"q": normal(seed, tokens, heads * group, dim, dtype=dtype), "k": normal(seed + 1, tokens, heads, dim, dtype=dtype),
         "v": normal(seed + 2, tokens, heads, dim, dtype=dtype, mul=mul), "log_decay": decays(heads, seed),
         "offsets": int32(front + np.concatenate([[0], np.cumsum(lengths)])), "scale": dim ** -0.5,
         "dout": normal(seed + 3, tokens, heads * group, dim, dtype=dtype, mul=mul)}
    if states:
        shape = (len(lengths), heads, dim, dim)
        x["states"] = normal(seed + 4, *shape, dtype=torch.float32, mul=4 * mul)
        x["dlast"] = normal(seed + 5, *shape, dtype=torch.float32, mul=mul)
    return x


def run(x, grads=True):
    import sparse
    leaves = {n: x[n].detach().requires_grad_(grads) for n in ("q", "k", "v", "states") if n in x}
    with_states = "states" in x
    got = sparse.packed_linear_attention(leaves["q"], leaves["k"], leaves["v"], x["log_decay"], x["offsets"], scale=x["scale"],
                                         states=leaves.get("states"), return_states=with_states)
    outs = got if with_states else (got,)
    found = dict(zip(("out", "last"), outs))
    if grads:
        made = torch.autograd.grad(outs, list(leaves.values()), [x["dout"], x["dlast"]] if with_states else [x["dout"]])
        found.update(zip(("dq", "dk", "dv", "dfirst"), made))
    return {n: t.detach() for n, t in found.items()}


def want(x, grads=True):
    given = [to_np(x[n]) for n in ("q", "k", "v", "log_decay")]
    first = to_np(x["states"]) if "states" in x else None
    more = (to_np(x["dout"]), to_np(x["dlast"]) if "dlast" in x else None) if grads else (None, None)
    return lo.bounds(*given, x["offsets"].cpu().numpy(), x["scale"], kind_of(x["q"].dtype), first, *more)


def check(x, found, grads=True, norms=True, more=None):
    unit = lo.UNIT[kind_of(x["q"].dtype)]
    for name, (value, bound) in want(x, grads).items():
        if name not in found:
            continue
        if more is not None:
            bound = bound + more[name]
        got = to_np(found[name])
        # fp16 has nothing between 65504 and infinity: from the middle on (65520) a result is rounded to infinity
        border = 65520.0 if found[name].dtype == torch.float16 else np.inf
        beyond = np.abs(value) - bound >= border
        assert (got[beyond] == np.sign(value[beyond]) * np.inf).all(), name
        inside = ~beyond & (np.abs(value) + bound < border)
        assert np.isfinite(got[inside]).all() and not np.isnan(got).any(), name
        off = np.abs(got - value)[inside]
        assert (off <= bound[inside]).all(), (name, float((off / np.maximum(bound[inside], 1e-300)).max()))
        size = np.linalg.norm(value[inside])
        if norms and size > 0 and inside.all():              # without the largest, what is left is where much cancels
            assert np.linalg.norm(off) <= (1e-6 if name in ("last", "dfirst") else unit) * size, (name, np.linalg.norm(off) / size)


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,group", [([1], 1, 1), ([31], 2, 1), ([32], 1, 3), ([33, 0, 1], 3, 1), ([64, 65, 2], 2, 2), ([130], 1, 1),
                                                 ([0], 2, 1), ([0, 0, 7, 96, 0], 5, 2)])
def test_results_and_gradients(lengths, heads, group, dim, dtype, states):
    x = inputs(lengths, heads, group, dim, dtype, states)
    check(x, run(x))


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,group", [([257], 2, 1), ([512, 1, 300], 1, 2), ([5, 1100, 0, 256, 255], 2, 1)])
def test_sequences_of_several_segments(lengths, heads, group, dim, dtype, states):
    x = inputs(lengths, heads, group, dim, dtype, states)
    check(x, run(x))


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_sequences_than_lanes(dtype):
    lengths = [int(n) for n in np.random.RandomState(3).randint(0, 40, 150)]
    x = inputs(lengths, 1, 2, 64, dtype)
    check(x, run(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("front,back", [(3, 0), (0, 5), (40, 33)])
def test_tokens_outside_every_sequence(front, back, dtype):
    x = inputs([20, 45], 2, 2, 64, dtype, front=front, back=back)
    for n in ("q", "k", "v", "dout"):
        x[n][:front] = float("nan")
        x[n][front + 65:] = float("inf")
    found = run(x)
    for n in ("out", "dq", "dk", "dv"):
        assert not found[n][:front].any() and not found[n][front + 65:].any(), n
    for n in ("q", "k", "v", "dout"):
        x[n][:front] = 0
        x[n][front + 65:] = 0
    check(x, found)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("log_decay", [0.0, -1e-6, -0.05, -3.0, -40.0, -float("inf")])
def test_decays(log_decay, dtype):
    x = inputs([300, 33], 2, 1, 64, dtype)
    x["log_decay"].fill_(log_decay)
    check(x, run(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("log_decay", [-8.0, -15.0, -25.0, -41.0])
@pytest.mark.parametrize("lengths", [[90, 33], [600]])
def test_what_enters_is_small_beside_a_state_that_goes(lengths, log_decay, dtype):
    """Towards the front every token's part comes with its own decay, to a state that still has dlast's size and is nothing after.
    Of 2^-59 the exponent alone is rounded by 2^-19, more than the 1e-6 of the norms."""
    x = inputs(lengths, 2, 1, 64, dtype)
    x["log_decay"].fill_(log_decay)
    check(x, run(x), norms=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("log_decay", [-0.1, -14.0])
@pytest.mark.parametrize("lengths", [[1, 2, 1], [33, 65]])
def test_states_of_few_tokens_have_their_small_columns_too(lengths, log_decay, dtype):
    """Each value of such a state is its own product: columns of 2^-12 of the others' size have bits of their own.

    In fp16 what enters a state in its last chunk travels times a power of two that brings the largest of it, X, to 2^13 .. 2^14, as a high part, cut,
    and a low part, rounded: it is off by 2^-22 of itself where the low part is a normal number and by half of fp16's smallest step,
    2^-25, where it is not, which is 2^-25 / 2^13 = 2^-38 of X.  Where the last token's k is zero or nearly so, what older tokens left is all there
    is, e^-14 a token of X: a value of row r may be off by the sum of |k_t[r]| times 2^-38 X besides (2^-37 below: both parts)."""
    x = inputs(lengths, 2, 1, 64, dtype)
    x["log_decay"].fill_(log_decay)
    for name in ("v", "dout"):
        x[name][..., ::2] *= 2.0 ** -12
    for name in ("states", "dlast"):
        x[name] *= 2.0 ** -12
    more = {name: 0.0 for name in ("out", "dq", "dk", "dv")}
    more.update({name: np.zeros((len(lengths), 2, 64, 1)) for name in ("last", "dfirst")})
    if dtype == torch.float16:
        offsets = np.cumsum([0] + lengths)
        for b, n in enumerate(lengths):
            ends, begins = slice(offsets[b] + (n - 1) // 32 * 32, offsets[b + 1]), slice(offsets[b], offsets[b] + min(n, 32))
            for h in range(2):
                q, k, v, dout = (to_np(x[name])[:, h] for name in ("q", "k", "v", "dout"))
                more["last"][b, h, :, 0] = 2.0 ** -37 * np.abs(v[ends]).max() * np.abs(k[ends]).sum(0)
                more["dfirst"][b, h, :, 0] = 2.0 ** -37 * np.abs(dout[begins]).max() * x["scale"] * np.exp(log_decay) * np.abs(q[begins]).sum(0)
    check(x, run(x), norms=False, more=more)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_of_different_sizes_in_one_chunk(dtype):
    """In fp16 P is an operand times 64 and a power of two that leaves the largest of a chunk at 4 or more: P_ts is off by 2^-11 of itself where it
    is a normal number and by half of fp16's smallest step, 2^-25, where it is not, 2^-27 of the chunk's largest.  A result is off by the sum
    of that times |c_s| besides, c being v, k, dout and q for out, dq, dv and dk."""
    x = inputs([90, 20], 2, 2, 64, dtype, states=False)
    x["log_decay"].fill_(-4.0)                               # a token's result is its own and its neighbours'
    size = torch.exp2(-(torch.arange(110, device="cuda") % 4).float() * 3.5).view(-1, 1, 1)
    for name in ("q", "v", "dout"):
        x[name] = (x[name].float() * size).to(dtype)
    more = {}
    q, k, v, dout = (to_np(x[name]) for name in ("q", "k", "v", "dout"))
    for name, (a, b, c) in {"out": (q, k, v), "dq": (dout, v, k), "dv": (k, q, dout), "dk": (v, dout, q)}.items():
        by_head = lambda y, h: y.reshape(110, 2, -1, 64)[:, h].transpose(1, 0, 2)          # [heads that share, tokens, 64]
        term = np.zeros(a.shape[:1] + (2, 1, 64))
        for h in range(2):
            most = abs(x["scale"]) * max(np.abs(one @ other.T).max() for one in by_head(a, h) for other in by_head(b, h))
            term[:, h, 0] = 2.0 ** -27 * most * np.abs(by_head(c, h)).sum((0, 1)) if dtype == torch.float16 else 0.0
        more[name] = np.broadcast_to(term, (110, 2, a.shape[1] // 2, 64)).reshape(a.shape)
    check(x, run(x), norms=False, more=more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("states", [False, True])
def test_small_values_behind_zeros(states, dtype):
    """Chunks of zeros say nothing about the size of what comes; 2^-13 of it has few bits in fp16 beside a state of nothing."""
    x = inputs([150, 70], 2, 1, 64, dtype, mul=2.0 ** -13)
    x["v"][:64] = 0
    x["dout"][-64:] = 0
    if states:
        x["states"].zero_()
        x["dlast"].zero_()
    check(x, run(x), norms=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(scale, dtype):
    x = inputs([70], 2, 1, 128, dtype)
    x["scale"] = scale
    check(x, run(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mul", [1e-4, 1e-2, 1e2, 1.5e3])
def test_small_and_large_values(mul, dtype):
    """v, dout and the states' own size: in fp16 the operands on the way would be subnormal, or infinite (a state of 1.5e3 times
    keys of 300 tokens is)."""
    x = inputs([300, 40], 2, 1, 64, dtype, mul=mul)
    norms = dtype == torch.bfloat16 or mul >= 1e-2           # fp16 results of 1e-4 are subnormal themselves
    check(x, run(x), norms=norms)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_whose_size_changes_along_the_sequence(dtype):
    x = inputs([200], 2, 1, 64, dtype)
    size = torch.ones(200, 1, 1, device="cuda")
    size[40:90] = 2.0 ** -9
    size[90:120] = 2.0 ** 9
    size[130:] = 2.0 ** -5
    x["v"] = (x["v"].float() * size).to(dtype)
    x["states"].zero_()
    check(x, run(x), norms=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_as_slices_and_odd_starts(dtype):
    x = inputs([37, 60], 2, 1, 64, dtype)
    tokens = x["q"].size(0)
    base = run(x)
    fused = torch.cat([x[n].reshape(tokens, -1) for n in "qkv"], 1)
    y = dict(x, **{n: fused[:, 128 * i:128 * (i + 1)].view(tokens, 2, 64) for i, n in enumerate("qkv")})
    odd = torch.empty(tokens * 128 + 3, dtype=dtype, device="cuda")[3:].view(tokens, 2, 64)
    odd.copy_(x["k"])
    turned = x["dout"].transpose(0, 1).contiguous().transpose(0, 1)
    shifted = torch.empty(x["states"].numel() + 1, device="cuda")[1:].view(x["states"].shape)
    shifted.copy_(x["states"])
    for other in (y, dict(x, k=odd), dict(x, dout=turned), dict(x, states=shifted), dict(x, dlast=x["dlast"].transpose(2, 3).contiguous().transpose(2, 3))):
        for n, t in run(other).items():
            assert torch.equal(t, base[n]), n


def test_a_broadcast_gradient():
    x = inputs([50], 2, 2, 64, torch.float16)
    x["dout"] = torch.ones(1, device="cuda", dtype=torch.float16).expand(x["q"].shape)
    check(x, run(x), norms=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name,at", [("v", 5), ("v", 40), ("k", 33), ("q", 7), ("dout", 50), ("v", 69)])
def test_values_that_are_no_numbers_reach_only_what_sees_them(name, at, value, dtype):
    x = inputs([30, 70, 11], 2, 2, 64, dtype)
    base = run(x)
    x[name][30 + at, 1, 3] = value
    found = run(x)
    token = torch.arange(111, device="cuda")
    seq = (token >= 30) & (token < 100)
    after, before = seq & (token >= 30 + at), seq & (token <= 30 + at)
    none = torch.zeros_like(seq)
    only = seq & (token == 30 + at)
    # tokens whose result may change, by operand
    reach = {"q": {"out": only, "dq": none, "dk": before, "dv": before}, "k": {"out": after, "dq": after, "dk": none, "dv": only},
             "v": {"out": after, "dq": after, "dk": only, "dv": none}, "dout": {"out": none, "dq": only, "dk": before, "dv": before}}[name]
    for n, may in reach.items():
        assert torch.equal(found[n][~may], base[n][~may]), n
        if may.any():
            assert not torch.isfinite(found[n][may].float()).all(), n
    head = 1 if name in "kv" else 0                          # query head 1 belongs to key head 0
    other = 1 - head
    for n in ("out", "dq"):
        assert torch.equal(found[n][:, 2 * other:2 * other + 2], base[n][:, 2 * other:2 * other + 2])
    for n in ("dk", "dv"):
        assert torch.equal(found[n][:, other], base[n][:, other])
    for n in ("last", "dfirst"):
        assert torch.equal(found[n][[0, 2]], base[n][[0, 2]])
    assert torch.isfinite(found["last"][1]).all() == (name in ("q", "dout"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,group,dim", [(1, 1, 64), (3, 2, 64), (2, 5, 128), (2, 1, 128), (1, 9, 64)])
def test_steps(heads, group, dim, dtype):
    import sparse
    batch, places = 7, 11
    q, k, v = normal(1, batch, heads * group, dim, dtype=dtype), normal(2, batch, heads, dim, dtype=dtype), normal(3, batch, heads, dim, dtype=dtype)
    states, log_decay = normal(4, places, heads, dim, dim, dtype=torch.float32), decays(heads)
    slots = int32([3, -1, 10, 0, 11, 2 ** 31 - 1, 7])
    before = states.clone()
    out = sparse.linear_attention_step(q, k, v, log_decay, states, slots, scale=0.3)
    exact, after = lo.step(*(to_np(t) for t in (q, k, v, log_decay, before)), slots.cpu().numpy(), 0.3)
    mags, mag_states = lo.step(*(np.abs(to_np(t)) for t in (q, k, v)), to_np(log_decay), np.abs(to_np(before)), slots.cpu().numpy(), 0.3)
    steps = (dim + 16) * lo.F32
    assert (np.abs(to_np(out) - exact) <= mags * steps + lo.UNIT[kind_of(dtype)] * np.abs(exact) + lo.TINY[kind_of(dtype)]).all()
    assert (np.abs(to_np(states) - after) <= 4 * lo.F32 * mag_states).all()
    rest = [i for i in range(places) if i not in (3, 10, 0, 7)]
    assert torch.equal(states[rest], before[rest]) and not out[[1, 4, 5]].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_and_steps_are_one_sequence(dtype):
    """States of packed prompts go on token by token; the same tokens in one call give the same."""
    import sparse
    lengths, more = [40, 1, 0, 300], 5
    x = inputs([n + more for n in lengths], 2, 2, 64, dtype, states=False)
    offsets = x["offsets"].cpu().numpy()
    whole, last = sparse.packed_linear_attention(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], scale=x["scale"], return_states=True)
    pick = np.concatenate([np.arange(o, o + n) for o, n in zip(offsets, lengths)])
    part = [x[n][torch.tensor(pick, device="cuda")] for n in "qkv"]
    out, states = sparse.packed_linear_attention(*part, x["log_decay"], int32(np.concatenate([[0], np.cumsum(lengths)])), scale=x["scale"],
                                                 return_states=True)
    value, bound = want(x, False)["out"]
    assert (np.abs(to_np(out) - value[pick]) <= bound[pick]).all()
    for t in range(more):
        at = torch.tensor([o + n + t for o, n in zip(offsets, lengths)], device="cuda")
        got = sparse.linear_attention_step(*(x[n][at] for n in "qkv"), x["log_decay"], states, int32(np.arange(4)), scale=x["scale"])
        assert (np.abs(to_np(got) - value[at.cpu().numpy()]) <= bound[at.cpu().numpy()]).all()
    assert (torch.linalg.norm(states - last) <= 2e-6 * torch.linalg.norm(last)).item()


def test_the_same_bits_in_every_call_and_on_every_stream():
    x = inputs([700, 30, 257], 2, 2, 128, torch.bfloat16)
    base = run(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side, side):
        with torch.cuda.stream(stream):
            again = run(x)
        stream.synchronize()
        for n, t in again.items():
            assert torch.equal(t, base[n]), n


def test_a_sequence_does_not_depend_on_the_batch():
    x = inputs([100, 33, 90], 2, 1, 64, torch.float16)
    base = run(x)
    alone = dict(x, **{n: x[n][100:133] for n in ("q", "k", "v", "dout")}, offsets=int32([0, 33]), states=x["states"][1:2], dlast=x["dlast"][1:2])
    found = run(alone)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(found[n], base[n][100:133]), n
    for n in ("last", "dfirst"):
        assert torch.equal(found[n][0], base[n][1]), n


def test_captured_calls_follow_what_changes_on_the_device():
    import sparse
    x = inputs([300, 20], 2, 1, 64, torch.float16)
    pool, slots = normal(9, 4, 2, 64, 64, dtype=torch.float32), int32([2, 0])
    token = [normal(i, 2, 2, 64) for i in (11, 12, 13)]

    def work():
        with torch.no_grad():
            out, last = sparse.packed_linear_attention(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], scale=x["scale"], states=x["states"],
                                                       return_states=True)
            return out, last, sparse.linear_attention_step(*token, x["log_decay"], pool, slots, scale=0.1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work()
    for offsets, at in (([0, 300, 320], [2, 0]), ([10, 64, 310], [1, -1]), ([0, 0, 320], [3, 2]), ([0, 300, 320], [0, 1])):
        x["offsets"].copy_(int32(offsets))
        slots.copy_(int32(at))
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        after = pool.clone()
        pool.copy_(before)
        for got, expected in zip(captured, work()):
            assert torch.equal(got, expected)
        assert torch.equal(after, pool)


def test_a_captured_training_step():
    import sparse
    x = inputs([300, 64], 2, 2, 64, torch.bfloat16)
    side = torch.cuda.Stream()
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "states")]

    def work():
        outs = sparse.packed_linear_attention(*leaves[:3], x["log_decay"], x["offsets"], scale=x["scale"], states=leaves[3], return_states=True)
        return torch.autograd.grad(outs, leaves, [x["dout"], x["dlast"]])
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work()
    for seed in (1, 2, 3):
        for t, shape_seed in zip(leaves, (seed, seed + 20, seed + 40, seed + 60)):
            with torch.no_grad():
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(shape_seed)))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in captured]
        fresh = run(dict(x, **dict(zip(("q", "k", "v", "states"), (t.detach().clone() for t in leaves)))))
        for got, n in zip(kept, ("dq", "dk", "dv", "dfirst")):
            assert torch.equal(got, fresh[n]), n


def test_gradients_of_parts_of_the_results():
    import sparse
    x = inputs([40, 300], 2, 1, 64, torch.float16)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "states")]
    out, last = sparse.packed_linear_attention(*leaves[:3], x["log_decay"], x["offsets"], scale=x["scale"], states=leaves[3], return_states=True)
    only = dict(zip(("dq", "dk", "dv", "dfirst"), torch.autograd.grad(out, leaves, x["dout"], retain_graph=True)))
    check(dict(x, dlast=torch.zeros_like(x["dlast"])), only)
    only = dict(zip(("dq", "dk", "dv", "dfirst"), torch.autograd.grad(last, leaves, x["dlast"], retain_graph=True)))
    check(dict(x, dout=torch.zeros_like(x["dout"])), only)
    with pytest.raises(RuntimeError, match="once_differentiable|twice|does not require grad"):
        g = torch.autograd.grad(out, leaves[:1], x["dout"], create_graph=True)[0]
        g.sum().backward()


def test_saved_tensors_that_come_back_from_elsewhere_and_the_call_without_native_code():
    import sparse
    from sparse import linear
    x = inputs([40, 300], 2, 2, 64, torch.float16)
    base = run(x)

    def gradients(call):
        leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "states")]
        outs = call(*leaves[:3], x["log_decay"], x["offsets"], x["scale"], leaves[3], True)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [x["dout"], x["dlast"]]))

    def spaced(t):                                           # the same values, in rows that are no multiple of 16 bytes apart
        return torch.cat([t, t[..., :3]], -1)[..., :t.size(-1)] if t.dim() == 3 else t.clone()
    found = [gradients(linear.general)]
    with torch.autograd.graph.save_on_cpu():
        found.append(gradients(sparse.packed_linear_attention))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spaced):
        found.append(gradients(sparse.packed_linear_attention))
    for made in found:
        for n, t in zip(("out", "last", "dq", "dk", "dv", "dfirst"), made):
            assert torch.equal(t, base[n]), n
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:1] if t.dtype == torch.float32 and t.dim() == 1 else t):
        with pytest.raises((ValueError, RuntimeError)):
            gradients(sparse.packed_linear_attention)


@pytest.mark.parametrize("odd", [False, True])
def test_a_step_between_a_pass_and_its_gradients_is_noticed(odd):
    import sparse
    x = inputs([40, 20], 2, 1, 64, torch.float16)
    leaves = [x[n].clone().requires_grad_() for n in "qkv"]
    pool = x["states"].clone()
    out = sparse.packed_linear_attention(*leaves, x["log_decay"], x["offsets"], scale=x["scale"], states=pool)
    rows = [x[n][:2] for n in "qkv"]
    if odd:                                                  # rows that the native call leaves to Python
        rows = [torch.cat([t, t[..., :3]], -1)[..., :64] for t in rows]
    sparse.linear_attention_step(*rows, x["log_decay"], pool, int32([1, 0]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(x["dout"])
    with torch.inference_mode():
        pool = x["states"].clone()
        sparse.linear_attention_step(*rows, x["log_decay"], pool, int32([1, 0]))


def call(**changed):
    import sparse
    given = dict(q=normal(1, 9, 4, 64), k=normal(2, 9, 2, 64), v=normal(3, 9, 2, 64), log_decay=decays(2), offsets=int32([0, 4, 9]), scale=0.125)
    return sparse.packed_linear_attention(**{**given, **changed})


@pytest.mark.parametrize("changed,error,needle", [
    (dict(q=lambda: normal(1, 9, 4, 64).float()), TypeError, "float16 or all bfloat16"),
    (dict(k=lambda: normal(1, 9, 2, 64).cpu()), ValueError, "same GPU"),
    (dict(q=lambda: normal(1, 9, 4, 80)), ValueError, "head dim"),
    (dict(q=lambda: normal(1, 9, 3, 64)), ValueError, "cannot share"),
    (dict(offsets=lambda: int32([0, 9]).long()), ValueError, "int32"),
    (dict(offsets=lambda: int32([])), ValueError, "one entry more"),
    (dict(log_decay=lambda: decays(4)), ValueError, "log_decay must"),
    (dict(log_decay=lambda: decays(2).half()), ValueError, "log_decay must"),
    (dict(log_decay=lambda: decays(4)[::2]), ValueError, "log_decay must"),
    (dict(log_decay=lambda: -0.5), ValueError, "log_decay must"),
    (dict(log_decay=lambda: decays(2).cpu()), ValueError, "GPU of the operands"),
    (dict(log_decay=lambda: decays(2).requires_grad_()), RuntimeError, "not differentiable"),
    (dict(states=lambda: torch.zeros(2, 2, 64, 64, device="cuda").half()), ValueError, "states must"),
    (dict(states=lambda: torch.zeros(1, 2, 64, 64, device="cuda")), ValueError, "states must"),
    (dict(states=lambda: torch.zeros(2, 4, 64, 64, device="cuda")), ValueError, "states must"),
    (dict(states=lambda: torch.zeros(2, 2, 64, 64)), ValueError, "states must live"),
    (dict(states=lambda: 0), ValueError, "states must"),
])
def test_refusals(changed, error, needle):
    with pytest.raises(error, match=needle):
        call(**{name: make() for name, make in changed.items()})


def step_call(**changed):
    import sparse
    given = dict(q=normal(1, 3, 4, 64), k=normal(2, 3, 2, 64), v=normal(3, 3, 2, 64), log_decay=decays(2),
                 states=torch.zeros(5, 2, 64, 64, device="cuda"), slots=int32([0, 1, 2]), scale=0.125)
    return sparse.linear_attention_step(**{**given, **changed})


@pytest.mark.parametrize("changed,error,needle", [
    (dict(q=lambda: normal(1, 3, 4, 64).float()), TypeError, "float16 or all bfloat16"),
    (dict(v=lambda: normal(1, 2, 2, 64)), ValueError, "belong together"),
    (dict(slots=lambda: int32([0, 1])), ValueError, "3 sequences"),
    (dict(slots=lambda: int32([0, 1, 2]).long()), ValueError, "slots must"),
    (dict(states=lambda: torch.zeros(5, 2, 64, 64, device="cuda").half()), ValueError, "states must"),
    (dict(states=lambda: torch.zeros(5, 2, 64, 128, device="cuda")[..., ::2]), ValueError, "updated in place"),
    (dict(states=lambda: torch.zeros(5 * 2 * 64 * 64 + 1, device="cuda")[1:].view(5, 2, 64, 64)), ValueError, "updated in place"),
    (dict(states=lambda: torch.zeros(5, 2, 64, 64)), ValueError, "states must live"),
    (dict(states=lambda: torch.zeros(5, 2, 64, 64, device="cuda").requires_grad_()), RuntimeError, "not differentiable"),
    (dict(q=lambda: normal(1, 3, 4, 64).requires_grad_()), RuntimeError, "not differentiable"),
    (dict(log_decay=lambda: decays(3)), ValueError, "log_decay must"),
])
def test_step_refusals(changed, error, needle):
    with pytest.raises(error, match=needle):
        step_call(**{name: make() for name, make in changed.items()})


def test_nothing_to_do():
    import sparse
    states = normal(1, 2, 2, 64, 64, dtype=torch.float32)
    empty = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    out, last = sparse.packed_linear_attention(empty, empty, empty, decays(2), int32([0, 0, 0]), states=states, return_states=True)
    assert out.shape == empty.shape and torch.equal(last, states)
    x = normal(2, 5, 2, 64)
    out, last = sparse.packed_linear_attention(x, x, x, decays(2), int32([3]), return_states=True)
    assert not out.any() and last.shape == (0, 2, 64, 64)
    assert sparse.linear_attention_step(empty, empty, empty, decays(2), states, int32([])).shape == empty.shape
    idle = sparse.linear_attention_step(x, x, x, decays(2), states[:0], int32([0, 1, -1, 5, 2]))
    assert not idle.any()
    q = x.clone().requires_grad_()
    grads = torch.autograd.grad(sparse.packed_linear_attention(q, x, x, decays(2), int32([3])), q, x)
    assert not grads[0].any()
