"""GPU: linear attention where a value is no number, or far from one, and what must not suffer from it.

The oracle and its bounds are those of ``test_gpu_linear_attention``; what each test adds is derived beside it."""
import numpy as np
import pytest
import torch

from helpers import to_np
from test_gpu_linear_attention import DTYPES, check, inputs, run, want

pytestmark = pytest.mark.gpu


REACH = {"q": ("dk", "dv", "out", "dfirst"), "k": ("out", "dq", "dv", "last"), "v": ("out", "dq", "dk", "last"), "dout": ("dq", "dk", "dv", "dfirst")}


def reached(name, result, at, dim, tokens, end):
    """Where a value of token ``at``, head 0, place 3 of operand ``name`` goes: tokens (results), rows or columns (states)."""
    if result in ("last", "dfirst"):
        place = torch.zeros(dim, dim, dtype=torch.bool, device="cuda")
        if name in ("k", "q"):
            place[3] = True
        else:
            place[:, 3] = True
        return place
    token = torch.arange(tokens, device="cuda")
    if (name, result) in (("q", "out"), ("k", "dv"), ("v", "dk"), ("dout", "dq")):
        return token == at
    return (token >= at) & (token < end) if result in ("out", "dq") else token <= at


def check_reach(x, name, at, value, end):
    """A value that is no number in the first sequence, whose tokens end at ``end``: all that it does not reach is what the oracle makes
    of a zero in its place, and some of what it reaches is no number either."""
    dim, tokens = x["k"].size(2), x["k"].size(0)
    x[name] = x[name].clone()
    x[name][at, 0, 3] = value
    found = run(x)
    x[name][at, 0, 3] = 0
    for result, (exact, bound) in want(x).items():
        got, far = to_np(found[result]), np.zeros(exact.shape, bool)
        if result in REACH[name]:
            places = reached(name, result, at, dim, tokens, end).cpu().numpy()
            if result in ("last", "dfirst"):
                far[0, 0] = places
            else:
                far[places, 0 if result in ("dk", "dv") else slice(0, x["q"].size(1) // x["k"].size(1))] = True
            assert not np.isfinite(got[places] if far.ndim == 3 else got[0, 0][places]).all(), result
        off = np.abs(got - exact)[~far]
        assert (off <= bound[~far]).all(), (result, float(np.nanmax(off / np.maximum(bound[~far], 1e-300))), np.isnan(off).sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("small", ["states", "k", "q"])
@pytest.mark.parametrize("at", [5, 40, 97])
@pytest.mark.parametrize("group,dim", [(1, 64), (2, 128)])
def test_a_nan_beside_small_states(group, dim, at, small, name, dtype):
    """A token that meets the state and is no number says nothing about the state's size, which here is 1e-4 of what enters it: given so and met
    by the first chunk from either end, or kept so by small k (towards the front, by small q)."""
    x = inputs([100, 11], 1, group, dim, dtype)
    for n in {"states", "dlast", small}:
        x[n] = (x[n].float() * 1e-4).to(x[n].dtype)
    check_reach(x, name, at, float("nan"), 100)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
@pytest.mark.parametrize("name,at", [("v", 5), ("v", 97), ("k", 97), ("dout", 5), ("dout", 97), ("q", 5)])
@pytest.mark.parametrize("small", [None, "states", "k", "q"])
@pytest.mark.parametrize("group,dim,lengths", [(1, 64, [700, 3]), (2, 128, [100, 11])])
def test_an_infinity_has_its_column_to_itself(group, dim, lengths, small, name, at, value, dtype):
    """What closes a walk is as large as its parts can be; an infinity among it is not what they are fitted to.  It ruins a column (k, q: a row)
    of the states and the tokens that see it.  At 97 of 100, or at 697 of 700, tokens from the end, in the chunk that closes the
    states; at 5 in the one that closes their gradients."""
    x = inputs(lengths, 1, group, dim, dtype)
    for n in {"states", "dlast", small} if small else ():
        x[n] = (x[n].float() * 1e-4).to(x[n].dtype)
    check_reach(x, name, at if at < 50 else lengths[0] - 3, value, lengths[0])


@pytest.mark.parametrize("log_decay", [-0.01, -2.5, -40.0])
@pytest.mark.parametrize("mul", [1.0, 2.0 ** -12])
@pytest.mark.parametrize("lengths", [[70, 33, 1], [700]])
def test_large_given_states_in_fp16(lengths, mul, log_decay):
    """States of 1e35 come back as what fp32 makes of them, not as infinities of their powers of two, and what enters is there when their decay
    has made them small."""
    x = inputs(lengths, 2, 1, 64, torch.float16)
    x["log_decay"].fill_(log_decay)
    for n in ("states", "dlast"):
        x[n] *= 1e35
    for n in ("v", "dout"):
        x[n] = (x[n].float() * mul).half()
    check(x, run(x), norms=False)


@pytest.mark.parametrize("large", ["v", "dout"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[70, 33, 1], [700]])
def test_bf16_goes_as_far_as_fp32(lengths, dim, large):
    """Values of 2^112, and states and sums of them up to 2^124: a decay that is put off, 2^-16 a chunk, makes nothing larger."""
    x = inputs(lengths, 3, 2, dim, torch.bfloat16)
    x["log_decay"].fill_(-0.35)
    x[large] *= 2.0 ** 112
    x["states" if large == "v" else "dlast"] *= 2.0 ** 112
    check(x, run(x))


@pytest.mark.parametrize("lengths", [[70, 33, 1], [700]])
def test_large_given_states_in_bf16(lengths):
    """1e35, and e^-2.5 a token: of 38 tokens that is 2^-137, which fp32 has few bits of; of 6 and of 32 it has all."""
    x = inputs(lengths, 2, 1, 64, torch.bfloat16)
    x["log_decay"].fill_(-2.5)
    for n in ("states", "dlast"):
        x[n] *= 1e35
    for n in ("v", "dout"):
        x[n] *= 2.0 ** -12
    check(x, run(x), norms=False)


@pytest.mark.parametrize("small", ["v", "dout"])
@pytest.mark.parametrize("lengths", [[70, 33, 1], [700]])
@pytest.mark.parametrize("mul", [-75, -100, -115])
def test_small_values_in_bf16(mul, lengths, small):
    """What enters a state (of the gradients' walk: with the scale) is held at least 2^-5 as large as it is, as three parts of bf16, whose smallest
    step is 2^-133: a value of row r of the states is off by the sum of |k_t[r]| (of their gradients: |q_t[r]|) times 2^5 2^-134
    besides, and by 2^5 2^-150 for each of the 700 roundings of the state.  Of a result that is 2^-129 of its terms' factors, which are 2^-115 or more: within its unit."""
    x = inputs(lengths, 2, 1, 64, torch.bfloat16)
    state, key = {"v": ("last", "k"), "dout": ("dfirst", "q")}[small]
    for n in (small, {"v": "states", "dout": "dlast"}[small]):
        x[n] *= 2.0 ** mul
    more, offsets = dict.fromkeys(("out", "last", "dq", "dk", "dv", "dfirst"), 0.0), np.cumsum([0] + lengths)
    sums = np.stack([np.abs(to_np(x[key])[offsets[b]:offsets[b + 1]]).sum(0) for b in range(len(lengths))])
    more[state] = 2.0 ** -129 * sums[..., None] + 700 * 2.0 ** -145
    check(x, run(x), norms=False, more=more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("walk", ["out", "dq", "dv", "dk"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_large_weights_beside_no_numbers(value, walk, dtype):
    """Weights P of 2^12 are more than fp16 holds at P's usual size.  Tokens 0 to 3 (or 28 to 31, seen from the end) have them; a value that is no
    number in the same chunk, in a place that shares their lanes and that tokens next to them do not see, hides them from the sum that tells
    P's size, but those tokens' results are numbers."""
    x = inputs([32], 1, 1, 64, dtype, states=False)
    x["scale"] = 1.0
    x["log_decay"].zero_()
    b, c = {"out": ("k", "v"), "dq": ("v", "k"), "dv": ("q", "dout"), "dk": ("dout", "q")}[walk]
    large, at = (slice(0, 4), 8) if walk in ("out", "dq") else (slice(24, 28), 16)
    x[b][large] *= 512
    x[c] = (x[c].float() / 64).to(dtype)
    value_at = x[b][at, 0, 3].clone()
    x[b][at, 0, 3] = value
    found = run(x)[walk]
    x[b][at, 0, 3] = value_at
    exact, bound = want(x)[walk]
    clear = slice(0, at) if walk in ("out", "dq") else slice(at + 1, 32)
    assert (np.abs(to_np(found) - exact) <= bound)[clear].all()


@pytest.mark.parametrize("tokens", [5, 513, 2000])
def test_gradients_without_sequences(tokens):
    """Offsets of one entry: all tokens are padding, also where they would be several segments of a sequence."""
    import sparse
    x = inputs([tokens], 2, 1, 64, torch.float16, states=False)
    leaves = [x[n].requires_grad_() for n in "qkv"]
    out = sparse.packed_linear_attention(*leaves, x["log_decay"], x["offsets"][:1])
    for t in (out, *torch.autograd.grad(out, leaves, x["dout"])):
        assert not t.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["states", "dlast"])
@pytest.mark.parametrize("lengths,dim", [([70, 20], 64), ([300, 0], 128)])
def test_given_states_with_a_value_that_is_no_number(lengths, dim, name, value, dtype):
    """Row 3, column 5 of the first state: column 5 of the results, column 3 of dq, and its own place in the last state; likewise of the last
    state's gradient: column 5 of dv, column 3 of dk, its place in the first state's gradient."""
    x = inputs(lengths, 2, 2, dim, dtype)
    x[name][0, 0, 3, 5] = value
    found = run(x)
    x[name][0, 0, 3, 5] = 0
    columns, place = ({"out": 5, "dq": 3}, "last") if name == "states" else ({"dv": 5, "dk": 3}, "dfirst")
    for result, (exact, bound) in want(x).items():
        got, reached = to_np(found[result]), np.zeros(exact.shape, bool)
        if result in columns:
            reached[:lengths[0], slice(0, 2) if result in ("out", "dq") else 0, columns[result]] = True
        if result == place:
            reached[0, 0, 3, 5] = True
        assert not np.isfinite(got[reached]).any(), result
        assert (np.abs(got - exact) <= bound)[~reached].all(), result
