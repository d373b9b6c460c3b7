"""CPU: the packed-attention and cache oracle against mathematics, torch and differences."""
import numpy as np
import pytest
import torch
from scipy.special import softmax as scipy_softmax

from oracle import packed_oracle as po


def _operands(tokens, heads, key_heads, d, seed=0):
    rng = np.random.RandomState(seed)
    return rng.randn(tokens, heads, d), rng.randn(tokens, key_heads, d), rng.randn(tokens, key_heads, d), rng.randn(tokens, heads, d)


@pytest.mark.parametrize("causal", [True, False])
def test_every_sequence_is_textbook_attention(causal):
    q, k, v, _ = _operands(12, 4, 2, 16)
    got = po.packed(q, k, v, [1, 4, 4, 11], 0.3, causal, "float16")["out"][0]
    assert not got[0].any() and not got[11].any()
    for a, b in ((1, 4), (4, 11)):
        for h in range(4):
            s = 0.3 * q[a:b, h] @ k[a:b, h // 2].T
            if causal:
                s = np.where(np.tril(np.ones(s.shape, dtype=bool)), s, -np.inf)
            assert np.allclose(got[a:b, h], scipy_softmax(s, axis=-1) @ v[a:b, h // 2], atol=1e-13)


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_are_those_of_torch_and_of_differences(causal):
    q, k, v, dout = _operands(7, 4, 2, 8, seed=3)
    offsets, scale = [0, 3, 3, 7], 0.4
    found = po.packed(q, k, v, offsets, scale, causal, "bfloat16", dout)
    leaves = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    loss = 0
    for a, b in ((0, 3), (3, 7)):
        for h in range(4):
            s = scale * leaves[0][a:b, h] @ leaves[1][a:b, h // 2].t()
            if causal:
                s = s.masked_fill(~torch.ones(b - a, b - a, dtype=torch.bool).tril(), float("-inf"))
            loss = loss + (s.softmax(-1) @ leaves[2][a:b, h // 2] * torch.tensor(dout[a:b, h])).sum()
    for name, want in zip(("dq", "dk", "dv"), torch.autograd.grad(loss, leaves)):
        assert np.allclose(found[name][0], want.numpy(), atol=1e-12), name
    rng = np.random.RandomState(1)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        along, step = rng.randn(*x[i].shape), 1e-5
        ends = []
        for sign in (1, -1):
            moved = list(x)
            moved[i] = x[i] + sign * step * along
            ends.append((po.packed(*moved, offsets, scale, causal, "bfloat16")["out"][0] * dout).sum())
        assert abs((ends[0] - ends[1]) / (2 * step) - (found[name][0] * along).sum()) < 1e-7


def test_bounds_hold_for_rounded_probabilities():
    """A model of the arithmetic that the bounds are for: probabilities and results rounded to 16 bits."""
    q, k, v, _ = _operands(40, 1, 1, 64, seed=5)
    q, k, v = (x.astype(np.float16).astype(np.float64) for x in (q, k, v))
    value, bound = po.packed(q, k, v, [0, 40], 0.125, True, "float16")["out"]
    s = np.where(np.tril(np.ones((40, 40), dtype=bool)), 0.125 * q[:, 0] @ k[:, 0].T, -np.inf)
    p = scipy_softmax(s, axis=-1).astype(np.float16).astype(np.float64)
    got = (p @ v[:, 0]).astype(np.float16).astype(np.float64)
    assert (np.abs(got - value[:, 0]) <= bound[:, 0]).all()
    assert (bound < 0.02).all()                                 # and are no wider than a few roundings


def test_e4m3_is_the_nearest_value_of_the_type():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    table = np.unique(table[np.isfinite(table)])
    assert np.array_equal(po.e4m3(table), table)
    x = np.concatenate([np.linspace(-448, 448, 40001), np.linspace(-0.05, 0.05, 4001), (table[1:] + table[:-1]) / 2])
    # ties go to the even value, as in torch's conversion
    ties = (table[1:] + table[:-1]) / 2
    assert np.array_equal(po.e4m3(ties), torch.tensor(ties, dtype=torch.float32).to(torch.float8_e4m3fn).double().numpy())
    assert (np.abs(po.e4m3(x) - x) <= np.abs(x[:, None] - table[None]).min(1) + 1e-15).all()


@pytest.mark.parametrize("kind,bound,half", [("int8", 127.0, 0.5), ("e4m3", 448.0, 16.0)])
def test_quantised_rows(kind, bound, half):
    rng = np.random.RandomState(2)
    x = rng.randn(20, 64)
    x[3] = 0
    x[4, 7], x[5, 9] = np.inf, np.nan
    held, scale = po.quantise(x, kind)
    fine = [i for i in range(20) if i not in (4, 5)]
    assert np.isnan(scale[[4, 5]]).all() and not held[[3, 4, 5]].any() and scale[3] == 0
    assert np.abs(held).max() == bound
    assert (np.abs(held * scale[:, None] - x)[fine] <= half * scale[fine, None] * (1 + 1e-12)).all()


def test_cached_is_attention_over_everything():
    rng = np.random.RandomState(4)
    q, k, v = rng.randn(2, 3, 4, 16), rng.randn(2, 3, 2, 16), rng.randn(2, 3, 2, 16)
    lengths = [5, 0]
    keys, values = ([rng.randn(2, n, 16) for n in lengths] for _ in range(2))
    chain = np.tril(np.ones((2, 3, 3), dtype=bool))
    got, _ = po.cached(q, k, v, keys, values, None, lengths, chain, 0.25, "float16")
    for b, n in enumerate(lengths):
        for h in range(2):                                      # the last rows of causal attention over cache and new tokens
            whole_q = np.concatenate([np.zeros((n, 2, 16)), q[b, :, 2 * h:2 * h + 2]])
            whole = [np.concatenate([held[b][h], new[b, :, h]])[:, None] for held, new in ((keys, k), (values, v))]
            want = po.packed(whole_q, *whole, [0, n + 3], 0.25, True, "float16")["out"][0][n:]
            assert np.allclose(got[b, :, 2 * h:2 * h + 2], want, atol=1e-13)
    none = np.zeros((2, 3, 3), dtype=bool)
    assert not po.cached(q, k, v, keys, values, None, lengths, none, 0.25, "float16")[0][1].any()


def fp16(x):
    return np.asarray(x).astype(np.float16).astype(np.float64)


def test_bounds_of_lifted_ds_hold_for_it_and_not_for_ds_as_it_is():
    """Gradients of 1e-4: dS of a key is rounded times a power of two that brings its largest below 2^4, against dS as it is."""
    n, d, scale = 400, 64, 0.125
    rng = np.random.RandomState(6)
    q, k, v, dout = (fp16(size * rng.randn(n, d)) for size in (1, 1, 1, 1e-4))
    visible = np.tril(np.ones((n, n), dtype=bool))
    want, bound = po.rows(q, k, v, visible, scale, "float16", dout, lifted=True)["dk"]
    p = scipy_softmax(np.where(visible, scale * q @ k.T, -np.inf), axis=-1)
    ds = p * (dout @ v.T - (dout * (p @ v)).sum(-1, keepdims=True))
    lift = 2.0 ** (4 - np.frexp(np.abs(ds).max(0))[1])
    assert (np.abs(fp16(scale / lift[:, None] * (fp16(ds * lift).T @ q)) - want) <= bound).all()
    assert (np.abs(fp16(scale * (fp16(ds).T @ q)) - want) > bound).any()          # worst cases are summed: few elements pass them


def test_bounds_by_weight_hold_for_the_largest_weight_and_not_for_the_largest_scale():
    """One value row 2^15 times as large as the others and of no weight: the others' weights, rounded relative to the largest p t, and to
    the largest t."""
    n, d = 600, 16
    rng = np.random.RandomState(7)
    q, k, v = rng.randn(1, 1, 1, d), rng.randn(1, 1, 1, d), rng.randn(1, 1, 1, d)
    keys, y, t = rng.randn(1, n, d), rng.randint(-127, 128, (1, n, d)).astype(float), np.full((1, n), 2.0 ** -9)
    keys[0, 0], t[0, 0] = -30 * q[0, 0, 0] / np.linalg.norm(q), 2.0 ** 6
    want, bound = po.cached(q, k, v, [keys], [y * t[..., None]], [t], [n], np.ones((1, 1, 1), dtype=bool), 1.0, "float16", by_weight=True)
    s = np.append(keys[0], k[0, :, 0], 0) @ q[0, 0, 0]
    e, scales, rows = np.exp(s - s.max()), np.append(t[0], 1.0), np.append(y[0], v[0, :, 0], 0)

    def result(top):                                            # of the cached rows' weights; the new row's are relative to their own
        held = fp16(e[:n] * scales[:n] / top) * top
        new = fp16(e[n:])
        return fp16((held @ rows[:n] + new @ rows[n:]) / e.sum())

    assert (np.abs(result((e[:n] * scales[:n]).max() / 16) - want[0, 0, 0]) <= bound[0, 0, 0]).all()
    assert (np.abs(result(2 * t.max()) - want[0, 0, 0]) > bound[0, 0, 0]).any()
