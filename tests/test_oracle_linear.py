"""CPU: the float64 restatement of linear attention against its closed sum, torch's autograd and differences."""
import numpy as np
import pytest
import torch

from oracle import linear_oracle as lo


def inputs(seed, lengths, heads, group, dim, states):
    r = np.random.RandomState(seed)
    tokens, count = sum(lengths), len(lengths)
    x = {"q": r.randn(tokens, heads * group, dim), "k": r.randn(tokens, heads, dim), "v": r.randn(tokens, heads, dim),
         "log_decay": -np.abs(r.randn(heads)) * 0.3, "offsets": np.concatenate([[0], np.cumsum(lengths)]), "scale": 0.37}
    x["log_decay"][0] = 0.0
    if states:
        x["first"] = r.randn(count, heads, dim, dim)
    return x


def closed(x, torch_out=False):
    """o_t = scale sum over s <= t of l^(t - s) (q_t . k_s) v_s + scale l^t q_t S_0, differentiable."""
    q, k, v = (torch.as_tensor(x[n]) for n in "qkv")
    first, group, outs, lasts = x.get("first"), q.size(1) // k.size(1), [], []
    for b in range(len(x["offsets"]) - 1):
        at = slice(x["offsets"][b], x["offsets"][b + 1])
        n = at.stop - at.start
        t = torch.arange(n, dtype=torch.float64)
        decay = torch.exp(torch.as_tensor(x["log_decay"])[:, None, None] * (t[:, None] - t[None, :])).tril()
        kk, vv = (y[at].repeat_interleave(group, 1).transpose(0, 1) for y in (k, v))
        p = torch.matmul(q[at].transpose(0, 1), kk.transpose(1, 2)) * decay.repeat_interleave(group, 0)
        o = torch.matmul(p, vv)
        last = torch.einsum("hn,nhd,nhe->hde", torch.exp(torch.as_tensor(x["log_decay"])[:, None] * (n - 1 - t)), k[at], v[at])
        if first is not None:
            f, grow = torch.as_tensor(first[b]), lambda e: torch.exp(torch.as_tensor(x["log_decay"])[:, None] * e)
            o = o + torch.matmul(q[at].transpose(0, 1), f.repeat_interleave(group, 0)) * grow(t + 1).repeat_interleave(group, 0)[..., None]
            last = last + grow(torch.tensor([float(n)], dtype=torch.float64))[..., None] * f
        outs.append(x["scale"] * o.transpose(0, 1))
        lasts.append(last)
    return torch.cat(outs), torch.stack(lasts)


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("lengths,heads,group,dim", [([5], 1, 1, 3), ([0, 1, 7, 0, 4], 2, 3, 4), ([33, 2], 3, 2, 5)])
def test_sums_and_gradients(lengths, heads, group, dim, states):
    x = inputs(1, lengths, heads, group, dim, states)
    leaves = [torch.as_tensor(x[n]).requires_grad_() for n in ("q", "k", "v") + (("first",) if states else ())]
    given = dict(x, **dict(zip(("q", "k", "v", "first"), leaves)))
    out, last = closed(given)
    r = np.random.RandomState(2)
    dout, dlast = r.randn(*out.shape), r.randn(*last.shape)
    grads = torch.autograd.grad((out, last), leaves, (torch.as_tensor(dout), torch.as_tensor(dlast)))
    found = lo.packed(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], x["scale"], x.get("first"), dout, dlast)
    for name, want in zip(("out", "last", "dq", "dk", "dv", "dfirst"), (out, last) + grads):
        assert np.allclose(found[name], want.detach().numpy(), rtol=1e-11, atol=1e-11), name


def test_gradients_against_differences():
    x = inputs(3, [6, 3], 2, 2, 3, True)
    r = np.random.RandomState(4)
    args = lambda: (x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], x["scale"], x["first"])
    base = lo.packed(*args())
    dout, dlast = r.randn(*base["out"].shape), r.randn(*base["last"].shape)
    found = lo.packed(*args(), dout, dlast)
    loss = lambda y: (y["out"] * dout).sum() + (y["last"] * dlast).sum()
    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("first", "dfirst")):
        for _ in range(5):
            at = tuple(r.randint(n) for n in x[name].shape)
            was = x[name][at]
            x[name][at] = was + 1e-5
            up = loss(lo.packed(*args()))
            x[name][at] = was - 1e-5
            down = loss(lo.packed(*args()))
            x[name][at] = was
            assert abs((up - down) / 2e-5 - found[grad][at]) < 1e-6, name


def test_steps_are_a_sequence():
    x = inputs(5, [9], 2, 2, 4, True)
    found = lo.packed(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], x["scale"], x["first"])
    states = np.concatenate([np.full((1, 2, 4, 4), 7.0), x["first"]])
    for t in range(9):
        out, states = lo.step(x["q"][t:t + 1], x["k"][t:t + 1], x["v"][t:t + 1], x["log_decay"], states, [1], x["scale"])
        assert np.allclose(out[0], found["out"][t], rtol=1e-12, atol=1e-12)
    assert np.allclose(states[1], found["last"][0]) and (states[0] == 7).all()


def test_outside_every_sequence_and_no_memory():
    x = inputs(6, [8], 2, 1, 4, False)
    found = lo.packed(x["q"], x["k"], x["v"], np.full(2, -np.inf), np.array([2, 5]), x["scale"], dout=np.ones((8, 2, 4)))
    inside = np.arange(2, 5)
    for name in ("out", "dq", "dk", "dv"):
        assert not found[name][[0, 1, 5, 6, 7]].any()
    want = x["scale"] * (x["q"] * x["k"]).sum(-1, keepdims=True) * x["v"]          # a token sees itself only
    assert np.allclose(found["out"][inside], want[inside])


@pytest.mark.parametrize("kind", ["float16", "bfloat16"])
def test_bounds_hold_for_rounded_arithmetic(kind):
    """A model of the arithmetic: weights rounded to 16 bits, sums in fp32."""
    x = inputs(7, [40], 1, 1, 64, False)
    to = torch.float16 if kind == "float16" else torch.bfloat16
    for n in "qkv":
        x[n] = torch.as_tensor(x[n]).to(to).double().numpy()
    t = np.arange(40)
    p = x["scale"] * np.exp(x["log_decay"][0] * (t[:, None] - t[None, :])) * (x["q"][:, 0] @ x["k"][:, 0].T)
    p = torch.as_tensor(np.tril(p)).float().to(to).float()
    out = torch.matmul(p, torch.as_tensor(x["v"][:, 0]).float()).to(to).double().numpy()
    want, off = lo.bounds(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], x["scale"], kind)["out"]
    assert (np.abs(out - want[:, 0]) <= off[:, 0]).all()
