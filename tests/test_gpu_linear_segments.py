"""GPU: linear attention over the heads, segments and boundaries that its launches are made of, against the float64 oracle.

Tolerances are those of ``test_gpu_linear_attention``."""
import numpy as np
import pytest
import torch

from test_gpu_linear_attention import DTYPES, check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,group,dim", [([33, 2], 4, 1, 64), ([300, 70], 4, 2, 128), ([257, 0, 40], 8, 1, 64), ([260], 8, 3, 64),
                                                     ([40, 200, 31], 12, 1, 64), ([210, 5], 16, 1, 64), ([230], 6, 2, 128)])
def test_heads_in_sets(lengths, heads, group, dim, dtype):
    """Key heads are dealt to the chip's eight parts in sets of 8, 4, 2 or 1, whichever divides them."""
    x = inputs(lengths, heads, group, dim, dtype)
    check(x, run(x))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,dim", [([2000], 64), ([33, 1700, 96], 128), ([1537 + 96, 1537], 64)])
def test_more_boundaries_than_are_read_at_once(lengths, dim, dtype):
    """Segments of 96 tokens: up to 20 states between them, which the running sum reads 16 at a time, from and to given states."""
    x = inputs(lengths, 1, 1, dim, dtype)
    check(x, run(x))


def by_segments(x, segment, monkeypatch):
    """The call without native code, whose segments can be chosen."""
    from sparse import linear
    monkeypatch.setattr(linear._k.lib, "bsa_linear_attention_segment", lambda *sizes: segment)
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "states")]
    outs = linear.general(*leaves[:3], x["log_decay"], x["offsets"], x["scale"], leaves[3], True)
    found = dict(zip(("out", "last"), (t.detach() for t in outs)))
    found.update(zip(("dq", "dk", "dv", "dfirst"), torch.autograd.grad(outs, leaves, [x["dout"], x["dlast"]])))
    return found


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("segment", [32, 64, 544, 800, 1 << 20])
def test_every_length_of_segments(segment, dtype, monkeypatch):
    x = inputs([1250, 0, 3, 700], 2, 1, 64, dtype)
    check(x, by_segments(x, segment, monkeypatch))


@pytest.mark.parametrize("dtype", DTYPES)
def test_segments_with_many_boundaries(dtype, monkeypatch):
    """40 states between segments of 32 tokens, of two key heads with three query heads each."""
    x = inputs([1300, 35], 2, 3, 64, dtype)
    check(x, by_segments(x, 32, monkeypatch))


def test_a_batch_of_single_tokens_and_one_prompt():
    x = inputs([1] * 40 + [900] + [1] * 30, 2, 1, 64, torch.bfloat16)
    check(x, run(x))
