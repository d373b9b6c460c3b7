"""CPU: what linear attention, its step, the page table and copies of pages ask of a call before anything is launched."""
import ctypes

import pytest

P = 0x1000  # any non-null address, a multiple of 16
F16, BF16, F32, I8, E4M3 = 1, 2, 0, 3, 4


@pytest.fixture(scope="module")
def k():
    import sparse.kernel as kernel
    return kernel


def refused(k, code, *needles):
    message = k.lib.bsa_last_error().decode()
    assert code in (-1, -3) and all(n in message for n in needles), (code, message)


def strides(n, **changed):
    values = [512, 64] * (n // 2 + 1)
    for at, value in changed.items():
        values[int(at[1:])] = value
    return (ctypes.c_int64 * n)(*values[:n])


def forward(k, dtype=F16, q=P, kk=P, v=P, out=P, decay=P, offsets=P, first=None, last=None, states=None, size=0, segment=256, tokens=64, sequences=1,
            heads=4, key_heads=2, dim=64, s=None):
    return k.lib.bsa_linear_attention_forward(dtype, q, kk, v, out, decay, offsets, first, last, states, size, segment, tokens, sequences, heads,
                                              key_heads, dim, strides(6) if s is None else s or None, 1.0, None)


def backward(k, dtype=F16, dout=P, dq=P, dk=P, dv=P, states=None, scratch=None, size=0, dlast=None, dfirst=None, tokens=64, dim=64, s=None):
    return k.lib.bsa_linear_attention_backward(dtype, P, P, P, dout, P, P, None, states, dlast, dq, dk, dv, dfirst, scratch, size, 256, tokens, 1, 4, 2,
                                               dim, strides(8) if s is None else s, 1.0, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(dim=96), "64 and 128"), (dict(heads=3), "cannot share"), (dict(key_heads=0), "cannot share"),
    (dict(tokens=0), "0 tokens"), (dict(tokens=(1 << 30) + 1), "tokens"), (dict(sequences=0), "0 sequences"), (dict(sequences=65536), "sequences"),
    (dict(tokens=1 << 30, heads=512, key_heads=512), "too many"), (dict(segment=0), "segments"), (dict(segment=100), "segments"),
    (dict(segment=16), "segments"), (dict(segment=1 << 21), "segments"), (dict(tokens=300), "states of"), (dict(tokens=300, states=P, size=32767), "states of"),
    (dict(q=None), "null"), (dict(kk=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"), (dict(decay=None), "null"),
    (dict(offsets=None), "null"), (dict(q=P + 8), "aligned to 16"), (dict(out=P + 8), "aligned to 16"), (dict(first=P + 4), "aligned to 16"),
    (dict(last=P + 8), "aligned to 16"), (dict(s=()), "null"), (dict(s=strides(6, _0=4)), "multiple of 8"), (dict(s=strides(6, _3=-8)), "multiple of 8"),
    (dict(s=strides(6, _2=(1 << 24) + 8)), "between tokens"), (dict(s=strides(6, _1=(1 << 40) + 8)), "too large"),
])
def test_linear_forward(k, kw, needle):
    refused(k, forward(k, **kw), "bsa_linear_attention_forward", needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(dim=32), "64 and 128"), (dict(tokens=0), "0 tokens"), (dict(dout=None), "null"), (dict(dq=None), "null"),
    (dict(dk=None), "null"), (dict(dv=None), "null"), (dict(dv=P + 8), "aligned to 16"), (dict(dlast=P + 8), "aligned to 16"),
    (dict(dfirst=P + 4), "aligned to 16"), (dict(tokens=257), "states of"), (dict(tokens=257, states=P, size=1 << 20), "states of"),
    (dict(s=strides(8, _7=4)), "multiple of 8"), (dict(s=strides(8, _6=(1 << 24) + 8)), "between tokens"),
])
def test_linear_backward(k, kw, needle):
    refused(k, backward(k, **kw), "bsa_linear_attention_backward", needle)


def test_states_between_segments(k):
    size = k.lib.bsa_linear_attention_states_bytes
    assert size(256, 2, 64, 256) == 0 and size(257, 2, 64, 256) == 4 * 2 * 64 * 64 and size(1000, 3, 128, 256) == 3 * 4 * 3 * 128 * 128
    assert size(0, 2, 64, 256) == 0 and size(5, 0, 64, 256) == 0
    for args in ((1, 1, 1, 64), (10 ** 6, 4, 64, 128), (2 ** 30, 65535, 8, 64)):
        segment = k.lib.bsa_linear_attention_segment(*args)
        assert segment >= 32 and segment % 32 == 0
    assert k.lib.bsa_linear_attention_segment(0, 0, 0, 64) >= 32


def step(k, dtype=F16, q=P, out=P, decay=P, states=P, slots=P, batch=3, places=4, heads=4, key_heads=2, dim=64, s=None):
    return k.lib.bsa_linear_attention_step(dtype, q, P, P, out, decay, states, slots, batch, places, heads, key_heads, dim,
                                           strides(6) if s is None else s, 1.0, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(dim=32), "64 and 128"), (dict(heads=5), "cannot share"), (dict(batch=0), "0 sequences"),
    (dict(batch=65536), "sequences"), (dict(places=-1), "states for"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(decay=None), "null"),
    (dict(states=None), "null"), (dict(slots=None), "null"), (dict(states=P + 8), "aligned to 16"), (dict(s=strides(6, _4=12)), "multiple of 8"),
])
def test_linear_step(k, kw, needle):
    refused(k, step(k, **kw), "bsa_linear_attention_step", needle)


SIZES = dict(sequences=4, width=3, pages=10, page=32)


@pytest.mark.parametrize("kw,needle", [
    (dict(page=48), "pages of 32"), (dict(pages=0), "0 pages"), (dict(pages=1 << 26), "pages of"), (dict(sequences=0), "0 sequences"),
    (dict(sequences=4097), "4097 sequences"), (dict(width=0), "sequences of 0"), (dict(width=1 << 26), "sequences of"),
    (dict(sequences=4096, width=1 << 19), "4096 sequences of"),
])
def test_tables(k, kw, needle):
    z = list({**SIZES, **kw}.values())
    refused(k, k.lib.bsa_pages_append(P, P, P, P, P, P, 5, *z, P, None), "bsa_pages_append", needle)
    refused(k, k.lib.bsa_pages_free(P, P, P, P, 2, *z, None), "bsa_pages_free", needle)
    refused(k, k.lib.bsa_pages_fork(P, P, P, P, P, P, P, P, 2, *z, P, 1 << 20, None), "bsa_pages_fork", needle)
    refused(k, k.lib.bsa_pages_compact(P, P, P, P, P, *z, P, None), "bsa_pages_compact", needle)


def test_table_pointers_and_counts(k):
    z = list(SIZES.values())
    for at in range(5):
        pointers = [None if i == at else P for i in range(5)]
        refused(k, k.lib.bsa_pages_append(*pointers, P, 5, *z, P, None), "null")
        refused(k, k.lib.bsa_pages_compact(*pointers, *z, P, None), "null")
    refused(k, k.lib.bsa_pages_append(P, P, P, P, P, None, 5, *z, P, None), "null")
    refused(k, k.lib.bsa_pages_append(P, P, P, P, P, P, 5, *z, None, None), "null")
    refused(k, k.lib.bsa_pages_append(P, P, P, P, P, P, -1, *z, P, None), "-1 tokens")
    refused(k, k.lib.bsa_pages_free(P, P, P, None, 2, *z, None), "null")
    refused(k, k.lib.bsa_pages_free(P, P, P, P, -2, *z, None), "-2 entries")
    refused(k, k.lib.bsa_pages_free(P, P, P, P, 4097, *z, None), "4097 entries")
    for at in range(8):
        pointers = [None if i == at else P for i in range(8)]
        refused(k, k.lib.bsa_pages_fork(*pointers, 2, *z, P, 1 << 20, None), "null")
    refused(k, k.lib.bsa_pages_fork(*[P] * 8, 2, *z, None, 1 << 20, None), "null")
    refused(k, k.lib.bsa_pages_fork(*[P] * 8, 2, *z, P, k.lib.bsa_pages_fork_scratch_bytes(2, 3) - 1, None), "scratch of")
    refused(k, k.lib.bsa_pages_fork(*[P] * 8, 2, *z, P + 4, 1 << 20, None), "aligned to 16")
    refused(k, k.lib.bsa_pages_compact(P, P, P, P, P, *z, None, None), "null")
    # nothing to do: nothing is launched
    assert k.lib.bsa_pages_free(P, P, P, None, 0, *z, None) == 0 and k.lib.bsa_pages_fork(P, P, P, *[None] * 5, 0, *z, None, 0, None) == 0
    assert k.lib.bsa_pages_fork_scratch_bytes(0, 3) == 0


def copying(k, dtype=I8, tensors=None, pages=5, from_pages=5, count=2, heads=2, dim=64, page=32, lists=(P, P)):
    t = tensors or [P] * 8
    return k.lib.bsa_cache_copy(dtype, *t[:4], from_pages, *t[4:], pages, *lists, count, heads, dim, page, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "int8 or e4m3"), (dict(dim=96), "64 and 128"), (dict(heads=0), "cannot share"), (dict(page=40), "pages of 32"),
    (dict(pages=0), "0 pages"), (dict(from_pages=0), "0 pages"), (dict(count=-1), "-1 pages"), (dict(count=(1 << 24) + 1), "pages to copy"),
    (dict(lists=(None, P)), "null"), (dict(lists=(P, None)), "null"),
] + [(dict(tensors=[None if i == at else P for i in range(8)]), "null") for at in range(8)]
  + [(dict(tensors=[P + 8 if i == at else P for i in range(8)]), "aligned to 16") for at in (0, 5, 7)])
def test_copies(k, kw, needle):
    refused(k, copying(k, **kw), "bsa_cache_copy", needle)


def test_copies_of_nothing(k):
    assert copying(k, count=0, lists=(None, None)) == 0 and copying(k, dtype=F16, tensors=[P, P, None, None] * 2, count=0) == 0


def test_lengths_of_segments(k):
    """What fills the machine where tokens are many, by the mean length where they are few, one launch where sequences are short."""
    segment = k.lib.bsa_linear_attention_segment
    assert segment(65519, 5, 4, 128) == 544 and segment(24575, 2, 16, 128) == 832 and segment(10 ** 7, 1, 64, 128) == 8192
    assert segment(65536, 1, 1, 64) == 320 and segment(2000, 1, 1, 64) == 96 and segment(368, 5, 12, 64) == 512
