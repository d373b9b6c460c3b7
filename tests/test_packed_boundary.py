"""CPU: what packed attention, the cache and attention over it ask of a call before anything is launched."""
import pytest
import torch

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
    import ctypes
    values = [512, 64] * (n // 2 + 1)
    for at, value in changed.items():
        values[int(at[1:])] = value
    return (ctypes.c_int64 * n)(*values[:n])


def forward(k, dtype=F16, q=P, kk=P, v=P, out=P, rest=None, offsets=P, tokens=64, sequences=1, heads=4, key_heads=2, dim=64, s=None):
    return k.lib.bsa_packed_attention_forward(dtype, q, kk, v, out, rest, None, offsets, tokens, sequences, heads, key_heads, dim,
                                              strides(6) if s is None else s or None, 1.0, 1, None)


def backward(k, dtype=F16, q=P, dout=P, out=P, rest=P, lse=P, delta=P, dq=P, dk=P, dv=P, tokens=64, dim=64, s=None):
    return k.lib.bsa_packed_attention_backward(dtype, q, P, P, dout, out, rest, lse, delta, dq, dk, dv, P, tokens, 1, 4, 2, dim,
                                               strides(8) if s is None else s, 1.0, 1, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(dtype=I8), "fp16 and bf16"), (dict(dim=96), "64 and 128"), (dict(dim=0), "64 and 128"),
    (dict(heads=3), "cannot share"), (dict(key_heads=0), "cannot share"), (dict(heads=0), "cannot share"), (dict(heads=65536), "cannot share"),
    (dict(tokens=0), "0 tokens"), (dict(tokens=-1), "tokens"), (dict(sequences=0), "0 sequences"), (dict(tokens=(1 << 30) + 1), "tokens"),
    (dict(tokens=1 << 30, heads=64, key_heads=8), "too many"), (dict(sequences=1 << 23), "too many"),
    (dict(q=None), "null"), (dict(kk=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"), (dict(offsets=None), "null"),
    (dict(q=P + 8), "aligned to 16"), (dict(v=P + 2), "aligned to 16"), (dict(out=P + 8), "aligned to 16"), (dict(rest=P + 8), "aligned to 16"),
    (dict(s=()), "null"), (dict(rest=P), "go together"),
])
def test_packed_forward(k, kw, needle):
    refused(k, forward(k, **kw), "bsa_packed_attention_forward", needle)


@pytest.mark.parametrize("at,value,needle", [(0, 4, "multiple of 8"), (3, 65, "multiple of 8"), (5, -8, "multiple of 8"),
                                             (2, (1 << 24) + 8, "between tokens"), (1, (1 << 40) + 8, "too large")])
def test_packed_strides(k, at, value, needle):
    refused(k, forward(k, s=strides(6, **{f"_{at}": value})), needle)
    refused(k, backward(k, s=strides(8, **{f"_{at}": value})), needle)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(dim=32), "64 and 128"), (dict(tokens=0), "0 tokens"),
    (dict(dout=None), "null"), (dict(out=None), "null"), (dict(rest=None), "null"), (dict(lse=None), "null"), (dict(delta=None), "null"),
    (dict(dq=None), "null"), (dict(dk=None), "go together"), (dict(dv=None), "go together"),
    (dict(dout=P + 4), "aligned to 16"), (dict(rest=P + 4), "aligned to 16"), (dict(dv=P + 8), "aligned to 16"),
])
def test_packed_backward(k, kw, needle):
    refused(k, backward(k, **kw), "bsa_packed_attention_backward", needle)


def write(k, dtype=F16, held=I8, rows=P, keys=P, scales=P, slots=P, tokens=4, heads=2, dim=64, pages=8, page=64, s=None):
    return k.lib.bsa_cache_write(dtype, held, rows, P, slots, keys, P, scales, P, tokens, heads, dim, pages, page, strides(4) if s is None else s, None)


def read(k, dtype=F16, held=I8, rows=P, keys=P, scales=P, slots=P, tokens=4, heads=2, dim=64, pages=8, page=64):
    return k.lib.bsa_cache_read(dtype, held, keys, P, scales, P, slots, rows, P, tokens, heads, dim, pages, page, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(held=F32), "a cache holds"), (dict(held=9), "a cache holds"), (dict(page=48), "pages of 32"), (dict(page=0), "pages of 32"),
    (dict(page=512), "pages of 32"), (dict(pages=0), "0 pages"), (dict(pages=1 << 25), "pages of 64"), (dict(dim=80), "64 and 128"),
    (dict(heads=0), "cannot share"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30, heads=64), "tokens of 64 heads"),
    (dict(rows=None), "null"), (dict(slots=None), "null"), (dict(keys=None), "null"), (dict(scales=None), "null"),
    (dict(rows=P + 8), "aligned to 16"), (dict(keys=P + 8), "aligned to 16"), (dict(scales=P + 4), "aligned to 16"),
])
def test_cache_rows(k, kw, needle):
    refused(k, write(k, **kw), "bsa_cache_write", needle)
    refused(k, read(k, **kw), "bsa_cache_read", needle)


def test_cache_row_types(k):
    refused(k, write(k, dtype=F32), "fp16 and bf16")
    refused(k, write(k, dtype=F16, held=BF16, scales=None), "its own type")
    refused(k, read(k, dtype=E4M3), "fp32, fp16 or bf16")
    refused(k, write(k, s=strides(4, _2=12)), "multiple of 8")
    assert write(k, tokens=0, rows=None, slots=None) == 0 and read(k, tokens=0, rows=None, slots=None) == 0


def attend(k, dtype=F16, held=I8, q=P, out=P, keys=P, scales=P, table=P, lengths=P, batch=2, drafts=1, heads=4, key_heads=2, dim=64,
           pages=8, page=64, width=4, workspace=P, size=1 << 40, s=None):
    return k.lib.bsa_cached_attention(dtype, held, q, P, P, out, keys, P, scales, P, table, lengths, None, 0, batch, drafts, heads, key_heads,
                                      dim, pages, page, width, strides(9) if s is None else s, 1.0, workspace, size, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=F32), "fp16 and bf16"), (dict(held=F32), "a cache holds"), (dict(held=BF16), "its own type"), (dict(dim=32), "64 and 128"),
    (dict(page=16), "pages of 32"), (dict(pages=0), "0 pages"), (dict(batch=0), "0 sequences"), (dict(drafts=0), "0 new tokens"),
    (dict(drafts=1025), "1025 new tokens"), (dict(width=-1), "-1 pages"), (dict(width=1 << 24), "pages of 64"),
    (dict(heads=6, key_heads=4), "cannot share"), (dict(batch=1 << 20, heads=64, key_heads=8), "too many"),
    (dict(batch=1 << 19, width=1 << 20), "too many"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(keys=None), "null"), (dict(scales=None), "null"), (dict(table=None), "null"),
    (dict(lengths=None), "null"), (dict(q=P + 8), "aligned to 16"), (dict(out=P + 4), "aligned to 16"), (dict(workspace=P + 8), "aligned to 16"),
    (dict(s=strides(9, _4=4)), "multiple of 8"),
])
def test_cached_attention(k, kw, needle):
    refused(k, attend(k, **kw), "bsa_cached_attention", needle)


@pytest.mark.parametrize("batch,drafts,heads,key_heads,dim", [(1, 1, 8, 8, 64), (64, 1, 32, 4, 128), (7, 61, 4, 4, 64), (3, 1024, 16, 2, 128)])
def test_cached_workspace(k, batch, drafts, heads, key_heads, dim):
    """Nothing for tables that one unit a sequence covers, and never more than every unit's rows; what is short is refused."""
    size = lambda width: k.lib.bsa_cached_attention_workspace_bytes(batch, drafts, heads, key_heads, dim, width, 64)
    assert size(0) == (0 if drafts <= 256 else size(1000))
    need = size(1000)
    rows = drafts * (heads // key_heads)
    assert rows * key_heads * (batch + 1) * (dim + 2) * 4 <= need <= (rows + 127) * key_heads * (batch + 768) * (dim + 2) * 4
    kw = dict(batch=batch, drafts=drafts, heads=heads, key_heads=key_heads, dim=dim, pages=1 << 20, width=1000)
    refused(k, attend(k, size=need - 1, **kw), "workspace of")
    refused(k, attend(k, workspace=None, **kw), "workspace of")


def test_python_side_refuses_before_the_device_is_touched():
    from sparse import KeyValueCache, cached_attention, packed_attention
    q, offsets = torch.zeros(4, 2, 64, dtype=torch.float16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="same GPU"):
        packed_attention(q, q, q, offsets)
    with pytest.raises(TypeError, match="float16 or all bfloat16"):
        packed_attention(q.float(), q, q, offsets)
    with pytest.raises(TypeError, match="float16 or all bfloat16"):
        packed_attention(q, q.bfloat16(), q, offsets)
    with pytest.raises(TypeError, match="must be a KeyValueCache"):
        cached_attention(q, q, q, None, offsets, offsets)
    for kw, error, needle in ((dict(dtype=torch.float32), TypeError, "a cache holds"), (dict(page=48), ValueError, "page must be"),
                              (dict(head_dim=96), ValueError, "head dim"), (dict(pages=0), ValueError, "addressed"),
                              (dict(heads=0), ValueError, "addressed"), (dict(pages=1 << 25), ValueError, "addressed"),
                              (dict(device="cpu"), ValueError, "lives on the GPU")):
        with pytest.raises(error, match=needle):
            KeyValueCache(**{**dict(pages=2, heads=2, head_dim=64), **kw})


def test_a_cache_loaded_off_the_gpu_is_refused():
    from sparse import KeyValueCache
    rows = torch.zeros(2, 1, 32, 64, dtype=torch.uint8)
    state = dict(pages=2, heads=1, head_dim=64, dtype=torch.int8, page=32, device=torch.device("cuda", 0),
                 _held=(rows, rows.clone(), torch.zeros(2, 1, 32), torch.zeros(2, 1, 32)))
    with pytest.raises(ValueError, match="lives on the GPU"):
        KeyValueCache.__new__(KeyValueCache).__setstate__(state)


@pytest.mark.parametrize("kind", ["slice", "heads first", "one token", "odd start", "odd stride", "broadcast"])
def test_operands_are_copied_only_where_a_row_cannot_be_read_in_place(kind):
    from sparse.packed import rows_of, strides_of
    flat = torch.arange(40 * 6 * 64, dtype=torch.float16)
    t = {"slice": lambda: flat.view(40, 6, 64)[3:30, 1:5],
         "heads first": lambda: flat.view(6, 40, 64).transpose(0, 1),
         "one token": lambda: flat.view(40, 6, 64)[3:4],
         "odd start": lambda: flat[1:1 + 39 * 6 * 64].view(39, 6, 64),
         "odd stride": lambda: flat[:40 * 6 * 63].view(40, 6, 63).as_strided((20, 6, 64), (6 * 65, 65, 1)),
         "broadcast": lambda: flat[:64].view(1, 1, 64).expand(10, 6, 64)}[kind]()
    got = rows_of(t)
    assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in strides_of(got))
    assert (got.data_ptr() == t.data_ptr()) == (kind not in ("odd start", "odd stride"))


@pytest.mark.parametrize("dim,sequences", [(64, (1 << 24) // 16), (128, (1 << 23) // 16)])
def test_a_training_step_whose_walk_over_the_keys_cannot_be_launched(k, dim, sequences):
    """256 threads a workgroup at head dim 64, 512 at 128, and 2^32 in a launch: refused before the first launch of the backward call, and
    by the forward call whose statistics are wanted."""
    lse = P
    given = (64, sequences, 16, 16, dim)
    code = k.lib.bsa_packed_attention_backward(F16, P, P, P, P, P, P, lse, P, P, P, P, P, *given, strides(8), 1.0, 1, None)
    refused(k, code, "bsa_packed_attention_backward", "too many")
    code = k.lib.bsa_packed_attention_forward(F16, P, P, P, P, P, lse, P, *given, strides(6), 1.0, 1, None)
    refused(k, code, "bsa_packed_attention_forward", "too many")


def test_many_tokens_are_refused_by_the_slots_of_64_keys(k):
    given = (600_000, 600_000, 16, 16, 128)
    code = k.lib.bsa_packed_attention_backward(F16, P, P, P, P, P, P, P, P, P, P, P, P, *given, strides(8), 1.0, 1, None)
    refused(k, code, "too many")


def test_the_backward_pass_looks_at_what_autograd_hands_it():
    """Hooks on saved tensors may give back anything: nothing off the GPU, of another type or shape gets to a kernel."""
    from sparse.packed import run_backward
    rows, keys, lse, offsets = torch.zeros(4, 2, 64).half(), torch.zeros(4, 1, 64).half(), torch.zeros(2, 4), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="same GPU"):
        run_backward(rows, keys, keys, rows, rows, rows, lse, offsets, 1.0, True, True)
    with pytest.raises(TypeError, match="float16 or all bfloat16"):
        run_backward(rows.float(), keys, keys, rows, rows, rows, lse, offsets, 1.0, True, True)
