"""GPU: ``KeyValueCache`` and ``cached_attention`` against the float64 oracle (oracle/packed_oracle.py)."""
import numpy as np
import pytest
import torch

from helpers import to_np
from oracle import packed_oracle as po

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
HELD = [torch.int8, torch.float8_e4m3fn]


def kind_of(dtype):
    return {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}.get(dtype, str(dtype).replace("torch.", ""))


def values_of(t):
    return t.float().cpu().double().numpy()


def rows_like_layers(seed, tokens, heads, dim, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp(torch.randn(1, heads, dim, generator=g)) * torch.exp(torch.randn(tokens, heads, 1, generator=g))
    return x.to(dtype).cuda()


def new_cache(pages, heads, dim, held, page, fill=0x5A):
    import sparse
    cache = sparse.KeyValueCache(pages, heads, dim, dtype=held, page=page)
    for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales):
        if t is not None:
            t.view(torch.uint8).fill_(fill)
    return cache


def buffers(cache):
    return [t.view(torch.uint8).clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales) if t is not None]


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 32), (3, 5, 64), (77, 3, 256), (300, 2, 128)])
def test_rows_are_quantised_as_defined(tokens, heads, page, dim, dtype, held):
    """Values to the bit, scales to half a step of fp32; everything else in the cache as it was."""
    cache = new_cache(-(-tokens // page) + 3, heads, dim, held, page)
    before = buffers(cache)
    k, v = rows_like_layers(1, tokens, heads, dim, dtype), rows_like_layers(2, tokens, heads, dim, dtype)
    slots = np.random.RandomState(5).permutation(cache.pages * page)[:tokens]
    slots[1::4] = -1
    slots[2::11] = cache.pages * page + 3          # behind the cache
    cache.write(k, v, torch.tensor(slots, dtype=torch.int32, device="cuda"))
    kept = (slots >= 0) & (slots < cache.pages * page)
    at, place = slots[kept] // page, slots[kept] % page
    written = np.zeros((cache.pages, heads, page), dtype=bool)
    written[at, :, place] = True
    for rows, values, scales in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
        y, s = po.quantise(to_np(rows), kind_of(held))
        assert np.array_equal(values_of(values)[at, :, place], y[kept])
        got = values_of(scales)[at, :, place]
        assert (np.abs(got - s[kept]) <= 2.0 ** -24 * s[kept]).all()
    for was, now in zip(before, buffers(cache)):
        per = now.shape[-1] * now[0, 0].numel() // now.shape[-1] // page
        same = (was == now).cpu().numpy().reshape(cache.pages, heads, page, per).all(-1)
        assert same[~written].all()


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_magnitude_of_a_row_at_every_maximum(dtype, held):
    """All quotients that 16-bit values of a few bits can make with one another, ties among them, and the ends of the
    type's range."""
    dim, top = 128, 2.0 ** (15 if dtype == torch.float16 else 120)
    maxima = [1.0, 127 / 128, 1.0078125, 1.5, 1.984375, 1.25, 0.5078125, 100.0, 127.0, 63.5]
    rows = []
    for m in maxima:
        for unit in (1.0, top / 128, 2.0 ** -10 if dtype == torch.float16 else 2.0 ** -120):
            rows.append(np.linspace(0, 1, dim) * m * unit)
            rows.append(-np.linspace(1, 0, dim) * m * unit)
    x = torch.tensor(np.array(rows), dtype=torch.float64).to(dtype)[:, None, :].cuda()
    cache = new_cache(4, 1, dim, held, 32)
    cache.write(x, x, torch.arange(len(rows), dtype=torch.int32, device="cuda"))
    y, s = po.quantise(to_np(x), kind_of(held))
    assert np.array_equal(values_of(cache.values)[:, 0].reshape(-1, dim)[:len(rows)], y[:, 0])
    got = values_of(cache.value_scales)[:, 0].reshape(-1)[:len(rows)]
    assert (np.abs(got - s[:, 0]) <= 2.0 ** -24 * s[:, 0] + 2.0 ** -150).all()


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_zero_rows_and_rows_that_are_no_numbers(dim, dtype, held):
    cache = new_cache(2, 2, dim, held, 32)
    x = rows_like_layers(3, 6, 2, dim, dtype)
    x[1] = 0
    x[2, 0, 7] = float("inf")
    x[3, 1, dim - 1] = float("nan")
    x[4, 0, 0] = -float("inf")
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    cache.write(x, x, slots)
    for t in cache.read(slots, torch.float32):
        bad = torch.zeros(6, 2, dtype=torch.bool)
        bad[2, 0] = bad[3, 1] = bad[4, 0] = True
        assert torch.isnan(t[bad]).all() and torch.isfinite(t[~bad]).all()
        assert not t[1].any()
    assert not values_of(cache.keys)[0, 0, 2].any() and values_of(cache.key_scales)[0, 0, 1] == 0


@pytest.mark.parametrize("held", HELD + DTYPES)
@pytest.mark.parametrize("to", [torch.float32] + DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_are_read_back(dim, to, held):
    dtype = held if held in DTYPES else torch.bfloat16
    cache = new_cache(5, 3, dim, held, 64)
    k, v = rows_like_layers(4, 90, 3, dim, dtype), rows_like_layers(5, 90, 3, dim, dtype)
    slots = torch.tensor(np.random.RandomState(1).permutation(320)[:90], dtype=torch.int32, device="cuda")
    cache.write(k, v, slots)
    ask = torch.cat([slots[::3], slots[:2], torch.tensor([-1, 320, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")])
    for rows, got in zip((k, v), cache.read(ask, to)):
        assert got.dtype == to and not got[-4:].any()
        rows = torch.cat([rows[::3], rows[:2]])
        if held in DTYPES:
            assert torch.equal(got[:-4], rows.to(to))
            continue
        y, s = po.quantise(to_np(rows), kind_of(held))
        exact = y * s[..., None]
        # the scale's rounding, the product's in fp32, the result's: all relative
        unit = 2.0 ** -24 * 2.01 + (0 if to == torch.float32 else po.UNIT[kind_of(to)] * (1 + 2.0 ** -20))
        assert (np.abs(to_np(got[:-4]) - exact) <= unit * np.abs(exact) + (2.0 ** -25 if to == torch.float16 else 0)).all()


def test_rows_from_slices_and_odd_starts():
    cache, other = (new_cache(4, 2, 64, torch.int8, 32) for _ in range(2))
    g = torch.Generator().manual_seed(6)
    fused = torch.randn(50, 3 * 2 * 64, generator=g).half().cuda()
    k, v = fused[:, 128:256].view(50, 2, 64), fused[:, 256:].view(50, 2, 64)
    odd = torch.randn(50 * 2 * 64 + 3, generator=g).half().cuda()[3:].view(50, 2, 64)
    slots = torch.arange(50, dtype=torch.int32, device="cuda")
    for a, b in ((k, v), (odd, v), (v, odd)):
        cache.write(a, b, slots)
        other.write(a.contiguous().clone(), b.contiguous().clone(), slots)
        assert all(torch.equal(x, y) for x, y in zip(buffers(cache), buffers(other)))


# ---- attention -----------------------------------------------------------------------------------------
def tree_of(seed, batch, drafts):
    rng, mask = np.random.RandomState(seed), np.zeros((batch, drafts, drafts), dtype=bool)
    for b in range(batch):
        for i in range(drafts):
            parent = rng.randint(-1, i)
            if parent >= 0:
                mask[b, i] = mask[b, parent]
            mask[b, i, i] = True
    return mask


def filled(seed, lengths, heads, dim, held, page, dtype, spare=3, width=None):
    """A cache with sequences of these lengths on pages in any order, its page table, what it holds of each."""
    per = [-(-n // page) for n in lengths]
    cache = new_cache(sum(per) + spare, heads, dim, held, page, fill=0x7F)       # NaN in e4m3, fp16's and bf16's scales
    order = np.random.RandomState(seed).permutation(cache.pages)[:sum(per)]
    width = max(max(per), 1) if width is None else width
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    slots, first = [], 0
    for b, n in enumerate(lengths):
        mine = order[first:first + per[b]]
        table[b, :per[b]] = mine
        slots.append((mine[:, None] * page + np.arange(page)).reshape(-1)[:n])
        first += per[b]
    flat = torch.tensor(np.concatenate(slots), dtype=torch.int32, device="cuda")
    if flat.numel():
        cache.write(rows_like_layers(seed + 1, flat.numel(), heads, dim, dtype), rows_like_layers(seed + 2, flat.numel(), heads, dim, dtype), flat)
    both, scales = [], None
    if held in HELD:
        t = values_of(cache.value_scales)
        scales = [t[s // page, :, s % page].T if len(s) else np.zeros((heads, 0)) for s in slots]
    for which in ("keys", "values"):
        y = values_of(getattr(cache, which))
        if held in HELD:
            y = y * values_of(getattr(cache, which[:-1] + "_scales"))[..., None]
        both.append([y[s // page, :, s % page].transpose(1, 0, 2) if len(s) else np.zeros((heads, 0, dim)) for s in slots])
    return cache, torch.tensor(table, device="cuda"), both + [scales]


def check(lengths, drafts, heads, key_heads, dim, held, page=64, dtype=torch.float16, tree=None, seed=1, scale=None, width=None):
    import sparse
    dtype = held if held in DTYPES else dtype
    batch = len(lengths)
    scale = dim ** -0.5 / 4 if scale is None else scale
    cache, table, (keys, values, scales) = filled(seed, lengths, key_heads, dim, held, page, dtype, width=width)
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(batch, drafts, heads, dim, generator=g).to(dtype).cuda()
    k, v = (torch.randn(batch, drafts, key_heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    given = None if tree is None else torch.from_numpy(tree).cuda()
    got = sparse.cached_attention(q, k, v, cache, table, lens, tree=given, scale=scale)
    mask = np.broadcast_to(np.tril(np.ones((drafts, drafts), dtype=bool)) if tree is None else tree, (batch, drafts, drafts))
    value, bound = po.cached(*(to_np(t) for t in (q, k, v)), keys, values, scales, lengths, mask, scale, kind_of(dtype))
    off = np.abs(to_np(got) - value)
    assert np.isfinite(to_np(got)).all()
    worst = (off - bound).argmax()
    assert (off <= bound).all(), (off.max(), off.flat[worst], bound.flat[worst], np.unravel_index(worst, off.shape))
    again = sparse.cached_attention(q, k, v, cache, table, lens, tree=given, scale=scale)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("held", HELD + DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [32, 256])
def test_one_new_token(page, dim, held):
    check([0, 1, 31, 32, 33, 63, 64, 65, 200, 255, 256, 257, 700], 1, 4, 2, dim, held, page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (8, 1), (32, 1), (33, 1), (12, 4), (5, 5)])
def test_shared_heads(heads, key_heads, dtype):
    check([70, 0, 300], 1, heads, key_heads, 64, torch.int8, dtype=dtype)
    check([70, 0, 300], 2, heads, key_heads, 128, torch.float8_e4m3fn, dtype=dtype)


@pytest.mark.parametrize("held", HELD + DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafts,group", [(2, 1), (27, 1), (27, 4), (33, 2), (64, 2), (65, 1), (100, 3)])
def test_trees(drafts, group, dim, held):
    check([0, 5, 130], drafts, 2 * group, 2, dim, held, tree=tree_of(drafts, 3, drafts))


@pytest.mark.parametrize("drafts", [1, 5, 40])
def test_one_tree_for_all_and_a_chain(drafts):
    import sparse
    got = check([100, 7], drafts, 4, 2, 64, torch.int8, tree=tree_of(1, 1, drafts)[0])
    assert torch.equal(got, check([100, 7], drafts, 4, 2, 64, torch.int8, tree=np.broadcast_to(tree_of(1, 1, drafts), (2, drafts, drafts)).copy()))
    chain = np.tril(np.ones((drafts, drafts), dtype=bool))
    assert torch.equal(check([100, 7], drafts, 4, 2, 64, torch.int8), check([100, 7], drafts, 4, 2, 64, torch.int8, tree=chain))


@pytest.mark.parametrize("drafts", [3, 40])
def test_a_new_token_that_sees_nothing_gets_zeros(drafts):
    tree = tree_of(2, 2, drafts)
    tree[:, 1] = False
    got = check([0, 40], drafts, 2, 1, 128, torch.int8, tree=tree)
    assert not got[0, 1].any() and got[1, 1].any()


@pytest.mark.parametrize("held", HELD + [torch.float16])
@pytest.mark.parametrize("drafts,group", [(1, 8), (40, 2)])
def test_long_sequences_in_chunks(drafts, group, held):
    check([9000, 3, 0, 2500, 1], drafts, group, 1, 64, held, page=128, tree=tree_of(3, 5, drafts))
    check([9000], drafts, group, 1, 128, held, page=32, tree=tree_of(3, 1, drafts))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(scale):
    check([300, 40], 3, 2, 1, 64, torch.int8, scale=scale)
    check([300, 40], 20, 4, 1, 128, torch.float16, scale=scale)


def test_a_page_table_wider_than_any_sequence():
    narrow = check([300, 40], 1, 2, 1, 64, torch.int8)
    wide = check([300, 40], 1, 2, 1, 64, torch.int8, width=4000)
    assert torch.allclose(narrow.float(), wide.float(), rtol=2 ** -8, atol=2 ** -8)


@pytest.mark.parametrize("drafts", [1, 40])
def test_many_sequences(drafts):
    rng = np.random.RandomState(4)
    check(rng.randint(0, 90, 150).tolist(), drafts if drafts == 1 else 20, 2, 1, 64, torch.int8, page=32)


def test_lengths_and_pages_outside_the_cache():
    """Tokens on a page that the cache does not have are not seen; a length past the table is the table's."""
    import sparse
    cache, table, _ = filled(7, [200, 200], 1, 64, torch.int8, 32, torch.float16, spare=0)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 3, 1, 64, generator=g).half().cuda() for _ in range(3))
    call = lambda pages, lengths: sparse.cached_attention(q, k, v, cache, pages, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=0.1)
    for bad in (-1, cache.pages, 2 ** 31 - 1, -2 ** 31):
        holes = table.clone()
        holes[1, 2:4] = bad
        closed = torch.cat([holes[1, :2], holes[1, 4:], holes[1, :2]])[None].contiguous()      # the same pages without the holes
        got = call(torch.cat([table[:1], holes[1:]]), [200, 200])[1]
        want = call(torch.cat([table[:1], closed]), [200, 136])[1]
        assert torch.allclose(got.float(), want.float(), rtol=2 ** -9, atol=2 ** -11)
    # behind the written tokens of the last page lie bytes that are large scales: NaN on both sides
    assert torch.allclose(call(table, [-7, 2 ** 31 - 1]), call(table, [0, 32 * table.size(1)]), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("held", [torch.int8, torch.float16])
def test_a_new_token_that_is_no_number_reaches_only_those_that_see_it(held):
    import sparse
    cache, table, _ = filled(8, [70, 33], 1, 64, held, 32, torch.float16)
    lengths = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    for drafts in (6, 50):
        q, k, v = (torch.randn(2, drafts, 2 if i == 0 else 1, 64, generator=g).half().cuda() for i in range(3))
        mask = tree_of(5, 2, drafts)
        call = lambda: sparse.cached_attention(q, k, v, cache, table, lengths, tree=torch.from_numpy(mask).cuda(), scale=0.1)
        clean = call()
        v[0, 2, 0, 3] = float("inf")
        v[1, 4] = float("nan")
        out = call()
        sees = torch.from_numpy(np.stack([mask[0][:, 2], mask[1][:, 4]]))
        assert torch.equal(out[~sees], clean[~sees])
        assert not torch.isfinite(out[0][sees[0]][:, :, 3]).any() and torch.isnan(out[1][sees[1]]).all()


def test_offsets_beyond_32_bits():
    """The last pages of a cache of more than 4 GiB of keys, and of more than 2^31 values."""
    import sparse
    pages, heads, dim, page = 8400, 8, 128, 256
    cache = sparse.KeyValueCache(pages * 2, heads, dim, dtype=torch.int8, page=page)
    assert cache.keys.numel() > 2 ** 32
    k, v = rows_like_layers(1, 300, heads, dim, torch.float16), rows_like_layers(2, 300, heads, dim, torch.float16)
    for at in (0, 2 * pages - 2):
        slots = torch.arange(300, dtype=torch.int32, device="cuda") + at * page
        cache.write(k, v, slots)
    first, last = cache.read(torch.arange(300, dtype=torch.int32, device="cuda"), torch.float32), cache.read(slots, torch.float32)
    assert torch.equal(first[0], last[0]) and torch.equal(first[1], last[1])
    q = torch.randn(1, 1, heads, dim, generator=torch.Generator().manual_seed(3)).half().cuda()
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    outs = [sparse.cached_attention(q, q, q, cache, torch.tensor([[at, at + 1]], dtype=torch.int32, device="cuda"), lengths, scale=0.1)
            for at in (0, 2 * pages - 2)]
    assert torch.equal(*outs)


def test_streams_and_two_graphs():
    """A step captured once and replayed while the sequences grow; a second graph of the same shapes shares nothing with it."""
    import sparse
    cache, table, _ = filled(9, [500, 2000], 2, 64, torch.int8, 64, torch.float16)
    lengths = torch.tensor([400, 1900], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(2, 1, 4 if i == 0 else 2, 64, generator=g).half().cuda() for i in range(3))
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")

    def step():
        out = sparse.cached_attention(q, k, v, cache, table, lengths, scale=0.1)
        cache.write(k[:, 0], v[:, 0], slots)
        lengths.add_(1)
        return out

    step()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    lengths.copy_(torch.tensor([400, 1900], dtype=torch.int32))
    for turn in range(6):
        at = lengths.cpu()
        slots.copy_(torch.tensor([int(table[b, at[b] // 64]) * 64 + int(at[b]) % 64 for b in range(2)], dtype=torch.int32))
        want = sparse.cached_attention(q, k, v, cache, table, lengths, scale=0.1)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], want) and torch.equal(lengths.cpu(), at + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = sparse.cached_attention(q, k, v, cache, table, lengths, scale=0.1)
    with torch.cuda.stream(side):
        got = sparse.cached_attention(q, k, v, cache, table, lengths, scale=0.1)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_request_from_prompt_to_accepted_drafts():
    """The operators as they are used together: prompts through packed attention, their rows into a 16-bit cache, a tree of drafts
    over it, the accepted branch into the cache, a decode step; every result is that of packed attention over the whole text."""
    import sparse
    lengths, drafts, heads, key_heads, dim, page = [75, 1, 130], 7, 4, 2, 64, 32
    g = torch.Generator().manual_seed(5)
    total = [n + drafts + 1 for n in lengths]
    text = [[torch.randn(n, h, dim, generator=g).half().cuda() for h in (heads, key_heads, key_heads)] for n in total]
    cache = sparse.KeyValueCache(16, key_heads, dim, dtype=torch.float16, page=page)
    table = torch.tensor([[3, 7, 1, 0, 9, 5], [2, 4, -1, -1, -1, -1], [6, 8, 10, 11, 12, 13]], dtype=torch.int32, device="cuda")
    slots = [[int(table[b, t // page]) * page + t % page for t in range(total[b])] for b in range(3)]
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")

    whole = [sparse.packed_attention(*t, int32([0, n]), 0.125) for t, n in zip(text, total)]
    prompt = [torch.cat([t[i][:n] for t, n in zip(text, lengths)]) for i in range(3)]
    out = sparse.packed_attention(*prompt, int32(np.cumsum([0] + lengths)), 0.125)
    assert torch.equal(out, torch.cat([w[:n] for w, n in zip(whole, lengths)]))
    cache.write(prompt[1], prompt[2], int32(sum([s[:n] for s, n in zip(slots, lengths)], [])))

    # a tree whose first branch, nodes 0 2 4 6, is the text; the others are other drafts
    parents, branch = [-1, -1, 0, 0, 2, 1, 4], [0, 2, 4, 6]
    tree = np.zeros((drafts, drafts), dtype=bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            tree[i] = tree[parent]
        tree[i, i] = True
    new = [torch.randn(3, drafts, h, dim, generator=g).half().cuda() for h in (heads, key_heads, key_heads)]
    for b, n in enumerate(lengths):
        for i in range(3):
            new[i][b, branch] = text[b][i][n:n + 4]
    out = sparse.cached_attention(*new, cache, table, int32(lengths), tree=torch.from_numpy(tree).cuda(), scale=0.125)
    close = lambda a, b: torch.allclose(a.float(), b.float(), rtol=2 ** -9, atol=2 ** -10)     # both rounded, summed in other orders
    for b, n in enumerate(lengths):
        assert close(out[b, branch], whole[b][n:n + 4])
    accepted = np.full((3, drafts), -1)
    for b, n in enumerate(lengths):
        accepted[b, branch] = slots[b][n:n + 4]
    cache.write(new[1].flatten(0, 1), new[2].flatten(0, 1), int32(accepted.reshape(-1)))
    step = [torch.stack([t[i][n + 4:n + 5] for t, n in zip(text, lengths)]) for i in range(3)]
    out = sparse.cached_attention(*step, cache, table, int32([n + 4 for n in lengths]), scale=0.125)
    for b, n in enumerate(lengths):
        assert close(out[b, 0], whole[b][n + 4])
    back = cache.read(int32(slots[2][:134]), torch.float16)
    assert torch.equal(back[0], text[2][1][:134]) and torch.equal(back[1], text[2][2][:134])


# ---- sizes of values --------------------------------------------------------------------------------------
def check_rows(k_rows, v_rows, drafts, group, held, low=None, small=1.0):
    """One sequence of these rows ``[tokens, 1, dim]``, page after page; the bound does not grow with the ratio of the value rows' sizes.  Token
    ``low`` has a score of -20 and less beside which the others' are a few: channel 0 of all queries is 8."""
    import sparse
    tokens, _, dim = k_rows.shape
    dtype, page = k_rows.dtype, 64
    cache = new_cache(-(-tokens // page), 1, dim, held, page)
    g = torch.Generator().manual_seed(21)
    q = torch.randn(1, drafts, group, dim, generator=g)
    q[..., 0] = 8
    k, v = torch.randn(1, drafts, 1, dim, generator=g), small * torch.randn(1, drafts, 1, dim, generator=g)
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    if low is not None:
        k_rows[:, :, 0] = 0
        k_rows[low] = 0
        k_rows[low, :, 0] = -20
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
    cache.write(k_rows, v_rows, slots)
    table = torch.arange(cache.pages, dtype=torch.int32, device="cuda")[None]
    got = sparse.cached_attention(q, k, v, cache, table, torch.tensor([tokens], dtype=torch.int32, device="cuda"), scale=0.125)
    rows = lambda which: values_of(getattr(cache, which)).transpose(1, 0, 2, 3).reshape(1, -1, dim)[:, :tokens]
    scales = lambda which: values_of(getattr(cache, which)).transpose(1, 0, 2).reshape(1, -1)[:, :tokens]
    mask = np.tril(np.ones((1, drafts, drafts), dtype=bool))
    t = scales("value_scales")
    value, bound = po.cached(*(values_of(x) for x in (q, k, v)), [rows("keys") * scales("key_scales")[..., None]], [rows("values") * t[..., None]],
                             [t], [tokens], mask, 0.125, kind_of(dtype), by_weight=True)
    bound = bound + (2.0 ** -134 if dtype == torch.bfloat16 else 0.0)       # half a step of its subnormal values
    off = np.abs(values_of(got) - value)
    assert torch.isfinite(got).all()
    worst = (off - bound).argmax()
    assert (off <= bound).all(), (off.max(), off.flat[worst], bound.flat[worst], np.unravel_index(worst, off.shape))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafts,group", [(1, 2), (50, 3)])
@pytest.mark.parametrize("low", [3, 1500])
def test_a_large_value_row_of_no_weight_costs_the_others_no_bits(low, drafts, group, dim, held):
    """One value row 2^15 times as large as the others, of a weight of 1e-9: in fp16 the others' weights relative to its size would
    have a few bits left."""
    g = torch.Generator().manual_seed(22)
    k, v = (torch.randn(2000, 1, dim, generator=g).half() for _ in range(2))
    v[low] *= 2.0 ** 13
    v[torch.arange(2000) != low] *= 0.25
    check_rows(k.cuda(), v.cuda(), drafts, group, held, low, 0.25)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("drafts,group,tokens", [(50, 3, 40), (50, 3, 96), (1, 2, 40)])
def test_small_cached_values_beside_new_tokens(drafts, group, tokens, held):
    """New tokens' rows come as they are, cached ones with scales of 2^-17: in one step with them they would lose 17 bits."""
    g = torch.Generator().manual_seed(23)
    k, v = torch.randn(tokens, 1, 64, generator=g).half(), (2.0 ** -11 * torch.randn(tokens, 1, 64, generator=g)).half()
    check_rows(k.cuda(), v.cuda(), drafts, group, held, small=2.0 ** -11)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("drafts,group", [(1, 2), (50, 3)])
@pytest.mark.parametrize("exponent", [-118, -60, 60, 110])
@pytest.mark.parametrize("flat", [True, False])
def test_values_of_any_size(flat, exponent, drafts, group, held):
    """bf16 rows near the ends of the type's range: weights relative to their scales must neither overflow nor vanish."""
    g = torch.Generator().manual_seed(24)
    k, v = (torch.randn(1500, 1, 64, generator=g) for _ in range(2))
    k, v = (k * (0 if flat else torch.linspace(0.1, 3, 1500)[:, None, None])).bfloat16(), (v * 2.0 ** exponent).bfloat16()
    check_rows(k.cuda(), v.cuda(), drafts, group, held, small=2.0 ** exponent)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("drafts,group", [(1, 2), (50, 3)])
@pytest.mark.parametrize("exponent", [-122, 100])
def test_value_rows_of_sizes_far_apart(exponent, drafts, group, held):
    """The first tiles are tiny or huge beside ordinary ones, which come later."""
    g = torch.Generator().manual_seed(25)
    k, v = (torch.randn(700, 1, 128, generator=g) for _ in range(2))
    v[:128] *= 2.0 ** exponent
    check_rows(k.bfloat16().cuda(), v.bfloat16().cuda(), drafts, group, held)
