"""GPU: ``PageTable`` and ``KeyValueCache.copy`` against the plain restatement (oracle/pages_oracle.py), to the bit, and together with
the attention over the cache and the recurrent states that they serve."""
import copy
import pickle

import numpy as np
import pytest
import torch

from oracle.pages_oracle import Pages

pytestmark = pytest.mark.gpu


def int32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def normal(seed, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def pair(pages, page, sequences, width):
    import sparse
    table = sparse.PageTable(pages, page, sequences, width)
    return table, Pages(table.table.cpu().numpy(), table.lengths.cpu().numpy(), table.uses.cpu().numpy(), page)


def same(table, plain, *results):
    for got, expected in zip((table.table, table.lengths, table.uses), plain.state()):
        assert np.array_equal(got.cpu().numpy(), expected)
    assert int(table.missing) == plain.missing
    for got, expected in results:
        assert np.array_equal(got.cpu().numpy(), expected)


def test_known_answers():
    table, plain = pair(8, 32, 4, 3)
    slots = table.append(int32([0, 33, 33, 65, 65]), 66)
    assert slots.tolist() == list(range(33)) + [64 + i for i in range(32)] + [-1]
    assert [t.tolist() for t in table.fork(int32([0, 0, 2]), int32([1, 3, 9]))] == [[1, 1, -1], [3, 4, -1]]
    assert table.table.tolist() == [[0, 1, -1], [0, 3, -1], [2, -1, -1], [0, 4, -1]] and table.uses.tolist() == [3, 1, 1, 1, 1, 0, 0, 0]
    table.free(int32([0, 0, 2, -1]))
    assert [t.tolist() for t in table.compact()] == [[3, 4, -1, -1], [1, 2, -1, -1]]
    assert [t.tolist() for t in table.fork(int32([1, 1]), int32([3, 1]))] == [[-1, 1], [-1, 2]]


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("sequences,width,pages,page", [(1, 1, 1, 32), (3, 2, 5, 256), (9, 5, 40, 32), (70, 4, 150, 64), (1100, 3, 2000, 32),
                                                        (40, 300, 9000, 32)])
def test_drawn_calls(sequences, width, pages, page, seed):
    r = np.random.RandomState(seed)
    table, plain = pair(pages, page, sequences, width)
    for _ in range(14):
        kind = r.randint(4)
        if kind == 0:
            new = r.randint(0, max(2, width * page // 2), sequences) * (r.rand(sequences) < r.choice([0.1, 0.5, 1.0]))
            if r.rand() < 0.3:
                new = np.minimum(new, 1)
            offsets = [0] + np.cumsum(new).tolist()
            tokens = int(new.sum()) + r.randint(0, 3)
            same(table, plain, (table.append(int32(offsets), tokens), plain.append(offsets, tokens)))
        elif kind == 1:
            which = r.randint(-1, sequences + 1, r.randint(0, sequences + 2)).tolist()
            plain.free(which)
            table.free(int32(which))
            same(table, plain)
        elif kind == 2:
            n = r.randint(0, 2 * sequences + 1)
            a, c = (r.randint(-1, sequences + 1, n).tolist() for _ in range(2))
            same(table, plain, *zip(table.fork(int32(a), int32(c)), plain.fork(a, c)))
        else:
            same(table, plain, *zip(table.compact(), plain.compact()))
        plain.check()


@pytest.mark.parametrize("seed", range(4))
def test_reordered_beams(seed):
    """Every beam goes on as one of the beams: nothing is lost, at most one copy less than heirs."""
    r = np.random.RandomState(seed)
    table, plain = pair(300, 32, 12, 9)
    offsets = (50 * np.arange(13)).tolist()
    table.append(int32(offsets), 600), plain.append(offsets, 600)
    for _ in range(6):
        parents, children = r.randint(0, 12, 12).tolist(), r.permutation(12).tolist()
        same(table, plain, *zip(table.fork(int32(parents), int32(children)), plain.fork(parents, children)))
        step = np.arange(13).tolist()
        same(table, plain, (table.append(int32(step), 12), plain.append(step, 12)))
        plain.check()


def test_many_tokens_and_offsets_off_the_end():
    table, plain = pair(2000, 32, 5, 1000)
    offsets = [0, 20000, 20000, 20001, 26000, 26001]
    same(table, plain, (table.append(int32(offsets), 26001), plain.append(offsets, 26001)))
    table, plain = pair(64, 32, 3, 10)                # outside [0, tokens] the nearer end
    same(table, plain, (table.append(int32([-5, 10, 40, 99]), 50), plain.append([0, 10, 40, 50], 50)))


def test_a_table_written_by_hand_is_clamped():
    table, _ = pair(4, 32, 3, 2)
    table.table.copy_(int32([[7, -9], [2 ** 31 - 1, 3], [0, 1]]))
    table.lengths.copy_(int32([64, 10 ** 9, -4]))
    table.uses.copy_(int32([0, 0, 0, 1]))
    assert table.append(int32([0, 0, 0, 2]), 2).tolist() == [0, 1]
    table.fork(int32([0, 1]), int32([2, 0]))
    table.compact()
    table.free(int32([0, 1, 2]))
    assert table.lengths.tolist() == [0, 0, 0]


HELD = [torch.int8, torch.float8_e4m3fn, torch.float16, torch.bfloat16]


def filled(pages, heads, dim, held, page, seed):
    import sparse
    cache = sparse.KeyValueCache(pages, heads, dim, dtype=held, page=page)
    for i, t in enumerate(buffers(cache)):
        t.copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed + i)))
    return cache


def buffers(cache):
    return [t.view(torch.uint8) for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales) if t is not None]


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 32), (3, 128, 64), (2, 64, 256), (5, 128, 128)])
def test_copies(heads, dim, page, held):
    cache, other = filled(9, heads, dim, held, page, 1), filled(6, heads, dim, held, page, 7)
    sources, targets = [0, 5, -1, 3, 9, 1, 2 ** 31 - 1, 5], [8, 7, 2, -1, 6, 9, 4, 6]
    for to in (cache, other):
        before, origin = [t.clone() for t in buffers(to)], [t.clone() for t in buffers(cache)]
        to.copy(int32(sources), int32(targets), origin=None if to is cache else cache)
        for now, was, first in zip(buffers(to), before, origin):
            for a, b in zip(sources, targets):
                if 0 <= a < 9 and 0 <= b < to.pages:
                    was[b] = first[a]
            assert torch.equal(now, was)


def test_many_copies():
    cache = filled(700, 2, 64, torch.int8, 32, 3)
    before = [t.clone() for t in buffers(cache)]
    sources, targets = np.arange(350), np.random.RandomState(1).permutation(350) + 350
    cache.copy(int32(sources), int32(targets))
    for now, was in zip(buffers(cache), before):
        was[torch.tensor(targets, device="cuda")] = was[torch.tensor(sources, device="cuda")]
        assert torch.equal(now, was)


def attend(cache, table, sequences, seed=1, heads=2, group=2, dim=64):
    import sparse
    q, k, v = normal(seed, sequences, 1, heads * group, dim), normal(seed + 1, sequences, 1, heads, dim), normal(seed + 2, sequences, 1, heads, dim)
    return sparse.cached_attention(q, k, v, cache, table.table, table.lengths, scale=0.125)


@pytest.mark.parametrize("held", [torch.int8, torch.float16])
def test_a_batch_that_is_served(held):
    """A hybrid model's two kinds of layers together: prompts, continuations, steps, answers that end, pages that move.  What each
    sequence attends to is at every point what one that never shared or moved a page attends to."""
    import sparse
    heads, dim, page, sequences = 2, 64, 32, 6
    table, plain = pair(60, page, sequences, 10)
    caches = [sparse.KeyValueCache(60, heads, dim, dtype=held, page=page) for _ in range(2)]
    log_decay = -torch.tensor([0.01, 0.2], device="cuda")
    states = torch.zeros(sequences, heads, dim, dim, device="cuda")
    rows = [[] for _ in range(sequences)]             # (layer rows of k, v) of every token, and the recurrent layer's
    kept = [torch.zeros(0, 2, heads, dim, dtype=torch.float16, device="cuda")] * sequences

    def grow(lengths, seed):
        offsets, tokens = [0] + np.cumsum(lengths).tolist(), sum(lengths)
        k, v, q = (normal(seed + i, tokens, heads, dim) for i in range(3))
        slots = table.append(int32(offsets), tokens)
        plain.append(offsets, tokens)
        for layer, cache in enumerate(caches):
            cache.write(k if layer == 0 else v, v if layer == 0 else k, slots)
        for b in range(sequences):
            kept[b] = torch.cat([kept[b], torch.stack([k, v], 1)[offsets[b]:offsets[b + 1]]])
        if max(lengths) <= 1:                         # a step: idle sequences have slot -1
            at = int32([b if n else -1 for b, n in enumerate(lengths)])
            full = [torch.zeros(sequences, heads, dim, dtype=torch.float16, device="cuda") for _ in range(3)]
            busy = torch.tensor([b for b, n in enumerate(lengths) if n], device="cuda")
            for to, t in zip(full, (q, k, v)):
                to[busy] = t
            sparse.linear_attention_step(*full, log_decay, states, at, scale=0.125)
        else:
            _, last = sparse.packed_linear_attention(q, k, v, log_decay, int32(offsets), scale=0.125, states=states, return_states=True)
            states.copy_(last)

    def fork(parents, children):
        moves = table.fork(int32(parents), int32(children))
        plain.fork(parents, children)
        for cache in caches:
            cache.copy(*moves)
        states[torch.tensor(children, device="cuda")] = states[torch.tensor(parents, device="cuda")]
        was = list(kept)
        for a, c in zip(parents, children):
            kept[c] = was[a]

    def agree():
        same(table, plain)
        plain.check()
        # caches that hold each sequence by itself, written at once
        per = 10
        own = [sparse.KeyValueCache(sequences * per, heads, dim, dtype=held, page=page) for _ in range(2)]
        alone, plain_alone = pair(sequences * per, page, sequences, per)
        lengths = [len(t) for t in kept]
        offsets = [0] + np.cumsum(lengths).tolist()
        slots, every = alone.append(int32(offsets), sum(lengths)), torch.cat(kept)
        for layer, cache in enumerate(own):
            if sum(lengths):
                cache.write(every[:, layer].contiguous(), every[:, 1 - layer].contiguous(), slots)
        for layer in range(2):
            assert torch.equal(attend(caches[layer], table, sequences, 5 + layer), attend(own[layer], alone, sequences, 5 + layer))
        _, last = sparse.packed_linear_attention(torch.zeros_like(every[:, 0]), every[:, 0].contiguous(), every[:, 1].contiguous(), log_decay,
                                                 int32(offsets), return_states=True)
        # by chunks or token by token: fp32 sums of the same terms
        assert (torch.linalg.norm(states - last) <= 1e-5 * torch.linalg.norm(last)).item()

    def end(which):
        table.free(int32(which))
        plain.free(which)
        for b in which:
            kept[b] = kept[b][:0]
            states[b] = 0

    grow([70, 0, 33, 0, 0, 0], 10)
    agree()
    fork([0, 0, 2], [1, 3, 4])
    agree()
    for t in range(3):
        grow([1, 1, 0, 1, 1, 0], 20 + 3 * t)
    agree()
    fork([3, 1, 3, 0], [0, 1, 3, 5])                  # beams in another order, one twice
    agree()
    end([2, 4])
    for cache, moves in zip(caches, [table.compact()] * 2):
        cache.copy(*moves)
    plain.compact()
    agree()
    grow([1, 1, 100, 1, 0, 1], 40)
    agree()
    # into a smaller cache: what is used are the lowest pages
    used = int((table.uses > 0).sum())
    smaller = sparse.KeyValueCache(used, heads, dim, dtype=held, page=page)
    for cache, moves in zip(caches, [table.compact()] * 2):
        cache.copy(*moves)
    smaller.copy(int32(range(used)), int32(range(used)), origin=caches[0])
    assert torch.equal(attend(smaller, table, sequences), attend(caches[0], table, sequences))


def test_captured_calls():
    """Growth, a fork and what it copies, in one graph: replays go on from the table as it is."""
    import sparse
    table, plain = pair(200, 32, 6, 8)
    cache = sparse.KeyValueCache(200, 1, 64, dtype=torch.float16, page=32)
    offsets, parents, children, ends = int32([0, 1, 2, 3, 4, 5, 6]), int32([0, 2, 4]), int32([1, 3, 5]), int32([-1])
    k = normal(1, 40, 1, 64)

    def work():
        slots = table.append(offsets, 40)
        cache.write(k, k, slots)
        moves = table.fork(parents, children)
        cache.copy(*moves)
        table.free(ends)
        return (slots, *moves)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work()
    r = np.random.RandomState(0)
    for _ in range(7):
        new = r.randint(0, 7, 6)
        o = [0] + np.cumsum(new).tolist()
        a, c = r.randint(0, 6, 3).tolist(), r.permutation(6)[:3].tolist()
        e = int(r.randint(-1, 6))
        for t, x in ((offsets, o), (parents, a), (children, c), (ends, [e])):
            t.copy_(int32(x))
        graph.replay()
        torch.cuda.synchronize()
        expected = (plain.append(o, 40), *plain.fork(a, c))
        plain.free([e])
        same(table, plain, *zip(captured, expected))


def test_on_another_stream_and_copies_of_a_table():
    table, plain = pair(30, 32, 4, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        slots = table.append(int32([0, 40, 40, 45, 46]), 46)
    side.synchronize()
    same(table, plain, (slots, plain.append([0, 40, 40, 45, 46], 46)))
    for other in (copy.deepcopy(table), pickle.loads(pickle.dumps(table))):
        other.free(int32([0]))
        assert other.lengths.tolist() == [0, 0, 5, 1] and table.lengths.tolist() == [40, 0, 5, 1]


@pytest.mark.parametrize("call,error,needle", [
    (lambda t: t.append(int32([0, 1]), 1), ValueError, "5 entries"),
    (lambda t: t.append(int32([0, 1, 1, 1, 1]).long(), 1), ValueError, "int32"),
    (lambda t: t.append(int32([0, 1, 1, 1, 1]).cpu(), 1), ValueError, "GPU of the operands"),
    (lambda t: t.append(int32([0, 1, 1, 1, 1]), -1), ValueError, "tokens"),
    (lambda t: t.free(int32([[0]])), ValueError, "which must"),
    (lambda t: t.free(int32([0] * 4097)), ValueError, "at most 4096"),
    (lambda t: t.fork(int32([0]), int32([1, 2])), ValueError, "1 parents and 2"),
    (lambda t: t.fork([0], int32([1])), ValueError, "parents must"),
    (lambda t: t.fork(int32([0]), int32([1]).cpu()), ValueError, "GPU of the operands"),
])
def test_refusals(call, error, needle):
    table, plain = pair(10, 32, 4, 3)
    with pytest.raises(error, match=needle):
        call(table)
    same(table, plain)


@pytest.mark.parametrize("given,needle", [
    (dict(page=48), "page must"), (dict(pages=0), "addressed"), (dict(pages=2 ** 26), "addressed"), (dict(sequences=0), "too large"),
    (dict(sequences=4097), "too large"), (dict(width=0), "too large"), (dict(width=2 ** 26), "too large"), (dict(device="cpu"), "on the GPU")])
def test_tables_that_cannot_be(given, needle):
    import sparse
    with pytest.raises(ValueError, match=needle):
        sparse.PageTable(**{**dict(pages=10, page=32, sequences=4, width=3), **given})


@pytest.mark.parametrize("make,error,needle", [
    (lambda c: c.copy(int32([0]), int32([1, 2])), ValueError, "1 sources and 2"),
    (lambda c: c.copy(int32([0]), int32([1]).long()), ValueError, "targets must"),
    (lambda c: c.copy(int32([0]).cpu(), int32([1])), ValueError, "GPU of the operands"),
    (lambda c: c.copy(int32([0]), int32([1]), origin=filled(3, 2, 64, torch.float16, 32, 1)), ValueError, "dtype"),
    (lambda c: c.copy(int32([0]), int32([1]), origin=filled(3, 1, 64, torch.int8, 32, 1)), ValueError, "heads"),
    (lambda c: c.copy(int32([0]), int32([1]), origin=filled(3, 2, 128, torch.int8, 32, 1)), ValueError, "head_dim"),
    (lambda c: c.copy(int32([0]), int32([1]), origin=filled(3, 2, 64, torch.int8, 64, 1)), ValueError, "page"),
    (lambda c: c.copy(int32([0]), int32([1]), origin=c.keys), TypeError, "KeyValueCache"),
])
def test_copy_refusals(make, error, needle):
    with pytest.raises(error, match=needle):
        make(filled(4, 2, 64, torch.int8, 32, 1))


def test_nothing_to_do():
    table, plain = pair(1, 32, 1, 1)
    none = int32([])
    assert table.append(int32([0, 0]), 0).numel() == 0 and table.compact()[0].numel() == 0
    table.free(none)
    assert table.fork(none, none)[0].numel() == 0
    filled(2, 1, 64, torch.int8, 32, 1).copy(none, none)
    same(table, plain)


def test_the_largest_table():
    """4096 sequences and as many entries: every one a child of one of a few, then what is left moves together."""
    table, plain = pair(9000, 32, 4096, 4)
    new = np.zeros(4096, int)
    new[::512] = np.arange(8) * 15 + 1
    offsets = [0] + np.cumsum(new).tolist()
    same(table, plain, (table.append(int32(offsets), offsets[-1]), plain.append(offsets, offsets[-1])))
    parents, children = (512 * (np.arange(4096) * 7 % 8)).tolist(), np.arange(4096)[::-1].tolist()
    same(table, plain, *zip(table.fork(int32(parents), int32(children)), plain.fork(parents, children)))
    gone = np.arange(0, 4096, 3).tolist()
    plain.free(gone)
    table.free(int32(gone))
    same(table, plain, *zip(table.compact(), plain.compact()))
    plain.check()
