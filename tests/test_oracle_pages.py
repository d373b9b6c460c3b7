"""CPU: the restatement of a page table against hand-derived tables and its own invariants over drawn calls."""
import numpy as np

from oracle.pages_oracle import Pages


def empty(sequences, width, pages, page):
    return Pages(np.full((sequences, width), -1, dtype=np.int32), np.zeros(sequences, int), np.zeros(pages, int), page)


def test_known_answers():
    p = empty(4, 3, 8, 32)
    assert list(p.append([0, 33, 33, 65, 65], 66)) == list(range(33)) + [64 + i for i in range(32)] + [-1]
    assert p.table().tolist() == [[0, 1, -1], [-1] * 3, [2, -1, -1], [-1] * 3] and p.lengths == [33, 0, 32, 0]
    assert [x.tolist() for x in p.fork([0, 0, 2], [1, 3, 9])] == [[1, 1, -1], [3, 4, -1]]
    assert p.table().tolist() == [[0, 1, -1], [0, 3, -1], [2, -1, -1], [0, 4, -1]] and p.uses == [3, 1, 1, 1, 1, 0, 0, 0]
    p.check()
    p.free([0, 0, 2, -1])
    assert p.uses == [2, 0, 0, 1, 1, 0, 0, 0]
    assert [x.tolist() for x in p.compact()] == [[3, 4, -1, -1], [1, 2, -1, -1]]
    assert p.table().tolist() == [[-1] * 3, [0, 1, -1], [-1] * 3, [0, 2, -1]]
    # a beam that goes on as two, and takes the other's place: the first heir keeps the last page
    assert [x.tolist() for x in p.fork([1, 1], [3, 1])] == [[-1, 1], [-1, 2]]
    p.check()


def test_requests_that_cannot_be_met():
    p = empty(3, 2, 3, 32)
    assert (p.append([0, 40, 80, 90], 90)[[0, 39, 40, 79, 80, 89]] == [0, 39, -1, -1, -1, -1]).all() and p.missing == 2
    p.append([0, 25, 25, 25], 25)                     # more than its row has
    assert p.missing == 3 and p.lengths == [40, 0, 0]
    p.check()


def test_drawn_calls_keep_the_invariants():
    r = np.random.RandomState(1)
    for _ in range(30):
        sequences, page = r.randint(1, 9), int(r.choice([32, 64]))
        p = empty(sequences, r.randint(1, 6), r.randint(1, 40), page)
        for _ in range(12):
            kind = r.randint(4)
            if kind == 0:
                new = r.randint(0, 3 * page, sequences) * r.randint(0, 2, sequences)
                p.append([0] + np.cumsum(new).tolist(), int(new.sum()))
            elif kind == 1:
                p.free(r.randint(-1, sequences + 1, r.randint(0, 4)).tolist())
            elif kind == 2:
                n = r.randint(0, 2 * sequences)
                p.fork(r.randint(-1, sequences + 1, n).tolist(), r.randint(-1, sequences + 1, n).tolist())
            else:
                p.compact()
                used = sum(1 for n in p.uses if n)
                assert all(p.uses[:used]) and not any(p.uses[used:])
            p.check()
