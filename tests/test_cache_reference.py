"""The books that the kernels are held to: no page is lost, none is written by two requests, and every request keeps its tokens."""

import random

from tests.cache_reference import Books


def test_books():
    rng = random.Random(0)
    for _ in range(40):
        page, batch = rng.choice((1, 3, 4, 16)), rng.choice((1, 2, 5, 9))
        books = Books(200, page, batch, 60)
        want = [[] for _ in range(batch)]
        for step in range(15):
            new = [[(step, b, i) for i in range(rng.randint(0, 7))] for b in range(batch)]
            books.append(new)
            want = [w + n for w, n in zip(want, new)]
            if step % 2:
                parents = [rng.choice((b, rng.randrange(batch), rng.randrange(batch), -1)) for b in range(batch)]
                books.fork(parents)
                want = [list(want[s]) if s >= 0 else [] for s in parents]
            if step % 5 == 4:
                books.compact(rng.choice((200, 250)))
            assert [books.values(b) for b in range(batch)] == want
            held = {p for t in books.tables for p in t}
            assert held.isdisjoint(books.free) and len(held) + len(books.free) == books.pages and len(set(books.free)) == len(books.free)


def test_a_few_by_hand():
    books = Books(6, 2, 3, 9)
    books.append([[1, 2, 3], [4], []])
    assert books.tables == [[0, 1], [2], []] and books.free == [3, 4, 5]
    books.fork([0, 0, 0])  # the second request's page is free, and the last one taken
    assert books.tables == [[0, 1], [0, 3], [0, 4]] and books.free == [5, 2] and books.shares() == [2, 0, 0, 0, 0, 0]
    books.append([[5], [6], [7]])
    assert [books.values(b) for b in range(3)] == [[1, 2, 3, 5], [1, 2, 3, 6], [1, 2, 3, 7]]
    books.fork([1, 1, -1])
    assert books.tables == [[0, 3], [0, 3], []] and books.free == [5, 2, 1, 4] and books.shares() == [1, 0, 0, 1, 0, 0]
    books.append([[8, 9, 10], [], []])
    books.fork([0, 0, 0])
    assert books.tables == [[0, 3, 5, 2], [0, 3, 5, 1], [0, 3, 5, 4]] and books.free == []
    books.append([[11], [12, 13], []])
    books.fork([-1, 2, 2])  # two free pages, of which one is taken
    assert books.lengths == [0, 7, 7] and books.tables[2] == [0, 3, 5, 4] and books.tables[1] == [0, 3, 5, 2] and books.free == [1]
    books = Books(3, 2, 3, 9)
    books.append([[1, 2, 3, 4, 5], [], []])
    books.fork([0, 0, 0])
    assert books.lengths == [5, 4, 4] and books.tables == [[0, 1, 2], [0, 1], [0, 1]]
    books.compact(1)
    assert books.lengths == [2, 2, 2] and books.tables == [[0], [0], [0]] and books.free == [] and books.shares() == [2]
