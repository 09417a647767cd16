"""The page bookkeeping of a key/value cache (mx4_pages_*): forks share, writes
copy, nothing is lost. Host code, no GPU."""
import random

import pytest


@pytest.fixture(scope="module")
def mx4():
    import mx4hip

    return mx4hip


def test_grow_fork_write_trim_close(mx4):
    p = mx4.Pages(8, 16)
    a = p.open()
    assert p.table(a) == (0, [])
    assert p.write(a, 0, 40) == [] and p.table(a) == (40, [0, 1, 2]) and p.free_count() == 5
    b = p.fork(a)
    assert p.table(b) == (40, [0, 1, 2]) and p.free_count() == 5
    # the page that holds 32..39 is shared: b writes from 40 into it, so it is copied
    assert p.write(b, 40, 49) == [(2, 3)] and p.table(b) == (49, [0, 1, 3, 4])
    # a has its page 2 alone now
    assert p.write(a, 40, 41) == [] and p.table(a) == (41, [0, 1, 2])
    # written from its first row on, a shared page is replaced without a copy, and what came behind is gone
    assert p.write(b, 16, 17) == [] and p.table(b) == (17, [0, 5])
    p.trim(b, 16)
    assert p.table(b) == (16, [0]) and p.free_count() == 5
    p.close_sequence(a)
    assert p.free_count() == 7
    p.close_sequence(b)
    assert p.free_count() == 8


def test_lengths_zero_and_one(mx4):
    p = mx4.Pages(1, 16)
    a = p.open()
    assert p.write(a, 0, 0) == [] and p.free_count() == 1
    assert p.write(a, 0, 1) == [] and p.table(a) == (1, [0])
    assert p.write(a, 1, 1) == [] and p.table(a) == (1, [0])
    p.trim(a, 1)
    p.trim(a, 0)
    assert p.table(a) == (0, []) and p.free_count() == 1


def test_refusals_change_nothing(mx4):
    for args in [(0, 16), (4, 8), (4, 24), (4, 8192)]:
        with pytest.raises(mx4.Mx4Error):
            mx4.Pages(*args)
    p = mx4.Pages(3, 16)
    a = p.open()
    p.write(a, 0, 20)
    b = p.fork(a)
    before = p.table(a), p.table(b), p.free_count()
    with pytest.raises(mx4.Mx4Error, match="NO_MEMORY"):
        p.write(b, 20, 60)  # a copy and two more: one is free
    for call in [lambda: p.write(a, 21, 30), lambda: p.write(a, 5, 4), lambda: p.trim(a, 21), lambda: p.write(99, 0, 1),
                 lambda: p.fork(99), lambda: p.close_sequence(99), lambda: p.table(99), lambda: p.trim(99, 0)]:
        with pytest.raises(mx4.Mx4Error, match="ARGUMENT"):
            call()
    assert (p.table(a), p.table(b), p.free_count()) == before
    assert p.write(b, 20, 32) == [(1, 2)]


@pytest.mark.parametrize("seed", range(6))
def test_against_contents(mx4, seed):
    """Random traffic on a model of the pages' contents: every sequence reads
    back what it wrote, whatever its relatives do, and no page is lost."""
    rng = random.Random(seed)
    pages, size = rng.choice([(7, 16), (40, 16), (64, 32)])
    p = mx4.Pages(pages, size)
    memory = {}  # (page, row): token
    want = {}
    fresh = 0
    for _ in range(400):
        kind = rng.choice(["open", "fork", "write", "write", "write", "trim", "close", "compact"])
        if kind == "open" and len(want) < 6:
            want[p.open()] = []
        elif kind == "fork" and want and len(want) < 6:
            s = rng.choice(list(want))
            want[p.fork(s)] = list(want[s])
        elif kind == "write" and want:
            s = rng.choice(list(want))
            start = rng.randint(max(0, len(want[s]) - 5), len(want[s]))
            end = start + rng.choice([0, 1, 3, size, 3 * size])
            try:
                copies = p.write(s, start, end)
            except mx4.Mx4Error as e:
                assert "too few free pages" in str(e)
                continue
            for a, b in copies:
                for r in range(size):
                    memory[b, r] = memory.get((a, r))
            table = p.table(s)[1]
            del want[s][start:]
            for at in range(start, end):
                fresh += 1
                want[s].append(fresh)
                memory[table[at // size], at % size] = fresh
        elif kind == "trim" and want:
            s = rng.choice(list(want))
            n = rng.randint(0, len(want[s]))
            p.trim(s, n)
            del want[s][n:]
        elif kind == "close" and len(want) > 2:
            s = rng.choice(list(want))
            p.close_sequence(s)
            del want[s]
        elif kind == "compact":
            pairs = p.compact()
            ends = {b for _, b in pairs}
            assert len(ends) == len(pairs) and not ends & {a for a, _ in pairs}
            for a, b in pairs:
                for r in range(size):
                    memory[b, r] = memory.get((a, r))
            used = sorted({q for s in want for q in p.table(s)[1]})
            assert used == list(range(len(used)))
        for s, tokens in want.items():
            n, table = p.table(s)
            assert n == len(tokens) and len(table) == -(-n // size)
            assert [memory[table[i // size], i % size] for i in range(n)] == tokens
        assert p.free_count() == pages - len({q for s in want for q in p.table(s)[1]})
