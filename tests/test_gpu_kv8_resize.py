"""Lengths, block tables and the list of free blocks on the device against the same bookkeeping in plain lists."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 64


def i32(x, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device="cuda")
    return t if shape is None else t.view(shape)


class Books:
    """What the operator does, in lists."""

    def __init__(self, batch, width, pool, shared=0, seed=0, lens=None):
        rng = random.Random(seed)
        order = list(range(pool))
        rng.shuffle(order)
        self.shared, self.width = shared, width
        self.lens = [shared * BLOCK] * batch if lens is None else list(lens)
        self.table = [order[:shared] + [-7] * (width - shared) for _ in range(batch)]
        self.stack, self.count, self.capacity = order[shared:] + [-9] * shared, pool - shared, pool
        for i, n in enumerate(self.lens):
            for j in range(shared, self.blocks(n)):
                self.count -= 1
                self.table[i][j] = self.stack[self.count]

    def blocks(self, n):
        return max(-(-n // BLOCK), self.shared)

    def change(self, by, rows=None):
        """(cu_tokens, positions, slots, status)"""
        after = [max(n + c, 0) for n, c in zip(self.lens, by)]
        had, needed = [self.blocks(n) for n in self.lens], [self.blocks(n) for n in after]
        new = [max(b - a, 0) for a, b in zip(self.lens, after)]
        back, taken = (sum(max(0, s * (a - b)) for a, b in zip(had, needed)) for s in (1, -1))
        status = 0
        if max(had + needed, default=0) > self.width:
            status = -1
        elif sum(new) > (2 ** 31 - 1 if rows is None else rows):
            status = -2
        elif not 0 <= self.count <= self.capacity - back:
            status = -3
        elif taken > self.count + back:
            status = taken - self.count - back
        cu, positions, slots = [0], [], []
        if status:
            cu = [0] * (len(by) + 1)
        else:
            for i, j in reversed([(i, j) for i in range(len(by)) for j in range(needed[i], had[i])]):
                self.stack[self.count] = self.table[i][j]
                self.count += 1
            for i in range(len(by)):
                for j in range(had[i], needed[i]):
                    self.count -= 1
                    self.table[i][j] = self.stack[self.count]
                for p in range(self.lens[i], after[i]):
                    positions.append(p)
                    slots.append(self.table[i][p // BLOCK] * BLOCK + p % BLOCK)
                self.lens[i] = after[i]
                cu.append(cu[-1] + new[i])
        if rows is not None:
            positions, slots = positions + [0] * (rows - len(positions)), slots + [-1] * (rows - len(slots))
        return cu, positions, slots, status

    def tensors(self):
        batch = len(self.lens)
        return (i32(self.table, (batch, self.width)), i32(self.lens, (batch,)), i32(self.stack, (self.capacity,)), i32([self.count]))


def check(got, want, state, books, rows):
    cu, positions, slots, status = got
    assert status.tolist() == [want[3]] and cu.tolist() == want[0]
    assert cu.dtype == status.dtype == torch.int32
    if rows is None:
        assert positions is None and slots is None
    else:
        assert positions.dtype == slots.dtype == torch.int64
        assert positions.tolist() == want[1] and slots.tolist() == want[2]
    for t, x in zip(state, (books.table, books.lens, books.stack, [books.count])):
        assert t.tolist() == x


@pytest.fixture(scope="module")
def resize(hip_lib):
    from latentq_llm_amd import ops
    return ops.kv8_resize


@pytest.mark.parametrize("batch, shared, longest", [(1, 0, 70), (1, 3, 5), (2, 0, 500), (5, 2, 130), (63, 0, 9), (64, 0, 64), (65, 1, 200), (300, 0, 3), (1024, 0, 3), (1025, 0, 3),
                                                    (4096, 1, 2)])
def test_steps_of_all_kinds(resize, batch, shared, longest):
    """Sequences grow, shrink, stay, are dropped and begin again; each pass is checked with all that it leaves."""
    rng = random.Random(batch)
    width = shared + 3 * longest // BLOCK + 4
    books = Books(batch, width, shared + batch * 2 * (longest // BLOCK + 1) + 3, shared, seed=batch)
    state = books.tensors()
    seen = set()
    for n in range(6 if batch > 1000 else 12):
        by = [rng.choice((0, 1, rng.randint(1, longest), rng.randint(1, longest), -rng.randint(1, longest), -1, shared * BLOCK - length if length > shared * BLOCK else 0))
              for length in books.lens]
        total = sum(max(0, max(a + c, 0) - a) for a, c in zip(books.lens, by))
        rows = None if n % 3 == 0 else total + n % 2 * 7
        want = books.change(by, rows)
        seen.add(min(want[3], 1))
        check(resize(*state, i32(by), rows=rows, shared=shared), want, state, books, rows)
        there = [b for row, length in zip(books.table, books.lens) for b in row[shared:books.blocks(length)]] + books.stack[:books.count]
        assert len(set(there)) == len(there)  # no block in two places
    assert 0 in seen


@pytest.mark.parametrize("lens, by", [([0], [20000]), ([5000], [15000]), ([1, 0, 700], [4096, 4095, 9000]), ([10, 0, 63], [0, 4097, 0])])
def test_many_rows(resize, lens, by):
    books = Books(len(lens), 400, 800, seed=3, lens=lens)
    state = books.tensors()
    for rows in (sum(by), ):
        want = books.change(by, rows + 100)
        check(resize(*state, i32(by), rows=rows + 100), want, state, books, rows + 100)


def test_many_rows_of_many_sequences(resize):
    by = [i % 5 for i in range(4096)]
    books = Books(4096, 2, 5000, seed=4)
    state = books.tensors()
    want = books.change(by, sum(by))
    check(resize(*state, i32(by), rows=sum(by)), want, state, books, sum(by))


def test_what_is_taken_and_given_back_leaves_the_list(resize):
    books = Books(7, 40, 300, 2, seed=5, lens=[128, 700, 130, 192, 1000, 129, 128])
    state = books.tensors()
    before = [t.clone() for t in state]
    by = [300, 64, 0, 1, 63, 500, 2]
    resize(*state, i32(by), shared=2)
    assert not torch.equal(state[3], before[3])
    resize(*state, i32([-x for x in by]), shared=2)
    assert all(torch.equal(a, b) for a, b in zip(state[1:], before[1:]))


def test_blocks_given_back_are_there_for_the_same_call(resize):
    books = Books(2, 10, 5, seed=6, lens=[320, 0])
    state = books.tensors()
    want = books.change([-320, 320], 320)
    assert want[3] == 0
    check(resize(*state, i32([-320, 320]), rows=320), want, state, books, 320)


@pytest.mark.parametrize("what, by, rows, status", [
    ("missing", [64, 200, 0], 300, 3), ("missing", [200, 0, 0], None, 2), ("narrow", [0, 0, 1000], 2000, -1), ("narrow", [2 ** 31 - 1, 0, 0], None, -1), ("rows", [10, 10, 10], 29, -2),
    ("rows", [0, 0, 1], 0, -2)])
def test_what_cannot_be_done_changes_nothing(resize, what, by, rows, status):
    books = Books(3, 8, 8, seed=7, lens=[64, 64, 100])
    if what == "missing":
        books.count = 2
    state = books.tensors()
    before = [t.clone() for t in state]
    want = books.change(by, rows)
    assert want[3] == status
    check(resize(*state, i32(by), rows=rows), want, state, books, rows)
    assert all(torch.equal(a, b) for a, b in zip(state, before))


def test_many_rows_of_a_call_that_cannot_be_done(resize):
    books = Books(3, 200, 100, seed=9, lens=[64, 64, 100])
    state = books.tensors()
    want = books.change([5000, 4000, 0], 9001)
    assert want[3] > 0
    check(resize(*state, i32([5000, 4000, 0]), rows=9001), want, state, books, 9001)


@pytest.mark.parametrize("count, by", [(-1, [0]), (9, [0]), (8, [-64]), (2 ** 31 - 1, [-64]), (-2 ** 31, [64])])
def test_a_broken_list(resize, count, by):
    table, lens, stack = i32([[3, 4]]), i32([64]), i32(list(range(8)))
    n = i32([count])
    got = resize(table, lens, stack, n, i32(by), rows=70)
    assert got[3].item() == -3 and got[0].tolist() == [0, 0] and got[2].tolist() == [-1] * 70
    assert lens.tolist() == [64] and n.tolist() == [count] and stack.tolist() == list(range(8)) and table.tolist() == [[3, 4]]


@pytest.mark.parametrize("length, by, status", [(-5, 10, 0), (-2 ** 31, -2 ** 31, 0), (2 ** 31 - 1, 2 ** 31 - 1, -1), (2 ** 31 - 1, -(2 ** 31 - 1), -1), (129, 0, -1)])
def test_broken_lengths(resize, length, by, status):
    """A negative length counts as none; one beyond the table's columns is refused as it stands."""
    table, lens, stack, n = i32([[3, 4]]), i32([length]), i32(list(range(8))), i32([2])
    got = resize(table, lens, stack, n, i32([by]))
    assert got[3].item() == status
    assert lens.item() == (max(max(length, 0) + by, 0) if status == 0 else length)


def test_no_sequences(resize):
    empty = i32([], (0, 4)), i32([]), i32([1, 2]), i32([2])
    got = resize(*empty, i32([]), rows=5)
    assert got[0].tolist() == [0] and got[1].tolist() == [0] * 5 and got[2].tolist() == [-1] * 5 and got[3].item() == 0


def test_another_stream_and_a_graph(resize):
    books = Books(9, 30, 300, 1, seed=8, lens=[64 + 50 * i for i in range(9)])
    state = books.tensors()
    by, back = i32([5, 0, 64, 1, 2, 3, 200, 0, 6]), i32([-2, 0, -63, 0, 0, -3, -150, 0, -5])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = resize(*state, by, rows=300, shared=1)
    torch.cuda.current_stream().wait_stream(stream)
    check(got, books.change(by.tolist(), 300), state, books, 300)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = resize(*state, by, rows=300, shared=1)
        second = resize(*state, back, shared=1)
    for n in range(5):
        graph.replay()
        one = books.change(by.tolist(), 300)
        two = books.change(back.tolist())
        assert one[3] == two[3] == 0
        torch.cuda.synchronize()
        assert first[0].tolist() == one[0] and first[1].tolist() == one[1] and first[2].tolist() == one[2]
        check(second, two, state, books, None)
        if n == 2:  # an eager call between the replays
            check(resize(*state, back, rows=3, shared=1), books.change(back.tolist(), 3), state, books, 3)


def test_refusals(resize):
    def args(**change):
        a = dict(table=i32([[0, 1]] * 3), lens=i32([0] * 3), free=i32([4, 5]), count=i32([2]), change=i32([1] * 3))
        a.update(change)
        return list(a.values())

    for kind, change, more in ((TypeError, dict(lens=i32([0] * 3).long()), {}), (ValueError, dict(lens=i32([0] * 2)), {}), (ValueError, dict(change=i32([0] * 4)), {}),
                               (ValueError, dict(count=i32([1, 2])), {}), (ValueError, dict(free=i32([[1, 2]])), {}), (ValueError, dict(table=i32([0, 1])), {}),
                               (ValueError, dict(table=i32([[0, 1]] * 6)[::2]), {}), (ValueError, {}, dict(rows=-1)), (ValueError, {}, dict(rows=1 << 31)),
                               (ValueError, {}, dict(shared=3)), (ValueError, {}, dict(shared=-1)), (Exception, dict(table=torch.zeros((3, 2), dtype=torch.int32)), {}),
                               ((TypeError, ValueError), {}, dict(rows="x"))):
        with pytest.raises(kind):
            resize(*args(**change), **more)
    with pytest.raises(RuntimeError, match="cannot be recorded in a trace"):
        torch.jit.trace(lambda x: resize(*args(change=x))[0], i32([0] * 3), check_trace=False)
    same = i32([0] * 3)
    from latentq_llm_amd import _C
    with pytest.raises(_C.LatentQError, match="overlap"):
        resize(*args(lens=same, change=same))
    with pytest.raises(_C.LatentQError, match="4096"):
        resize(i32([[0]] * 4097), i32([0] * 4097), i32([1]), i32([1]), i32([0] * 4097))
