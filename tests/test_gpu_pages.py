"""Pages of a shared cache (enx_pages_*) against the host twin, entry for entry: all results are
integers, so every comparison is exact."""

import random

import pytest
import torch

from enargeia_b200 import kernels as K
from enargeia_b200._lib import EnxError
from pages_twin import BAD_LIST, NONE_FREE, Pages

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Both:
    """The same operations on the device and on the twin, compared after each."""

    def __init__(self, rows, width, pages, page):
        self.twin = Pages(rows, width, pages, page)
        self.table = i32(self.twin.table)
        self.lengths, self.refs, self.status = i32([0] * rows), i32([0] * pages), i32([0])
        self.pairs, self.count = i32([[-7, -7]] * max(rows, pages)), i32([-7, -7])
        self.page = page

    def same(self):
        assert self.table.tolist() == self.twin.table
        assert self.lengths.tolist() == self.twin.lengths
        assert self.refs.tolist() == self.twin.refs
        assert self.status.item() == self.twin.status

    def free(self, rows, keep):
        K.pages_free(self.table, self.lengths, self.refs, i32(rows), i32(keep), self.status, self.page)
        self.twin.free(rows, keep)
        self.same()

    def fork(self, src, dst):
        K.pages_fork(self.table, self.lengths, self.refs, i32(src), i32(dst), self.status, self.page)
        self.twin.fork(src, dst)
        self.same()

    def _pairs(self, want, taken):
        assert self.count.tolist() == [len(want), taken]
        assert [tuple(p) for p in self.pairs[: len(want)].tolist()] == want
        assert (self.pairs[len(want):] == -7).all()
        self.pairs.fill_(-7)

    def grow(self, rows, add):
        K.pages_grow(self.table, self.lengths, self.refs, i32(rows), i32(add), self.pairs, self.count, self.status, self.page)
        self._pairs(*self.twin.grow(rows, add))
        self.same()

    def compact(self, in_place):
        table, refs = (self.table, self.refs) if in_place else (torch.zeros_like(self.table), torch.zeros_like(self.refs))
        K.pages_compact(self.table, self.lengths, self.refs, table, refs, self.pairs, self.count, self.status, self.page)
        self.table, self.refs = table, refs
        self._pairs(*self.twin.compact())
        self.same()


@pytest.mark.parametrize("rows,width,pages,page,seed", [(5, 3, 9, 16, 0), (40, 17, 300, 32, 1), (300, 40, 5000, 64, 2),
                                                        (1500, 8, 9000, 16, 3), (3, 700, 2100, 1, 4)])
def test_random_turns(gpu, rows, width, pages, page, seed):
    rng = random.Random(seed)
    b = Both(rows, width, pages, page)
    for turn in range(25):
        some = rng.sample(range(rows), rng.randint(1, rows))
        b.grow(some, [rng.randint(0, max(1, min(page * width - b.twin.lengths[r], 2 * page))) for r in some])
        empty = [r for r in range(rows) if b.twin.lengths[r] == 0]
        held = [r for r in range(rows) if b.twin.lengths[r]]
        if empty and held:
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            b.fork([rng.choice(held) for _ in dst], dst)
            # all holders of shared last pages write at once, and some of them
            again = rng.sample(range(rows), rng.randint(1, rows))
            b.grow(again, [min(rng.randint(0, 3), page * width - b.twin.lengths[r]) for r in again])
        some = rng.sample(range(rows), rng.randint(1, rows))
        b.free(some, [rng.choice([0, rng.randint(0, b.twin.lengths[r] + 1), 1 << 30]) for r in some])
        if turn % 6 == 5:
            b.compact(in_place=turn % 12 == 5)


def test_sole_holders_that_all_write(gpu):
    b = Both(4, 4, 12, 16)
    b.grow([0], [20])
    b.fork([0, 0, 0], [3, 1, 2])
    b.grow([2, 0, 3, 1], [1, 0, 1, 1])  # row 0 does not write: the three others copy
    b.grow([0], [1])  # and row 0 holds its page alone now
    assert b.count.tolist() == [0, 0]
    b.free([1, 2, 3], [0, 0, 0])
    b.fork([0], [1])
    b.grow([1, 0], [1, 1])  # both holders write: the first of the list keeps the page
    assert b.twin.table[1][1] == 1


def test_a_cut_into_shared_pages_is_copied_before_writing(gpu):
    b = Both(2, 8, 16, 16)
    b.grow([0], [64])
    b.fork([0], [1])
    b.free([1], [40])  # the middle of a full page that both hold
    b.grow([1], [3])
    assert b.count.tolist() == [1, 1]


def test_refusals_change_nothing(gpu):
    b = Both(4, 3, 5, 16)
    b.grow([0, 1], [33, 16])
    b.status.zero_()
    for call in (lambda: b.grow([2, 3], [16, 16]), lambda: b.grow([1], [40]), lambda: b.grow([2, 2], [1, 1]),
                 lambda: b.grow([4], [1]), lambda: b.grow([-1], [1]), lambda: b.grow([2], [-1]),
                 lambda: b.free([0, 0], [0, 0]), lambda: b.free([0], [-1]), lambda: b.free([9], [0]),
                 lambda: b.fork([0], [1]), lambda: b.fork([0], [0]), lambda: b.fork([2], [2]), lambda: b.fork([0, 0], [2, 2]),
                 lambda: b.fork([0, 2], [2, 3]), lambda: b.fork([4], [2]), lambda: b.fork([0], [4])):
        b.twin.status = 0
        b.status.zero_()
        call()
        assert b.twin.status in (NONE_FREE, BAD_LIST)


def test_empty_lists_and_full_pool(gpu):
    b = Both(2, 2, 4, 16)
    for n in range(2):
        b.grow([], [])
        b.free([], [])
        b.fork([], [])
        b.grow([1, 0], [32 if n == 0 else 0] * 2)
    b.compact(in_place=False)


def test_corrupt_page_numbers_are_passed_over(gpu):
    table, lengths, refs = i32([[0, 99, -5], [-1, -1, -1]]), i32([48, 0]), i32([1, 0])
    status, pairs, count = i32([0]), i32([[0, 0]] * 2), i32([0, 0])
    K.pages_fork(table, lengths, refs, i32([0]), i32([1]), status, 16)
    assert status.item() == 4 and refs.tolist() == [2, 0] and table[1].tolist() == [0, 99, -5]
    K.pages_compact(table, lengths, refs, table, refs, pairs, count, status, 16)
    assert table.tolist() == [[0, -1, -1], [0, -1, -1]] and count.tolist() == [0, 1]
    status.zero_()
    K.pages_free(table, lengths, refs, i32([1, 0]), i32([0, 0]), status, 16)
    assert status.item() == 4 and refs.tolist() == [0, 0] and lengths.tolist() == [0, 0]
    # a partly filled last page that is no page: growing is refused
    table, lengths = i32([[7, -1]]), i32([3])
    status.zero_()
    K.pages_grow(table, lengths, refs, i32([0]), i32([1]), pairs, count, status, 16)
    assert status.item() == 2 and lengths.tolist() == [3] and count.tolist() == [0, 0]


@pytest.mark.parametrize("layers,pages,nbytes,n", [(1, 4, 16, 2), (3, 9, 1168, 4), (24, 70, 9216, 33), (2, 33, 48, 16)])
def test_copy(gpu, layers, pages, nbytes, n):
    gen = torch.Generator(device="cuda").manual_seed(layers)
    pool = torch.randint(0, 256, (layers, pages, nbytes), generator=gen, device="cuda", dtype=torch.uint8)
    order = torch.randperm(pages, generator=gen, device="cuda")[: 2 * n].reshape(n, 2).int()
    pairs = torch.cat([order, i32([[0, 0]] * 3)])
    want = pool.clone()
    want[:, order[:, 1].long()] = want[:, order[:, 0].long()]
    status = i32([0])
    K.pages_copy(pool, pairs, i32([n, 0]), status)
    assert torch.equal(pool, want) and status.item() == 0
    K.pages_copy(pool, pairs[:0], i32([n, 0]), status)  # no room for pairs: nothing is copied
    assert torch.equal(pool, want)


def test_copy_passes_over_bad_pairs_and_counts(gpu):
    pool = torch.arange(4, dtype=torch.uint8, device="cuda")[None, :, None].repeat(2, 1, 32).contiguous()
    status = i32([0])
    K.pages_copy(pool, i32([[4, 0], [0, -1], [1, 2]]), i32([9]), status)
    assert status.item() == 4 and pool[:, :, 0].tolist() == [[0, 1, 1, 3]] * 2
    K.pages_copy(pool, i32([[3, 0]]), i32([-1]), status)
    assert pool[0, 0, 0].item() == 0
    # offsets behind 32 bits: the last layers of a pool over 4 GB
    big = torch.empty(5, 70000, 16384, dtype=torch.uint8, device="cuda")
    big[4, 69998] = 9
    big[4, 69999] = 1
    K.pages_copy(big, i32([[69998, 69999]]), i32([1]), status)
    assert int(big[4, 69999].min()) == 9


def test_a_captured_turn_replays(gpu):
    b = Both(8, 6, 40, 16)
    b.grow([0, 1], [21, 50])
    src, dst, zero, one = i32([0, 1, 0]), i32([2, 3, 4]), i32([0, 0, 0]), i32([1, 1, 1])
    ws = torch.empty(K._lib.load().enx_pages_workspace_bytes(8, 40), dtype=torch.uint8, device="cuda")

    def turn():
        K.pages_free(b.table, b.lengths, b.refs, dst, zero, b.status, 16)
        K.pages_fork(b.table, b.lengths, b.refs, src, dst, b.status, 16)
        K.pages_grow(b.table, b.lengths, b.refs, dst, one, b.pairs, b.count, b.status, 16, ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        turn()
    for _ in range(3):
        g.replay()
    b.twin.fork([0, 1, 0], [2, 3, 4])
    b.twin.grow([2, 3, 4], [1, 1, 1])
    b.same()


def test_refused_arguments(gpu):
    t, l, r, st = i32([[0]]), i32([0]), i32([0]), i32([0])
    with pytest.raises(ValueError):
        K.pages_free(t.long(), l, r, l, l, st, 16)
    with pytest.raises(ValueError):
        K.pages_free(t, i32([0, 0]), r, l, l, st, 16)
    with pytest.raises(ValueError):
        K.pages_free(t, l, r, l, i32([0, 0]), st, 16)
    with pytest.raises(ValueError):
        K.pages_free(t.cpu(), l, r, l, l, st, 16)
    with pytest.raises(EnxError):
        K.pages_free(t, l, r, l, l, st, 0)
    with pytest.raises(EnxError):
        K.pages_free(t, l, r, i32([0, 1]), i32([0, 0]), st, 16)
    with pytest.raises(ValueError):
        K.pages_grow(t, l, r, l, l, i32([[0, 0]])[:0], i32([0, 0]), st, 16)
    with pytest.raises(ValueError):
        K.pages_grow(t, l, r, l, l, i32([[0, 0]]), i32([0, 0]), st, 16, torch.empty(4, dtype=torch.uint8, device="cuda"))
    with pytest.raises(EnxError):
        K.pages_copy(torch.zeros(1, 2, 24, dtype=torch.uint8, device="cuda"), i32([[0, 1]]), i32([1]), st)


def test_more_pages_wanted_than_32_bits_hold(gpu):
    """The largest table: 262144 rows of 16384 pages that all want to be filled, 2^32 pages, which a 32-bit
    sum takes for none.  The call is refused and changes nothing."""
    rows, width, pages = 1 << 18, 1 << 14, 64
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")  # 17 GB
    lengths, refs, status = i32([0] * rows), i32([0] * pages), i32([0])
    every, add = torch.arange(rows, dtype=torch.int32, device="cuda"), torch.full((rows,), width, dtype=torch.int32, device="cuda")
    pairs, count = torch.full((rows, 2), -7, dtype=torch.int32, device="cuda"), i32([-7, -7])
    K.pages_grow(table, lengths, refs, every, add, pairs, count, status, 1)
    assert status.item() == NONE_FREE and count.tolist() == [0, 0]
    assert not lengths.any() and not refs.any() and bool((pairs == -7).all())
    assert all(bool((table[i:i + 4096] == -1).all()) for i in range(0, rows, 4096))
    # a few rows in its last corner, as far behind 2^32 bytes as a table goes
    some = [rows - 1, 0, rows - 2]
    K.pages_grow(table, lengths, refs, i32(some), i32([40, 3, 21]), pairs, count, status, 1)
    assert status.item() == NONE_FREE and count.tolist() == [0, 64]
    assert table[-1, :41].tolist() == [*range(40), -1] and table[0, :4].tolist() == [40, 41, 42, -1]
    assert table[-2, :22].tolist() == [*range(43, 64), -1] and refs.tolist() == [1] * 64
