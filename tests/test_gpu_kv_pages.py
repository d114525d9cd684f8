"""The pages of a step against one sequence after the other: every whole number is compared."""

import pytest
import torch

from lighthouse_amd import ops
from tests import packed_reference as ref

pytestmark = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


class Pool:
    def __init__(self, lengths, size, P, pages, seed=0, extra=0):
        """Sequences hold what their lengths need (`extra` more), scattered; the rest is free."""
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(pages, generator=g).tolist()
        self.size, self.pages = size, pages
        self.table = []
        for n in lengths:
            held = min(-(-n // size) + extra, P)
            self.table.append([order.pop() for _ in range(held)] + [-1] * (P - held))
        self.free = order + [-7] * (pages - len(order))
        self.n_free, self.lengths = len(order), list(lengths)
        wide = torch.full((max(len(lengths), 1), P + 3), 99, dtype=torch.int32, device="cuda")
        self.d_table = wide[: len(lengths), :P]
        if lengths:
            self.d_table.copy_(dev(self.table))
        self.wide = wide
        self.d_free, self.d_n, self.d_lengths = dev(self.free), dev([self.n_free]), dev(self.lengths)

    def step(self, counts, N, in_place=True):
        want = ref.pages(self.table, self.lengths, counts, self.free, self.n_free, self.size, N)
        got = ops.kv_pages(self.d_table, self.d_lengths, dev(counts), self.d_free, self.d_n, self.size, N, out=self.d_lengths if in_place else None)
        lengths, starts, positions, slots = got
        assert (lengths is self.d_lengths) == in_place
        if not in_place:
            assert self.d_lengths.tolist() == self.lengths
            self.d_lengths = lengths
        for name, x, y in zip(("lengths", "starts", "positions", "slots", "table", "free", "n_free"),
                              (lengths, starts, positions, slots, self.d_table, self.d_free, self.d_n), (*want[:6], [want[6]])):
            assert x.tolist() == y, name
        assert (self.wide[:, -3:] == 99).all()
        self.lengths, _, _, _, self.table, self.free, self.n_free = want
        return want

    def whole(self):
        """Every page is in one place."""
        held = [p for row in self.table for p in row if p >= 0] + self.free[: self.n_free]
        assert sorted(held) == list(range(self.pages))


@pytest.mark.parametrize("size", [1, 7, 16, 64])
@pytest.mark.parametrize("lengths,counts", [
    ([0], [1]), ([15], [1]), ([16], [1]), ([0, 0, 0], [0, 0, 0]), ([5, 16, 31, 0], [11, 1, 1, 40]), ([30, 40, 50], [-1, 3, -1]), ([64] * 70, [1] * 70),
    ([3, 0, 17, 100], [20, -1, 0, 5]),
])
def test_steps(size, lengths, counts):
    p = Pool(lengths, size, 200, 8000 // size + 300, seed=size)
    N = sum(max(c, 0) for c in counts)
    p.step(counts, N)
    p.step(counts, N + 5, in_place=False)
    p.whole()


@pytest.mark.parametrize("B", [1, 63, 64, 65, 1023, 1024, 1025, 2500])
def test_many_sequences_that_come_and_go(B):
    g = torch.Generator().manual_seed(B)
    p = Pool([0] * B, 4, 12, 5 * B + 8, seed=B)
    for step in range(4):
        counts = torch.randint(-3, 14, (B,), generator=g).tolist()
        N = sum(max(c, 0) for c in counts)
        p.step(counts, N if step % 2 else N + 300, in_place=step % 2 == 0)
        p.whole()


def test_pages_that_go_back_are_taken_in_the_same_step():
    p = Pool([64, 64, 0], 16, 8, 8)
    assert p.n_free == 0
    p.step([-1, 0, 64], 64)
    assert p.lengths == [0, 64, 64] and p.n_free == 0
    p.whole()


def test_too_few_pages():
    """The second sequence misses more than there are; so does, with it, every later one that needs any."""
    p = Pool([16, 16, 16, 10, 16], 16, 8, 8)
    want = p.step([16, 64, 16, 6, 0], 110)
    assert p.lengths == [32, 16, 16, 16, 16]
    assert want[2][16:96] == [-1] * 80 and want[2][96:102] == [10, 11, 12, 13, 14, 15] and want[2][102:] == [-1] * 8
    p.whole()
    p.step([0, 16, 16, 0, 0], 32)  # (now there is enough for one of them)
    p.whole()


def test_a_length_beyond_the_table_and_rows_beyond_the_step():
    p = Pool([30, 10, 10], 16, 3, 20)
    p.step([19, 2, 5], 26)
    assert p.lengths == [30, 12, 15]
    p.step([2, 3, 30], 4)  # the second one's rows end behind the fourth
    assert p.lengths == [32, 12, 15]
    p.step([2**31 - 1, 2**31 - 1, 1], 4)
    assert p.lengths == [32, 12, 15]
    p.whole()


def test_sequences_that_hold_more_or_less_than_their_lengths_need():
    """As after an eviction, or tokens that were not kept: what is too much goes back, what is missing is taken."""
    p = Pool([40, 7, 0, 33], 8, 10, 60, extra=3)
    p.lengths = [9, 70, 0, 34]
    p.d_lengths.copy_(dev(p.lengths))
    p.step([1, 2, 0, 0], 3)
    p.whole()


def test_lengths_are_clamped_and_lists_too_long_are_cut():
    p = Pool([10, 10], 4, 5, 30)
    p.lengths = [-5, 1000]
    p.d_lengths.copy_(dev(p.lengths))
    p.n_free = 99
    p.d_n.fill_(99)
    p.free = [i % 30 for i in range(30)]
    p.d_free.copy_(dev(p.free))
    p.step([3, 0], 3)


def test_no_sequences_and_no_tokens():
    p = Pool([], 4, 5, 10)
    p.step([], 0)
    p.step([], 3)
    q = Pool([9] * 1500, 4, 5, 4600)
    q.step([0] * 1500, 0)


@pytest.mark.parametrize("B,T", [(3, 2000), (1030, 7), (8, 513)])
def test_more_tokens_than_one_workgroup_places(B, T):
    p = Pool([b % 37 for b in range(B)], 16, (T + 60) // 16 + 1, B * ((T + 60) // 16 + 1), seed=T)
    counts = [T if b % 3 == 0 else -1 if b % 5 == 1 else 1 for b in range(B)]
    p.step(counts, sum(max(c, 0) for c in counts) + 77)
    p.whole()


@pytest.mark.parametrize("B", [255, 256, 257])
@pytest.mark.parametrize("N", [1023, 1024, 1025])
def test_around_the_sizes_of_the_smaller_workgroup(B, N):
    g = torch.Generator().manual_seed(B + N)
    p = Pool(torch.randint(0, 40, (B,), generator=g).tolist(), 4, 16, 20 * B, seed=B)
    counts = [(3, 5, -1, 0, 7)[b % 5] for b in range(B)]
    counts[-1] += N - sum(max(c, 0) for c in counts[:-1]) - max(counts[-1], 0) if N > sum(max(c, 0) for c in counts) else 0
    p.step(counts, N)
    p.step([1] * B, N, in_place=False)
    p.whole()


def test_a_captured_step_goes_on_from_replay_to_replay():
    p = Pool([3, 16, 0, 30], 16, 6, 24, seed=3)
    counts, N = dev([1, 1, 1, 1]), 6
    run = lambda: ops.kv_pages(p.d_table, p.d_lengths, counts, p.d_free, p.d_n, 16, N, out=p.d_lengths)  # noqa: E731
    state = (p.d_table.clone(), p.d_lengths.clone(), p.d_free.clone(), p.d_n.clone())
    run()
    torch.cuda.synchronize()
    for x, y in zip((p.d_table, p.d_lengths, p.d_free, p.d_n), state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for c in ([1, 1, 1, 1], [2, -1, 1, 1], [0, 3, 1, -1], [1, 1, 1, 1]) * 3:
        counts.copy_(dev(c))
        want = ref.pages(p.table, p.lengths, c, p.free, p.n_free, 16, N)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((*out, p.d_table, p.d_free, p.d_n), (*want[:6], [want[6]])):
            assert x.tolist() == y
        p.lengths, _, _, _, p.table, p.free, p.n_free = want
