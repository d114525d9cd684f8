"""Sequences that get no tokens, or have ended, behind ones whose rows pass the step's: they are not refused."""

import pytest
import torch

from lighthouse_amd import ops

pytestmark = pytest.mark.gpu


def statement(table, lengths, counts, free, n_free, size, N):
    """One sequence after the other, as lists: refused is one whose length would pass the table, or that gets tokens which pass the N rows, or that
    misses more pages than there are; then nothing of it changes."""
    table, free, B, P = [list(row) for row in table], list(free), len(table), len(table[0])
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + max(c, 0))
    new = [0 if c < 0 else n + c for n, c in zip(lengths, counts)]
    ok = [new[b] <= P * size and (counts[b] <= 0 or starts[b + 1] <= N) for b in range(B)]
    held = [sum(p >= 0 for p in row) for row in table]
    need = [-(-n // size) for n in new]
    for b in range(B):
        for j in range(need[b], held[b]) if ok[b] else ():
            free[n_free], table[b][j] = table[b][j], -1
            n_free += 1
    there, missed = n_free, 0
    positions, slots = [-1] * N, [-1] * N
    for b in range(B):
        more = max(need[b] - held[b], 0) if ok[b] else 0
        missed += more
        ok[b] = ok[b] and (more == 0 or missed <= there)
        if not ok[b]:
            continue
        for j in range(held[b], need[b]):
            n_free -= 1
            table[b][j] = free[n_free]
        for i in range(max(counts[b], 0)):
            at = lengths[b] + i
            positions[starts[b] + i], slots[starts[b] + i] = at, table[b][at // size] * size + at % size
    return [n if k else o for n, o, k in zip(new, lengths, ok)], [min(s, N) for s in starts], positions, slots, table, free, n_free


def check(lengths, counts, size, P, N, extra=0):
    """`extra`: pages that each sequence has beyond what its length needs."""
    held = [min(-(-n // size) + extra, P) for n in lengths]
    pages = sum(held) + sum(-(-max(c, 0) // size) for c in counts) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(len(lengths))).tolist()
    table = [[order.pop() for _ in range(h)] + [-1] * (P - h) for h in held]
    free, n_free = order + [-1] * (pages - len(order)), len(order)
    want = statement(table, lengths, counts, free, n_free, size, N)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    d_table, d_free, d_n = dev(table), dev(free), dev([n_free])
    got = ops.kv_pages(d_table, dev(lengths), dev(counts), d_free, d_n, size, N)
    for name, x, y in zip(("lengths", "starts", "positions", "slots", "table", "free", "n_free"), (*got, d_table, d_free, d_n), (*want[:6], [want[6]])):
        assert x.tolist() == y, name
    return want


def test_one_that_ended_gives_its_pages_back_whatever_came_before():
    lengths, table = check([8, 8, 4], [10, -1, 0], 4, 8, 4)[0::4][:2]
    assert lengths == [8, 0, 4] and table[1] == [-1] * 8 and table[0][1] >= 0
    assert check([8, 8, 4], [-1, 10, 0], 4, 8, 4)[0] == [0, 8, 4]
    assert check([8, 8, 4, 7], [10, -1, 0, 1], 4, 8, 4)[0] == [8, 0, 4, 7]  # (the last one's token passes the rows, too)
    assert check([8, 8], [1, -1], 4, 8, 0)[0] == [8, 0]


def test_one_without_tokens_gives_back_what_it_does_not_need():
    want = check([8, 8, 5], [10, 0, -1], 4, 8, 4, extra=2)
    assert want[0] == [8, 8, 0] and sum(p >= 0 for p in want[4][1]) == 2 and sum(p >= 0 for p in want[4][0]) == 4


@pytest.mark.parametrize("B", [70, 1024, 1025, 2500])
@pytest.mark.parametrize("part", [0, 40, 1])
def test_many_of_them(B, part):
    """A step with room for none, a fortieth and all but the last of the tokens (with more than 4096 of these in a second launch)."""
    g = torch.Generator().manual_seed(B + part)
    lengths = torch.randint(0, 40, (B,), generator=g).tolist()
    counts = torch.randint(-6, 9, (B,), generator=g).tolist()
    counts[-2:] = [3, -1]
    total = sum(max(c, 0) for c in counts)
    want = check(lengths, counts, 4, 12, total // part - (part == 1) if part else 0, extra=1)
    assert all(n == 0 for n, c in zip(want[0], counts) if c < 0)
