"""GPU: books of a step with less room for slots than tokens: what has no room is not held, and can be asked for again."""
import pytest
import torch

from aotriton_b200 import paged

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _books(table, lengths, new, free, page, room, taken):
    """Slots, lengths and pages taken, one token after another."""
    slots, lengths = [], list(lengths)
    for z, m in enumerate(new):
        for _ in range(m):
            if len(slots) == room:
                return slots, lengths, taken
            i, p = lengths[z] // page, lengths[z]
            lengths[z] += 1
            if i >= len(table[z]):
                slots.append(-1)
                continue
            if p % page == 0:
                table[z][i] = free[taken] if taken < len(free) else -1
                taken += 1
            slots.append(-1 if table[z][i] < 0 else table[z][i] * page + p % page)
    return slots, lengths, taken


CASES = [([0, 0], [40, 5], 16, 8), ([3, 30, 0, 17], [10, 0, 50, 40], 16, 8), ([5] * 3, [7] * 3, 1, 30), ([i % 40 for i in range(700)], [i % 7 for i in range(700)], 16, 4),
         ([0, 2], [9000, 700], 64, 200), ([14, 0], [40, 3], 16, 2), ([i % 5 for i in range(300)], [1] * 300, 4, 3)]


@pytest.mark.parametrize("lengths,new,page,width", CASES)
@pytest.mark.parametrize("python", [False, True])
def test_steps_with_too_little_room(lengths, new, page, width, python, monkeypatch):
    if python:
        monkeypatch.setattr(paged._native, "block_tables", lambda *a: None)
    total = sum(new)
    held = [[1000 + 50 * z + i for i in range(min(-(-n // page), width))] for z, n in enumerate(lengths)]
    free = list(range(50000, 50000 + total + len(new)))
    for room in sorted({0, 1, page, total // 3, total // 2, total - 1, total}):
        rows = [h + [-1] * (width - len(h)) for h in held]
        table, n, taken, left = _ints(rows), list(lengths), 0, list(new)
        for _ in range(3):      # (what had no room is asked for again, twice)
            r = paged.block_tables(table, _ints(n), _ints(left), _ints(free), page, room, _ints([taken]))
            slots, m, taken = _books(rows, n, left, free, page, room, taken)
            assert r.slots.tolist() == slots + [-1] * (room - len(slots)) and r.lengths.tolist() == m and r.taken.tolist() == [taken] and table.tolist() == rows
            assert r.cu_seqlens.tolist() == [0] + torch.tensor(left).cumsum(0).tolist()
            left = [x - (b - a) for x, a, b in zip(left, n, m)]
            n = m
