"""GPU tests of a step's batch metadata (ops.paged_batch_plan, ops.shared_prefix_groups) against
plain Python; whole numbers, compared exactly."""

import numpy as np
import pytest
import torch

from turboquant_kv import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def plan(new, old, tables, free, bs, n, start=0):
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    at, lens, slots, pos, req = [0], [], [-1] * n, [0] * n, [-1] * n
    used, i = 0, 0
    for r, (k, p) in enumerate(zip(new, old)):
        k, p = max(0, k), max(0, p)
        k = min(k, n - i)
        held = -(-p // bs)
        lens.append(p + k)
        fresh = {}
        for t in range(p, p + k):
            j = t // bs
            if j >= held and j not in fresh:
                f = start + used
                fresh[j] = free[f] if 0 <= f < len(free) else -1
                used += 1
                if j < width:
                    tables[r][j] = fresh[j]
            b = tables[r][j] if j < width else -1
            slots[i], pos[i], req[i] = (b * bs + t % bs if b >= 0 else -1), t, r
            i += 1
        at.append(i)
    return at, lens, slots, pos, req, [used], tables


def check(new, old, tables, free, bs, n, start=None):
    t = _ints(tables).view(len(new), -1)
    got = ops.paged_batch_plan(_ints(new), _ints(old), t, _ints(free), bs, n, None if start is None else _ints([start]))
    ref = plan(new, old, tables, free, bs, n, start or 0)
    for g, w, dt in zip(got, ref, [torch.int32, torch.int32, torch.int64, torch.int64, torch.int32, torch.int32]):
        assert g.dtype == dt and g.tolist() == w
    assert t.tolist() == ref[6]
    return got


@pytest.mark.parametrize("bs", [1, 16, 48, 64])
@pytest.mark.parametrize("R,most,pad", [(1, 1, 0), (3, 40, 5), (300, 9, 0), (1025, 3, 100), (2, 3000, 1)])
def test_plan(bs, R, most, pad):
    rs = np.random.RandomState(R + bs)
    new = rs.randint(0, most + 1, R).tolist()
    old = rs.randint(0, 200, R).tolist()
    width = max(-(-(a + b) // bs) for a, b in zip(new, old)) + 2
    tables = rs.randint(0, 10 ** 6, (R, width)).tolist()
    need = sum(-(-(a + b) // bs) - -(-b // bs) for a, b in zip(new, old))
    check(new, old, tables, rs.permutation(need + 7).tolist(), bs, sum(new) + pad)
    check(new, old, tables, rs.permutation(need + 7).tolist(), bs, sum(new) + pad, start=4)


def test_plan_edges():
    """Too few token rows, blocks or table entries; negative lengths and entries; no requests."""
    rs = np.random.RandomState(1)
    tables = rs.randint(0, 99, (4, 5)).tolist()
    check([10, 20, 30, 5], [3, 16, 0, 70], tables, list(range(100, 120)), 16, 33)       # the rows end inside request 2
    check([10, 20, 30, 5], [3, 16, 0, 70], tables, list(range(100, 102)), 16, 65)       # two blocks are left
    check([10, 20, 30, 5], [3, 16, 0, 70], tables, [], 16, 65)
    check([10, 20, 90, 5], [3, 16, 0, 78], tables, list(range(100, 120)), 16, 125)      # past the table's width
    check([-3, 2, 0, 1], [5, -7, 3, 0], tables, list(range(9)), 16, 6)
    check([2, 1], [20, 0], [[-1, -1], [4, 4]], [7, 8], 16, 3)                           # a held entry that is none
    check([1, 1], [0, 0], [[1], [2]], [5, 6], 16, 2, start=-1)
    check([1, 1], [0, 0], [[1], [2]], [5, 6], 16, 2, start=1)
    check([0, 0], [4, 0], [[1], [2]], [5], 16, 0)
    got = ops.paged_batch_plan(_ints([]), _ints([]), torch.empty(0, 3, dtype=torch.int32, device=DEV), _ints([1]), 16, 2)
    assert [g.tolist() for g in got] == [[0], [], [-1, -1], [0, 0], [-1, -1], [0]]


def test_plan_most_requests_and_long_positions():
    R = 8192
    new, old = [1] * R, [16 * (r % 3) for r in range(R)]
    check(new, old, [[5, 6, 7]] * R, list(range(R)), 16, R)
    old = [2 ** 31 - 40]
    t = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    got = ops.paged_batch_plan(_ints([30]), _ints(old), t, _ints([1, 2, 3]), 16, 30)
    assert got[1].tolist() == [2 ** 31 - 10] and got[3][-1].item() == 2 ** 31 - 11 and set(got[2].tolist()) == {-1}


def test_plan_table_slice_and_large_pool():
    """Tables that are a slice of a wider tensor; slots past 2^31."""
    wide = torch.full((2, 9), -5, dtype=torch.int32, device=DEV)
    t = wide[:, 2:6]
    got = ops.paged_batch_plan(_ints([3, 17]), _ints([0, 0]), t, _ints([2 ** 30, 3, 4]), 16, 20)
    assert got[2][:3].tolist() == [2 ** 34, 2 ** 34 + 1, 2 ** 34 + 2]
    assert t.tolist() == [[2 ** 30, -5, -5, -5], [3, 4, -5, -5]]
    assert bool((wide[:, :2] == -5).all()) and bool((wide[:, 6:] == -5).all())


def groups(tables, lens, bs, least):
    n, starts, shared = len(lens), [0] if lens else [], [0] if lens else []
    for r in range(1, n):
        k, full = 0, max(0, min(lens[r - 1], lens[r])) // bs
        while k < min(full, len(tables[r])) and tables[r - 1][k] == tables[r][k] >= 0:
            k += 1
        if k * bs >= least:
            shared[-1] = min(shared[-1], k * bs) if starts[-1] < r - 1 else k * bs
        else:
            starts.append(r)
            shared.append(0)
    return starts + [n] * (n + 1 - len(starts)), shared + [0] * (n - len(shared))


@pytest.mark.parametrize("R,width", [(1, 3), (2, 1), (9, 70), (70, 300), (1500, 5), (8192, 2), (5, 1000)])
@pytest.mark.parametrize("least", [1, 64, 500])
def test_groups(R, width, least):
    rs = np.random.RandomState(R)
    bs = 16
    tables, row = [], None
    for r in range(R):
        if row is None or rs.rand() < 0.2:
            row = rs.randint(0, 5, width)
        else:
            row = row.copy()
            row[rs.randint(0, width):] = rs.randint(0, 5, 1)
        tables.append(row.tolist())
    lens = rs.randint(0, width * bs + 40, R).tolist()
    got = ops.shared_prefix_groups(_ints(tables), _ints(lens), bs, least)
    ref = groups(tables, lens, bs, least)
    assert got[0].tolist() == ref[0] and got[1].tolist() == ref[1]
    assert got[0].dtype == got[1].dtype == torch.int32


def test_groups_edges():
    got = ops.shared_prefix_groups(torch.empty(0, 4, dtype=torch.int32, device=DEV), _ints([]), 16, 1)
    assert got[0].tolist() == [0] and got[1].tolist() == []
    got = ops.shared_prefix_groups(_ints([[-1, 2], [-1, 2], [3, 2]]), _ints([32, 32, 32]), 16, 1)
    assert got[0].tolist() == [0, 1, 2, 3] and got[1].tolist() == [0, 0, 0]
    got = ops.shared_prefix_groups(torch.empty(2, 0, dtype=torch.int32, device=DEV), _ints([9, 9]), 16, 1)
    assert got[0].tolist() == [0, 1, 2]
    # a group shares what its least alike neighbours do
    got = ops.shared_prefix_groups(_ints([[1, 2, 3], [1, 2, 3], [1, 2, 9], [4, 2, 9]]), _ints([48] * 4), 16, 16)
    assert got[0].tolist() == [0, 3, 4, 4, 4] and got[1].tolist() == [32, 0, 0, 0]


def test_captured_and_replayed():
    new, old = _ints([1, 5, 1]), _ints([15, 30, 64])
    t = torch.zeros(3, 8, dtype=torch.int32, device=DEV)
    free = torch.arange(50, 90, dtype=torch.int32, device=DEV)
    start = _ints([0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_batch_plan(new, old, t.clone(), free, 16, 9, start)
        ops.shared_prefix_groups(t, old, 16, 16)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.paged_batch_plan(new, old, t, free, 16, 9, start)
        grp = ops.shared_prefix_groups(t, old, 16, 16)
    tables = t.tolist()
    for step in range(4):
        graph.replay()
        ref = plan(new.tolist(), old.tolist(), tables, free.tolist(), 16, 9, start.item())
        assert [g.tolist() for g in got] == list(ref[:6]) and t.tolist() == ref[6]
        assert [g.tolist() for g in grp] == list(groups(ref[6], old.tolist(), 16, 16))
        tables = ref[6]
        old.copy_(got[1])
        start.add_(got[5])
        new.copy_(_ints([step, 1, 2]))
        torch.cuda.synchronize()


def test_refusals():
    t = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    a = [_ints([1, 1]), _ints([0, 0]), t, _ints([1, 2]), 16, 2]
    ops.paged_batch_plan(*a)
    for i, bad in ((0, _ints([1])), (0, torch.ones(2, device=DEV)), (1, _ints([1, 2, 3])), (2, t.long()),
                   (2, t.t()), (2, t[:1]), (2, t[:1].expand(2, 3)), (2, t.cpu()), (3, t), (4, 0), (5, -1)):
        b = list(a)
        b[i] = bad
        with pytest.raises(RuntimeError):
            ops.paged_batch_plan(*b)
    with pytest.raises(RuntimeError):
        ops.paged_batch_plan(*a, _ints([1, 2]))
    many = torch.zeros(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        ops.paged_batch_plan(many, many, torch.zeros(8193, 1, dtype=torch.int32, device=DEV), many, 16, 1)
    for args in ((t[0], a[1], 16, 1), (t, a[1][:1], 16, 1), (t, a[1], 0, 1), (t, a[1], 16, 0), (t.cpu(), a[1], 16, 1),
                 (t.float(), a[1], 16, 1)):
        with pytest.raises(RuntimeError):
            ops.shared_prefix_groups(*args)
