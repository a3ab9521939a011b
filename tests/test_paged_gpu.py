"""Block tables and slot maps built on the GPU, against a walk over the requests."""
import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def check_grow(mcb, table, lens, new, free, count, block, tokens, columns=None):
    import torch
    want = ref.grow(table, lens, new, free, count, block, tokens)
    t = dev(table)
    if columns:  # rows of a wider table
        wide = torch.full((table.shape[0], columns), -7, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = t
        t = wide[:, :table.shape[1]]
    out = mcb.paged_grow(t, dev(lens), dev(new), dev(free), dev([count]), block, tokens=tokens)
    for name, g, w in zip(("table", "slots", "positions", "cu", "after", "left"), (t, *out),
                          (*want[:5], [want[5]])):
        assert np.array_equal(g.cpu().numpy(), w), name


def requests(rng, b, context, new, block, columns):
    lens, add = rng.integers(0, context + 1, b), rng.integers(0, new + 1, b)
    table = np.full((b, columns), -1, np.int64)
    blocks = ref.ceil_div(lens, block)
    order = rng.permutation(int(blocks.sum()) + 1)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    return lens, add, table, at


@pytest.mark.parametrize("b,context,new,block,pool", [
    (1, 0, 1, 16, 1.0), (1, 100, 1, 1, 1.0), (3, 50, 5, 8, 1.0), (64, 300, 1, 16, 1.0),
    (33, 40, 90, 24, 0.5), (1500, 60, 3, 16, 0.7), (5000, 20, 2, 4, 0.9), (7, 1000, 900, 64, 1.0),
    (40, 10, 0, 16, 1.0)])
def test_grow(mcb, b, context, new, block, pool):
    rng = np.random.default_rng(b + context)
    columns = (context + new) // block + 2
    lens, add, table, used = requests(rng, b, context, new, block, columns)
    need = int((ref.ceil_div(lens + add, block) - ref.ceil_div(lens, block)).sum())
    count = int(need * pool)
    free = np.concatenate([used + rng.permutation(count), [-1, -1]])
    check_grow(mcb, table, lens, add, free, count, block, int(add.sum()))


def test_grow_room_and_refusals(mcb):
    """More room than tokens; less room than tokens; a row that is too long for the table; a stack
    that a later request without new blocks does not need; strided rows; negative lengths."""
    rng = np.random.default_rng(5)
    lens, add, table, used = requests(rng, 9, 60, 20, 16, 6)
    free = used + rng.permutation(40)
    check_grow(mcb, table, lens, add, free, 40, 16, int(add.sum()) + 13, columns=11)
    check_grow(mcb, table, lens, add, free, 40, 16, int(add[:5].sum()) + 1)
    check_grow(mcb, table, lens, add, free, 40, 16, 0)
    long = add.copy()
    long[3] = 2000
    check_grow(mcb, table, lens, long, free, 40, 16, int(long.sum()))
    lens, add = np.array([16, 5, 32, 3]), np.array([40, 4, 1, 2])
    table = np.array([[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, -1, -1], [4, -1, -1, -1]])
    check_grow(mcb, table, lens, add, np.array([9, 8]), 2, 16, 47)
    check_grow(mcb, table, lens, add, np.array([9, 8]), 50, 16, 47)   # a count past the stack
    check_grow(mcb, table, lens, add, np.array([9, 8]), -4, 16, 47)
    check_grow(mcb, table, np.array([-3, 5, -1, 3]), np.array([2, -5, 3, 2]), np.arange(9), 9, 16, 7)


def test_grow_nothing(mcb):
    table = np.zeros((0, 4), np.int64)
    check_grow(mcb, table, np.zeros(0), np.zeros(0), np.arange(5), 3, 16, 6)


@pytest.mark.parametrize("b,context,block", [(1, 0, 16), (1, 5000, 8), (3, 70, 24), (32, 100, 16),
                                             (33, 100, 16), (1000, 300, 32)])
def test_release(mcb, b, context, block):
    rng = np.random.default_rng(b * 7 + context)
    lens, _, table, used = requests(rng, b, context, 0, block, context // block + 2)
    keep = (lens * rng.random(b) * 1.3).astype(np.int64)
    for room in (used + 9, used // 2 + 4):
        free = np.full(room, -1, np.int64)
        free[:3] = [100000, 100001, 100002]
        want, left = ref.release(table, lens, keep, free, 3, block)
        f = dev(free)
        got = mcb.paged_release(dev(table), dev(lens), dev(keep), f, dev([3]), block)
        assert np.array_equal(f.cpu().numpy(), want)
        assert got.cpu().tolist() == [left]


def test_grow_after_release_in_a_graph(mcb):
    """Both calls captured into one CUDA graph and replayed with other lengths."""
    import torch
    rng = np.random.default_rng(0)
    lens, add, table, used = requests(rng, 20, 100, 9, 16, 8)
    keep = lens // 2
    free = np.concatenate([used + rng.permutation(30), np.full(used + 5, -1)])
    g_table, g_lens, g_keep, g_add = dev(table), dev(lens), dev(keep), dev(add)
    g_free, count, left = dev(free), dev([30]), dev([0])
    e = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    out = (e(180), e(180), e(21), e(20), e(1))

    def step():
        mcb.paged_release(g_table, g_lens, g_keep, g_free, count, 16, out=left)
        mcb.paged_grow(g_table, g_keep, g_add, g_free, left, 16, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    add2, keep2 = rng.integers(0, 9, 20), lens // 3
    for g, a in ((g_table, table), (g_free, free), (g_keep, keep2), (g_add, add2)):
        g.copy_(dev(a))
    graph.replay()
    torch.cuda.synchronize()
    want_free, want_left = ref.release(table, lens, keep2, free, 30, 16)
    want = ref.grow(table, keep2, add2, want_free, want_left, 16, 180)
    for g, w in zip((g_table, *out), (*want[:5], [want[5]])):
        assert np.array_equal(g.cpu().numpy(), w)
