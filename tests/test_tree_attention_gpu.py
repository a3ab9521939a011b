"""Attention of drafted tokens over a paged cache, against 64 bits, with tolerances from the
arithmetic (serving_ref.attention)."""
import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


class Case:
    """Requests with `new` tokens over `kv` keys each, in a cache of random blocks whose unused
    rows hold NaN."""

    def __init__(self, new, kv, heads, kv_heads, dim, block, dtype, tree=True, columns=None, seed=0,
                 spread=1.0):
        import torch
        rng = np.random.default_rng(seed + sum(kv) + heads)
        self.dtype, self.scale = dtype, dim ** -0.5
        self.cu, self.kv = np.concatenate([[0], np.cumsum(new)]), np.array(kv, np.int64)
        blocks = [ref.ceil_div(max(0, n), block) for n in kv]
        columns = columns or max(1, max(blocks, default=1))
        total = sum(blocks) + 2
        order, at = rng.permutation(total), 0
        self.table = np.full((len(kv), columns), -1, np.int64)
        shape = (total, block, kv_heads, dim)
        k, v = np.full(shape, np.nan), np.full(shape, np.nan)
        for b, n in enumerate(kv):
            ids = order[at:at + blocks[b]]
            at += blocks[b]
            self.table[b, :min(columns, len(ids))] = ids[:columns]
            pos = np.arange(max(0, n))
            k[ids[pos // block], pos % block] = rng.standard_normal((len(pos), kv_heads, dim)) * spread
            v[ids[pos // block], pos % block] = rng.standard_normal((len(pos), kv_heads, dim))
        to = lambda a: torch.from_numpy(a).to(ref.torch_dtype(dtype)).cuda()  # noqa: E731
        self.k, self.v = to(k), to(v)
        self.q = to(rng.standard_normal((int(self.cu[-1]), heads, dim)) * spread)
        self.mask = None
        if tree:
            words = ref.ceil_div(max(1, max(new, default=1)), 32)
            bits = np.zeros((int(self.cu[-1]), words * 32), bool)
            for b, n in enumerate(new):
                for i in range(n):
                    row = bits[self.cu[b] + i]
                    if i:
                        row |= bits[self.cu[b] + rng.integers(max(0, i - 4), i)]
                    row[i] = True
            self.set_bits(bits)

    def set_bits(self, bits):
        self.bits = bits
        words = bits.shape[1] // 32
        w = (bits.reshape(-1, words, 32).astype(np.int64) << np.arange(32)).sum(2)
        self.mask = np.where(w >= 2 ** 31, w - 2 ** 32, w)

    def check(self, mcb, route=None, lse=True, q=None, out=None):
        import torch
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
        q = self.q if q is None else q
        t, h, d = q.shape
        z = torch.full((t, h), 7.0, device="cuda") if lse else None
        got = mcb.tree_attention(q, self.k, self.v, i32(self.table), i32(self.cu), i32(self.kv),
                                 None if self.mask is None else i32(self.mask), scale=self.scale,
                                 out=out, lse=z)
        if route:
            assert mcb.api.last_result.route == route
        f64 = lambda x: x.double().cpu().numpy()  # noqa: E731
        o, s, o_tol, s_tol = ref.attention(f64(q), f64(self.k), f64(self.v), self.table, self.cu,
                                           self.kv, self.mask, self.scale, ref.HALF_ULP[self.dtype])
        g = f64(got)
        tol = o_tol[:, :, None] + 1.01 * ref.HALF_ULP[self.dtype] * np.abs(o) + ref.TINY[self.dtype]
        assert np.array_equal(np.isnan(g), np.isnan(o))
        bad = ~(np.abs(g - o) <= tol) & ~np.isnan(o)
        assert not bad.any(), (np.argwhere(bad)[:4].tolist(), np.nanmax(np.abs(g - o)))
        if lse:
            g = f64(z)
            assert np.array_equal(np.isneginf(g), np.isneginf(s))
            fin = np.isfinite(s)
            assert np.all(np.abs(g - s)[fin] <= s_tol[fin])


SHAPES = [  # new, kv, heads, kv_heads, dim, block
    ([1], [1], 1, 1, 128, 16),
    ([1], [2], 8, 1, 64, 16),
    ([1, 1, 1], [127, 128, 129], 8, 2, 128, 16),
    ([5], [700], 32, 8, 128, 16),
    ([3, 0, 12, 1], [40, 0, 12, 1000], 6, 2, 128, 24),
    ([64, 17, 33], [64, 300, 257], 8, 2, 128, 32),
    ([40, 40], [500, 41], 16, 1, 64, 8),
    ([2] * 70, [i * 5 + 2 for i in range(70)], 4, 4, 64, 64),
    ([130], [400], 4, 2, 128, 128),
    ([7], [3000], 16, 1, 128, 48),
    ([9, 1], [20, 2500], 40, 8, 128, 1),
    ([7, 1], [20, 1900], 40, 8, 128, 1),
    ([1] * 9, [i * 250 for i in range(9)], 32, 1, 128, 16),
    ([4, 2, 9], [900, 2, 2000], 16, 4, 64, 40),
    ([3], [1000], 8, 2, 64, 256),
    ([33], [700], 8, 2, 128, 256)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tree", [True, False])
def test_sixteen_bits(mcb, shape, dtype, tree):
    new, _, heads, kv_heads = shape[:4]
    c = Case(*shape, dtype, tree)
    rows, n = sum(new) * (heads // kv_heads), len(new)
    tile = 16 if sum(new) == n else 12
    few = rows <= tile * n or (rows <= 2 * tile * n and c.table.shape[1] * shape[5] <= 2048)
    c.check(
        mcb, "tree_attention_few_rows" if few else "tcgen05_tree_attention")


@pytest.mark.parametrize("shape", [
    ([1], [1], 1, 1, 1, 4), ([3, 2], [50, 2], 3, 3, 80, 16), ([1], [4000], 9, 1, 128, 16),
    ([6], [90], 12, 4, 256, 8), ([2], [333], 4, 2, 33, 16), ([20], [45], 2, 1, 64, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tree", [True, False])
def test_any_size(mcb, shape, dtype, tree):
    Case(*shape, dtype, tree).check(mcb)


@pytest.mark.parametrize("shape", [
    ([40, 0, 1, 70, 33, 3, 5], [40, 0, 900, 75, 300, 2, 64], 8, 4, 128, 16),
    ([9] * 70, [9 + 7 * i for i in range(70)], 1, 1, 80, 24), ([2] * 200, [50] * 200, 4, 2, 33, 8),
    ([150, 160, 1], [1500, 161, 3], 3, 1, 256, 64), ([5, 2] * 40, [33, 90] * 40, 20, 4, 64, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tree", [True, False])
def test_any_size_many_tokens(mcb, shape, dtype, tree):
    """Enough tokens for several of them to share a CTA, across the borders of requests."""
    c = Case(*shape, dtype, tree)
    if tree:
        bits = c.bits.copy()
        bits[::11] = False
        c.set_bits(bits)
    c.check(mcb)


@pytest.mark.parametrize("heads", [2, 6])
def test_many_tokens_do_not_see_each_others_values(mcb, heads):
    """Infinities in the values of some drafts, in f32: they reach the rows that see them, no other."""
    import torch
    new = [7, 3, 12, 30] * 10
    c = Case(new, [n + 20 for n in new], heads, 2, 128, 16, "f32")
    hit = {}
    for b in range(0, 40, 3):
        j = new[b] // 2
        pos = 20 + j
        c.v[int(c.table[b, pos // 16]), pos % 16, :, ::3] = float("inf")
        hit[b] = j
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
    got = mcb.tree_attention(c.q, c.k, c.v, i32(c.table), i32(c.cu), i32(c.kv), i32(c.mask))
    assert mcb.api.last_result.route == "simt_tree_attention"
    got = got.cpu().numpy()
    for b in range(40):
        for t in range(c.cu[b], c.cu[b + 1]):
            if b in hit and c.bits[t, hit[b]]:
                assert np.isposinf(got[t, :, ::3]).all()
            else:
                assert np.isfinite(got[t, :, ::3]).all()
            assert np.isfinite(np.delete(got[t], np.s_[::3], 1)).all()


def test_large_scores(mcb):
    """Scores whose largest grows along the keys, far past where a first maximum would overflow."""
    for dtype in ("bf16", "f32"):
        c = Case([4], [900], 8, 2, 128, 16, dtype, spread=2.0)
        at = np.arange(900)
        import torch
        ramp = torch.from_numpy(1 + at / 60.0).to(c.k.dtype).cuda()
        blk = torch.from_numpy(c.table[0, at // 16]).cuda()
        c.k[blk, torch.from_numpy(at % 16).cuda()] *= ramp[:, None, None]
        c.check(mcb)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.5])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scales(mcb, scale, dtype):
    c = Case([3, 20], [150, 260], 4, 2, 128, 16, dtype)
    c.scale = scale
    c.check(mcb)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [2, 24])
def test_rows_that_see_nothing(mcb, dtype, heads):
    """No prefix and an empty mask row; keys fewer than new tokens; a mask narrower than the tree."""
    c = Case([6, 4, 40], [6, 2, 60], heads, 2, 128, 16, dtype)
    bits = c.bits.copy()
    bits[2] = False
    bits[5] = False
    c.set_bits(bits)
    c.check(mcb)
    c.set_bits(bits[:, :32])  # new tokens from 32 on are seen by nobody
    c.check(mcb)
    c.mask = None
    c.check(mcb)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads", [4, 64])
def test_what_is_not_seen_has_no_influence(mcb, dtype, heads):
    """NaN and infinities in keys and values of drafts that a row does not see; those that see them
    get them."""
    import torch
    c = Case([9, 5], [200, 5], heads, 2, 128, 16, dtype)
    for b, j, what in ((0, 3, float("nan")), (0, 6, float("inf")), (1, 2, float("-inf"))):
        pos = int(c.kv[b] - (c.cu[b + 1] - c.cu[b])) + j
        blk = int(c.table[b, pos // 16])
        c.v[blk, pos % 16, :, ::3] = what
        c.k[blk, pos % 16] = torch.nan
    bits = c.bits.copy()
    for b, j in ((0, 3), (0, 6), (1, 2)):
        bits[c.cu[b]:c.cu[b + 1], j] = False  # seen by no row at all
    c.set_bits(bits)
    c.check(mcb)
    # values only: seen by some rows
    c = Case([9, 5], [200, 5], heads, 2, 128, 16, dtype)
    for b, j, what in ((0, 3, float("nan")), (0, 6, float("inf")), (1, 2, float("-inf"))):
        pos = int(c.kv[b] - (c.cu[b + 1] - c.cu[b])) + j
        c.v[int(c.table[b, pos // 16]), pos % 16, :, ::3] = what
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
    got = mcb.tree_attention(c.q, c.k, c.v, i32(c.table), i32(c.cu), i32(c.kv), i32(c.mask)).float()
    got = got.cpu().numpy()
    for t in range(14):
        b = 0 if t < 9 else 1
        hit = [c.bits[t, j] for j in ((3, 6) if b == 0 else (2,))]
        column = got[t, :, ::3]
        if b == 0 and hit[0]:
            assert np.isnan(column).all()
        elif hit[-1]:
            assert np.isinf(column).all() and (np.sign(column) == (1 if b == 0 else -1)).all()
        else:
            assert np.isfinite(column).all()
        assert np.isfinite(np.delete(got[t], np.s_[::3], 1)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tables(mcb, dtype):
    """Entries outside the cache, keys past the table's columns, tokens of no request."""
    c = Case([3, 2], [300, 90], 8, 2, 128, 16, dtype)
    c.table[0, 4], c.table[0, 11], c.table[1, 0] = -1, 10 ** 6, c.k.shape[0]
    c.check(mcb)
    c = Case([3, 2], [300, 90], 8, 2, 128, 16, dtype, columns=15)
    c.check(mcb)
    c = Case([3, 2], [30, 20], 8, 2, 128, 16, dtype)
    c.cu = np.array([0, 2, 4])  # the fifth token belongs to nobody
    c.check(mcb)
    c.kv[1] = -5
    c.check(mcb)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_no_request_and_no_block(mcb, dtype):
    """Tokens of no request at all; a cache without blocks: zeros, and -inf."""
    c = Case([3], [30], 8, 2, 128, 16, dtype)
    c.cu, c.kv, c.table = np.array([0]), np.array([], np.int64), c.table[:0]
    c.check(mcb)
    c = Case([3], [30], 8, 2, 128, 16, dtype)
    c.k, c.v = c.k[:0], c.v[:0]
    c.check(mcb)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_strides(mcb, dtype):
    """Queries and outputs inside packed rows; a cache with the heads before the rows; a cache row
    that starts off a 16-byte boundary."""
    import torch
    c = Case([5, 1], [60, 200], 8, 2, 128, 16, dtype)
    packed = torch.randn(6, 12 * 128, device="cuda").to(c.q.dtype)
    q = packed[:, :8 * 128].unflatten(1, (8, 128))
    q.copy_(c.q)
    out = torch.zeros(6, 9, 128, device="cuda", dtype=c.q.dtype)
    c.k, c.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.k, c.v))
    c.check(mcb, q=q, out=out[:, 1:], lse=False)
    assert (out[:, 0] == 0).all()
    c.k, c.v = (torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in (c.k, c.v))
    c.check(mcb)


def test_other_stream_and_graph(mcb):
    import torch
    c = Case([4, 1, 9], [500, 77, 2000], 16, 4, 128, 16, "bf16")
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
    args = (c.q, c.k, c.v, i32(c.table), i32(c.cu), i32(c.kv), i32(c.mask))
    want = mcb.tree_attention(*args)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mcb.tree_attention(*args, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mcb.tree_attention(*args, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)  # bit for bit, every time


def test_offsets_past_32_bits(mcb):
    """A cache of more than 2^32 elements, with the blocks in use at its end."""
    import torch
    c = Case([2], [90], 4, 1, 64, 16, "bf16")
    blocks = (2 ** 32 + 2 ** 20) // (16 * 64)
    big = [torch.empty(blocks, 16, 1, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    last = blocks - c.k.shape[0]
    for b, x in zip(big, (c.k, c.v)):
        b[last:] = x
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
    rest = (i32(c.cu), i32(c.kv), i32(c.mask))
    want = mcb.tree_attention(c.q, c.k, c.v, i32(c.table), *rest)
    got = mcb.tree_attention(c.q, *big, i32(np.where(c.table >= 0, c.table + last, -1)), *rest)
    assert torch.equal(got, want)
