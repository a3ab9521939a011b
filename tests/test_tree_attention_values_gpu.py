"""Attention of drafted tokens over a paged cache on values that say where they come from.

A key's score is 0 or so low that its weight is exactly 0, at random; values are small whole numbers.
The weights are then 1 or 0 and the sums whole, whatever the order and wherever the parts of a
context are joined, so the output is known but for the rounding of one quotient: any key or value
row that is lost, doubled or taken from another place shows, at any length."""
import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

LOW = -1024.0  # a score: exp(LOW) is 0 in f32


class Coded:
    def __init__(self, new, kv, heads, kv_heads, dim, block, dtype, tree, seed=0):
        import torch
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
        dt = ref.torch_dtype(dtype)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.dtype, cu = dtype, np.concatenate([[0], np.cumsum(new)]).tolist()
        blocks = [ref.ceil_div(n, block) for n in kv]
        total, columns = sum(blocks) + 1, max(blocks)
        order = torch.randperm(total, generator=g, device="cuda")
        table = torch.full((len(kv), columns), -1, dtype=torch.int32, device="cuda")
        # what no request holds is not a number
        k = torch.full((total * block, kv_heads, dim), float("nan"), dtype=dt, device="cuda")
        v = k.clone()
        t = cu[-1]
        self.q = (rand(t, heads, dim) - 0.5).to(dt)
        self.q[:, :, 0] = 32.0
        self.want = torch.zeros(t, heads, dim, dtype=torch.float64, device="cuda")
        self.want_lse = torch.zeros(t, heads, dtype=torch.float64, device="cuda")
        words = ref.ceil_div(max(new), 32)
        seen = torch.zeros(t, words * 32, dtype=torch.bool, device="cuda")
        at = 0
        for b, (n, length) in enumerate(zip(new, kv)):
            ids = order[at:at + blocks[b]]
            at += blocks[b]
            table[b, :blocks[b]] = ids.int()
            prefix = length - n
            counts = rand(length, kv_heads) < 0.5
            counts[0] = counts[prefix] = True  # every row sees one of them
            values = torch.floor(rand(length, kv_heads, dim) * 17) - 8
            pos = torch.arange(length, device="cuda")
            rows = ids[pos // block] * block + pos % block
            keys = torch.zeros(length, kv_heads, dim, device="cuda")
            keys[:, :, 0] = torch.where(counts, 0.0, LOW / 32)
            k[rows], v[rows] = keys.to(dt), values.to(dt)
            see = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            if tree:
                parents = (torch.arange(n, device="cuda")
                           - (rand(n) ** 3 * 6).long() - 1).clamp(min=0).tolist()
                see = torch.eye(n, dtype=torch.bool, device="cuda")
                for i in range(1, n):
                    see[i] |= see[parents[i]]
                seen[cu[b]:cu[b + 1], :n] = see
            w = counts.double()
            wv = w[:, :, None] * values.double()
            s, c = wv[:prefix].sum(0), w[:prefix].sum(0)
            s = s + torch.einsum("ij,jhd->ihd", see.double(), wv[prefix:])
            c = c + torch.einsum("ij,jh->ih", see.double(), w[prefix:])
            group = heads // kv_heads
            self.want[cu[b]:cu[b + 1]] = (s / c[..., None]).repeat_interleave(group, 1)
            self.want_lse[cu[b]:cu[b + 1]] = torch.log(c).repeat_interleave(group, 1)
        shape = (total, block, kv_heads, dim)
        self.mask = None
        if tree:
            bit = 1 << torch.arange(32, device="cuda", dtype=torch.int64)
            self.mask = (seen.view(t, words, 32) * bit).sum(2).to(torch.int32)
        self.args = (self.q, k.view(shape), v.view(shape), table, i32(cu), i32(kv), self.mask)

    def check(self, mcb, route=None):
        import torch
        lse = torch.empty(self.want_lse.shape, device="cuda")
        got = mcb.tree_attention(*self.args, scale=1.0, lse=lse)
        if route:
            assert mcb.api.last_result.route == route
        # the sum's reciprocal, the product, and the rounding to the type
        tol = (ref.HALF_ULP[self.dtype] + 2.0 ** -22) * self.want.abs() + ref.TINY[self.dtype]
        off = (got.double() - self.want).abs()
        assert bool((off <= tol).all()), (int((off > tol).sum()), float(off.max()))
        # a logarithm in f32 (2 units in the last place) and two products
        off = (lse.double() - self.want_lse).abs()
        assert bool((off <= 2.0 ** -21 * self.want_lse.abs().clamp(min=1)).all()), float(off.max())
        return got, lse


FEW, TC = "tree_attention_few_rows", "tcgen05_tree_attention"

SHAPES = [  # new, kv, heads, kv_heads, dim, block, route
    ([1] * 8, [1, 128, 129, 700, 5000, 9000, 2, 3], 8, 2, 128, 16, FEW),
    ([1] * 3, [9000, 70, 4000], 8, 1, 64, 24, FEW),
    ([3] * 5, [3, 2000, 333, 9, 128], 8, 2, 128, 64, FEW),
    # units of 1, 2, 5, 6 and 9 key tiles, one after the other in a CTA
    ([40] * 60, [(128, 256, 640, 700, 1100)[i % 5] for i in range(60)], 32, 8, 128, 16, TC),
    ([17] * 90, [(100, 500, 130, 600)[i % 4] for i in range(90)], 16, 4, 64, 8, TC),
    ([20] * 64, [40 + i for i in range(64)], 16, 8, 128, 48, TC),
    ([33, 20, 64], [20000, 30, 9000], 4, 2, 128, 32, TC),
    # many row tiles of a request
    ([700, 1, 130], [5000, 900, 130], 8, 2, 128, 16, TC),
    ([1500], [1500], 16, 4, 64, 64, TC)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tree", [True, False])
def test_every_key_and_value_is_the_right_one(mcb, shape, dtype, tree):
    Coded(*shape[:-1], dtype, tree).check(mcb, shape[-1])


@pytest.mark.parametrize("shape", [
    ([2, 1, 5], [300, 2000, 5], 6, 2, 96, 16), ([9, 1], [70, 900], 3, 3, 256, 24)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_key_and_value_is_the_right_one_on_cuda_cores(mcb, shape, dtype):
    Coded(*shape, dtype, True).check(mcb, "simt_tree_attention")


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("rows", [64, 128, 256])
def test_short_units_follow_each_other(mcb, tree, rows):
    """Units of one key tile and of five: the last values of one and the first keys of the next are
    on their way together, and what describes them shares a ring of four places. Every call of
    many gives the same bits."""
    import torch
    new = rows // 4
    c = Coded([new] * 300, [new + (0, 30, 500, 560)[i % 4] for i in range(300)], 16, 4, 128, 16,
              "bf16", tree)
    got, lse = c.check(mcb, TC)
    again, again_lse = torch.empty_like(got), torch.empty_like(lse)
    for _ in range(100):
        mcb.tree_attention(*c.args, scale=1.0, out=again, lse=again_lse)
        assert torch.equal(again, got) and torch.equal(again_lse, lse)


@pytest.mark.parametrize("dim,new,block", [(128, 1, 256), (128, 4, 16), (64, 1, 128)])
def test_few_rows_call_after_call(mcb, dim, new, block):
    """Keys and values from L2 come so fast that a stage is written again as soon as it is given back:
    whoever still reads it then gets rows of the next keys. One call in some thousands did."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(dim + new)
    n, pool = 300, 640 // (block // 16 if block > 16 else 1)
    kv = (new + torch.rand(n, generator=g, device="cuda") * 4000).int()
    table = torch.randint(0, pool, (n, 4096 // block + 1), generator=g, device="cuda").int()
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.float16)  # noqa: E731
    k, v = (rand(pool, block, 8, dim) for _ in range(2))
    args = (rand(n * new, 8 * (8 if new == 1 else 2), dim), k, v, table,
            torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda"), kv)
    want = mcb.tree_attention(*args)
    assert mcb.api.last_result.route == FEW
    out, wrong = torch.empty_like(want), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(6000):
        mcb.tree_attention(*args, out=out)
        wrong += (out != want).any()
    assert int(wrong) == 0
