"""Attention of drafted tokens over a paged cache: what cu_new and the mask may hold, the same on all
three routes."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.test_tree_attention_gpu import Case
from tests.test_tree_attention_values_gpu import Coded

pytestmark = pytest.mark.gpu

# dtype, heads (2 key heads, 4 requests of 5 tokens), route
ROUTES = [("bf16", 4, "tree_attention_few_rows"), ("f16", 16, "tcgen05_tree_attention"),
          ("bf16", 128, "tcgen05_tree_attention"), ("f32", 4, "simt_tree_attention")]


def run(mcb, c, cu, route):
    import torch
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).int().cuda()  # noqa: E731
    t, h, _ = c.q.shape
    out, lse = torch.full_like(c.q, 7.0), torch.full((t, h), 7.0, device="cuda")
    mcb.tree_attention(c.q, c.k, c.v, i32(c.table), i32(cu), i32(c.kv),
                       None if c.mask is None else i32(c.mask), scale=c.scale, out=out, lse=lse)
    assert mcb.api.last_result.route == route
    return out, lse


@pytest.mark.parametrize("dtype,heads,route", ROUTES)
@pytest.mark.parametrize("tree", [True, False])
def test_descending(mcb, dtype, heads, route, tree):
    """Where it descends anywhere, no token belongs to a request: zeros, and -inf."""
    c = Case([5] * 4, [300, 5, 140, 20], heads, 2, 128, 16, dtype, tree)
    for cu in ([0, 20, 0, 20, 0], [0, 5, 10, 9, 20], [3, 2, 10, 15, 20], [0, 5, 10, 15, -1]):
        out, lse = run(mcb, c, np.array(cu), route)
        assert (out == 0).all() and (lse == float("-inf")).all()
    c.check(mcb, route)


@pytest.mark.parametrize("dtype,heads,route", ROUTES)
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("cut", [(1, 0), (3, 2), (6, 0), (9, 7)])
def test_requests_that_begin_before_the_first_token(mcb, dtype, heads, route, tree, cut):
    """Entries below 0, and past the last token: what lies inside is computed as it would be with all
    of them there."""
    import torch
    c = Coded([5] * 4, [300, 5, 140, 20], heads, 2, 128, 16, dtype, tree, seed=heads)
    q, k, v, table, cu, kv, mask = c.args
    here = slice(cut[0], 20 - cut[1])
    out = torch.full_like(q[here], 7.0)
    lse = torch.full(out.shape[:2], 7.0, device="cuda")
    mcb.tree_attention(q[here], k, v, table, cu - cut[0], kv, None if mask is None else mask[here],
                       scale=1.0, out=out, lse=lse)
    if heads != 16 or cut != (9, 7):  # 8 heads a key head and one token a request are few rows
        assert mcb.api.last_result.route == route
    want, want_lse = c.want[here], c.want_lse[here]
    tol = (ref.HALF_ULP[dtype] + 2.0 ** -22) * want.abs() + ref.TINY[dtype]
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -21 * want_lse.abs().clamp(min=1)).all()


@pytest.mark.parametrize("dtype,heads,route", ROUTES)
def test_a_mask_of_no_words(mcb, dtype, heads, route):
    """It has no bit set: no token sees a new one, its own included."""
    import torch
    c = Case([5] * 4, [300, 5, 140, 20], heads, 2, 128, 16, dtype)
    c.mask = np.zeros((20, 1), np.int64)
    want, want_lse = run(mcb, c, c.cu, route)
    c.mask = np.zeros((20, 0), np.int64)
    out, lse = run(mcb, c, c.cu, route)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert (out[5:10] == 0).all() and (lse[5:10] == float("-inf")).all()  # no prefix either
    assert (lse[:5] > 0).all()


@pytest.mark.parametrize("dtype,heads,route", ROUTES)
@pytest.mark.parametrize("new", [True, False])
def test_an_infinite_value_whose_weight_is_too_small(mcb, dtype, heads, route, new):
    """Seen all the same: infinity or not a number in its place, nothing elsewhere. Among the new
    tokens' values and among those before them."""
    import torch
    c = Case([5] * 4, [300, 5, 140, 20], heads, 2, 128, 16, dtype, tree=False)
    c.q[:] = 1.0
    pos = 295 if new else 200
    blk = int(c.table[0, pos // 16])
    c.k[blk, pos % 16] = -64.0  # a score 700 below the others'
    c.v[blk, pos % 16, :, ::3] = float("inf")
    out, lse = run(mcb, c, c.cu, route)
    assert not torch.isfinite(out[:5, :, ::3]).any()
    out[:5, :, ::3] = 0.0
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
