"""Attention of drafted tokens over a paged cache: what cu_new may hold, the same on all three routes."""
import numpy as np
import pytest

from tests.test_tree_attention_gpu import Case

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
