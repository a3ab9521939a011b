"""GPU: keys and values in one tensor, whatever its order: appending and attending give the bits that two
tensors give."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("order", ["blocks 2 rows heads", "blocks rows 2 heads", "blocks rows heads 2",
                                   "blocks 2 heads rows"])
def test_one_tensor_for_keys_and_values(mcb, order, dtype):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    size = {"blocks": 9, "2": 2, "rows": 16, "heads": 2}
    names = order.split()
    both = torch.zeros(*(size[n] for n in names), 64, dtype=dt, device="cuda")
    back = [names.index(n) for n in ("2", "blocks", "rows", "heads")] + [4]
    k1, v1 = both.permute(back)
    k0, v0 = torch.zeros(2, 9, 16, 2, 64, dtype=dt, device="cuda")
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    q, k, v = rand(90, 8, 64), rand(90, 2, 64), rand(90, 2, 64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cos_sin = torch.rand(100, 64, generator=g, device="cuda")
    slots = torch.randperm(9 * 16, generator=g, device="cuda")[:90].int()
    positions = torch.arange(90, dtype=torch.int32, device="cuda")
    outs = [mcb.rope_append(q, k, v, cos_sin, positions, slots, *c) for c in ((k0, v0), (k1, v1))]
    assert torch.equal(*outs) and torch.equal(k0, k1) and torch.equal(v0, v1) and (k0 != 0).any()
    table = torch.randperm(9, generator=g, device="cuda").int()[None]
    outs = [mcb.tree_attention(q[:5], *c, table, i32([0, 5]), i32([140])) for c in ((k0, v0), (k1, v1))]
    assert torch.equal(*outs)
