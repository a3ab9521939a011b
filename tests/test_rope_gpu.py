"""Rotary positions with several axes, and the append to a paged cache, against 64 bits."""
import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


def table(rows, pairs):
    import torch
    a = np.arange(rows)[:, None] * 1000.0 ** (-np.arange(pairs) / max(1, pairs))
    return torch.from_numpy(np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)).cuda()


def close(got, want, size, dtype):
    """Two products and a sum in f32, rounded once to the type."""
    g = got.double().cpu().numpy()
    tol = ref.HALF_ULP[dtype] * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -23 * size + ref.TINY[dtype]
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(g), nan)
    assert np.all(np.abs(g - want)[~nan] <= tol[~nan])


def f64(t):
    return t.double().cpu().numpy()


CASES = [  # tokens, heads, kv_heads, dim, rotary, axes, paired, dtype
    (1, 1, 1, 2, 2, 1, False, "f32"), (1, 32, 8, 128, 128, 1, False, "bf16"),
    (5, 4, 2, 64, 64, 1, True, "f16"), (37, 7, 1, 128, 64, 3, False, "bf16"),
    (16, 3, 3, 80, 80, 2, True, "f32"), (3, 5, 5, 6, 4, 2, False, "bf16"),
    (130, 2, 1, 256, 256, 4, False, "f16"), (9, 8, 8, 72, 36, 3, True, "bf16"),
    (11, 2, 2, 96, 96, 2, False, "f32"), (4, 3, 1, 40, 0, 1, False, "bf16")]


def inputs(case, packed=True, seed=0):
    import torch
    t, h, hk, d, rotary, axes, paired, dtype = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + t)
    x = torch.randn(t, (h + 2 * hk) * d + (0 if packed else 3), generator=g, device="cuda")
    x = x.to(ref.torch_dtype(dtype))
    if not packed:
        x = x[:, 3:]  # rows that no 16-byte load could take
    q, k, v = (y.unflatten(1, (-1, d)) for y in x.split([h * d, hk * d, hk * d], 1))
    pos = torch.randint(0, 50, (axes, t), generator=g, device="cuda", dtype=torch.int32)
    axis = [i % axes for i in range(rotary // 2)]
    return q, k, v, table(50, rotary // 2), pos, axis


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("packed", [True, False])
def test_rope(mcb, case, inverse, packed):
    q, k, _, cs, pos, axis = inputs(case, packed)
    for axes_used in (axis, sorted(axis)):
        got = mcb.rope(q, k, cs, pos, axis_map=axes_used, paired=case[6], inverse=inverse)
        for g, x in zip(got, (q, k)):
            close(g, *ref.rope(f64(x), f64(cs), pos.cpu().numpy(), axes_used, case[6], inverse),
                  case[7])


@pytest.mark.parametrize("case", CASES[:8])
def test_rope_in_place(mcb, case):
    q, k, v, cs, pos, axis = inputs(case)
    before = v.clone()
    want = [ref.rope(f64(x), f64(cs), pos.cpu().numpy(), axis, case[6], False) for x in (q, k)]
    mcb.rope(q, k, cs, pos, axis_map=axis, paired=case[6], out=(q, k))
    for g, w in zip((q, k), want):
        close(g, *w, case[7])
    assert (v == before).all()


def test_positions(mcb):
    """One row of positions without an axis map; positions outside the table give NaN in the turned
    elements only."""
    import torch
    q, k, _, cs, pos, _ = inputs((6, 2, 1, 32, 16, 1, False, "f32"))
    p = pos[0].clone()
    p[1], p[4] = -1, 50
    got = mcb.rope(q, k, cs, p)
    for g, x in zip(got, (q, k)):
        close(g, *ref.rope(f64(x), f64(cs), p.cpu().numpy(), [0] * 8, False, False), "f32")
    assert torch.isnan(got[0][1, :, :16]).all() and not torch.isnan(got[0][1, :, 16:]).any()


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("block", [1, 8, 24])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append(mcb, case, block, heads_first):
    import torch
    t, h, hk, d, rotary, axes, paired, dtype = case
    q, k, v, cs, pos, axis = inputs(case, seed=3)
    blocks = 2 * t // block + 3
    shape = (blocks, hk, block, d) if heads_first else (blocks, block, hk, d)
    caches = [torch.randn(shape, device="cuda").to(q.dtype) for _ in range(2)]
    if heads_first:
        caches = [c.transpose(1, 2) for c in caches]
    rng = np.random.default_rng(t)
    slots = rng.permutation(blocks * block)[:t]
    slots[rng.random(t) < 0.2] = -1
    if t > 4:
        slots[2], slots[3] = blocks * block, 2 ** 31 - 1  # outside the cache
    want = [f64(c) for c in caches]
    sizes = [np.abs(w) for w in want]
    turned, turned_size = ref.rope(f64(k), f64(cs), pos.cpu().numpy(), axis, paired, False)
    for i, s in enumerate(slots):
        if 0 <= s < blocks * block:
            want[0][s // block, s % block], sizes[0][s // block, s % block] = turned[i], turned_size[i]
            want[1][s // block, s % block] = f64(v)[i]
    out = mcb.rope_append(q, k, v, cs, pos, torch.from_numpy(slots.astype(np.int32)).cuda(), *caches,
                          axis_map=axis, paired=paired)
    close(out, *ref.rope(f64(q), f64(cs), pos.cpu().numpy(), axis, paired, False), dtype)
    close(caches[0], want[0], sizes[0], dtype)
    assert np.array_equal(f64(caches[1]), want[1])


def test_gradient(mcb):
    """The inverse is the gradient: against the rotation's differences, and as its transpose."""
    import torch
    q, k, _, cs, pos, axis = inputs((5, 3, 2, 24, 16, 2, True, "f32"))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    dq, dk = mcb.rope(gq, gk, cs, pos, axis_map=axis, paired=True, inverse=True)
    rng = np.random.default_rng(1)
    step = 0.5  # the rotation is linear: any step does
    for x, g, d, at in ((q, gq, dq, 0), (k, gk, dk, 1)):
        for _ in range(6):
            i = tuple(int(rng.integers(0, n)) for n in x.shape)
            up, down = x.clone(), x.clone()
            up[i] += step
            down[i] -= step
            f = [(mcb.rope(*((y, k) if at == 0 else (q, y)), cs, pos, axis_map=axis,
                           paired=True)[at].double() * g.double()).sum().item() for y in (up, down)]
            size = float((x.abs().double() * g.abs().double()).sum()) + 1
            assert abs((f[0] - f[1]) / (2 * step) - d[i].item()) <= 8 * 2.0 ** -24 * size / step
