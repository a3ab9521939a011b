"""Penalties, biases and grammar masks on logits, against 64 bits."""
import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


def make(rows, vocab, history, biases, seed=0):
    rng = np.random.default_rng(seed + rows * vocab)
    lens = rng.integers(0, history + 1, rows)
    lens[rng.integers(0, rows)] = history
    cu = np.concatenate([[0], np.cumsum(lens)])
    ids = (rng.random(cu[-1]) ** 3 * vocab).astype(np.int64)
    blens = rng.integers(0, biases + 1, rows)
    bias_cu = np.concatenate([[0], np.cumsum(blens)])
    return dict(x=rng.standard_normal((rows, vocab)) * 4, ids=ids, cu=cu,
                prompt=(lens * rng.random(rows)).astype(np.int64),
                rep=rng.uniform(0.8, 1.6, rows).astype(np.float32),
                pre=rng.uniform(-1, 1, rows).astype(np.float32),
                fre=rng.uniform(-0.2, 0.5, rows).astype(np.float32),
                bias_ids=rng.integers(0, max(1, vocab // 2), bias_cu[-1]),
                bias_values=rng.standard_normal(bias_cu[-1]).astype(np.float32), bias_cu=bias_cu,
                allowed=rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)))


def check(mcb, c, dtype, out_dtype, use=("rep", "pre", "fre", "bias", "allowed"), in_place=False,
          pad=0):
    import torch
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int64)).int().cuda()  # noqa: E731
    f32 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()  # noqa: E731
    x = torch.from_numpy(c["x"]).to(ref.torch_dtype(dtype)).cuda()
    if pad:
        wide = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device="cuda")
        wide[:, pad - 1:-1] = x
        x = wide[:, pad - 1:-1]
    v = x.double().cpu().numpy()
    on = {n: c[n] if n in use else None for n in ("rep", "pre", "fre", "allowed")}
    bias = [c[n] if "bias" in use else None for n in ("bias_ids", "bias_values", "bias_cu")]
    want, size = ref.logits(v, c["ids"], c["cu"], c["prompt"], on["rep"], on["pre"], on["fre"], *bias,
                            on["allowed"])
    kw = {} if bias[0] is None else dict(bias_ids=i32(bias[0]), bias_values=f32(bias[1]),
                                         bias_cu=i32(bias[2]))
    for name, key in (("repetition", "rep"), ("presence", "pre"), ("frequency", "fre")):
        if on[key] is not None:
            kw[name] = f32(on[key])
    if on["allowed"] is not None:
        kw["allowed"] = i32(on["allowed"])
    got = mcb.adjust_logits(x, i32(c["ids"]), i32(c["cu"]), i32(c["prompt"]),
                            out=x if in_place else None, out_dtype=None if in_place else out_dtype,
                            **kw)
    assert got.dtype == ref.torch_dtype(dtype if in_place else out_dtype)
    g = got.double().cpu().numpy()
    fin = np.isfinite(want)
    assert np.array_equal(g[~fin], want[~fin], equal_nan=True)
    # at most six roundings to f32 of numbers no larger than the terms' sum, and the output's
    kind = dtype if in_place else out_dtype
    tol = ref.HALF_ULP[kind] * np.abs(want) * (1 + 2.0 ** -10) + 6 * 2.0 ** -24 * size + ref.TINY[kind]
    assert np.all(np.abs(g - want)[fin] <= tol[fin])


@pytest.mark.parametrize("rows,vocab,history,biases", [
    (1, 1, 0, 0), (1, 1, 3, 2), (3, 31, 5, 4), (2, 33, 100, 0), (5, 8192, 50, 9), (4, 8193, 700, 33),
    (1, 50001, 3000, 400), (9, 20000, 1, 1), (2, 131072, 5000, 5)])
@pytest.mark.parametrize("dtype,out_dtype", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"),
                                             ("f16", "f32"), ("f16", "f16")])
def test_logits(mcb, rows, vocab, history, biases, dtype, out_dtype):
    check(mcb, make(rows, vocab, history, biases), dtype, out_dtype)


@pytest.mark.parametrize("rows,vocab,history,dtype,pad", [
    (40, 50001, 20000, "bf16", 0), (3, 131072, 65000, "f32", 0), (300, 16385, 5000, "f16", 1)])
def test_long_histories(mcb, rows, vocab, history, dtype, pad):
    """Histories read in many rounds by every slice, some ids outside the vocabulary, a row
    without any."""
    c = make(rows, vocab, history, 5)
    c["ids"][::97] = -1
    c["ids"][5::97] = vocab + np.arange(len(c["ids"][5::97]))
    c["ids"][9::31] = vocab - 1
    cu = c["cu"].copy()
    cu[1] = 0  # row 0 has none, row 1 takes them
    c["cu"], c["prompt"][0] = cu, 0
    check(mcb, c, dtype, "f32", pad=pad)
    check(mcb, c, dtype, "f32", ("fre",), pad=pad)


@pytest.mark.parametrize("use", [(), ("rep",), ("pre",), ("fre",), ("bias",), ("allowed",),
                                 ("rep", "bias")])
def test_parts(mcb, use):
    check(mcb, make(3, 9000, 200, 20), "f32", "f32", use)


@pytest.mark.parametrize("pad", [0, 1, 5, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_and_strides(mcb, pad, dtype):
    c = make(4, 5000, 300, 30)
    check(mcb, c, dtype, dtype, in_place=True, pad=pad)
    check(mcb, c, dtype, "f32", pad=pad)


def test_special_values(mcb):
    """Infinities and NaN pass through; a row whose grammar allows nothing is all -inf; ids outside
    the vocabulary and the last of several biases."""
    c = make(3, 100, 40, 10)
    c["x"][0, :4] = [np.inf, -np.inf, np.nan, 0.0]
    c["allowed"][0] = -1
    c["allowed"][1] = 0
    c["ids"][:6] = [-1, 100, 0, 1, 2, 2 ** 31 - 1]
    c["bias_ids"] = np.where(np.arange(len(c["bias_ids"])) % 2 == 0, 7, c["bias_ids"])
    c["bias_ids"][-1] = -5
    check(mcb, c, "f32", "f32")
