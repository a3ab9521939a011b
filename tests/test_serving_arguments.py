"""CPU: what the serving operators refuse, before any device is touched. Descriptors claim device
memory at made-up addresses; nothing reads them."""
import ctypes

import pytest


@pytest.fixture
def lib(mcb):
    return mcb.load()


class Args:
    """Descriptors by name, laid out one after the other so that none overlap."""

    def __init__(self, **shapes):
        self.at = 1 << 20
        self.t = {}
        for name, (dtype, shape) in shapes.items():
            self.put(name, dtype, shape)

    def put(self, name, dtype, shape, strides=None, data=None, device=True):
        from matcoredsl_b200 import _abi
        if strides is None:
            strides, n = [], 1
            for d in reversed(shape):
                strides.insert(0, n)
                n *= d
        if data is None:
            data = self.at
            self.at += 1 << 24
        self.t[name] = _abi.make_tensor(data, dtype, shape, strides, device)

    def ref(self, names):
        return [ctypes.byref(self.t[n]) if n in self.t else None for n in names.split()]


def name_of(code):
    from matcoredsl_b200 import _abi
    return _abi.STATUS[code]


def ok(code):
    """Accepted: the call got as far as a device."""
    return name_of(code) in ("CANDIDATE_UNAVAILABLE",)


@pytest.fixture(autouse=True)
def no_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where no kernel can run")


GROW = "table slots positions cu after left lens new free count"


def grow_args():
    return Args(table=("i32", (4, 8)), slots=("i32", (20,)), positions=("i32", (20,)),
                cu=("i32", (5,)), after=("i32", (4,)), left=("i32", (1,)), lens=("i32", (4,)),
                new=("i32", (4,)), free=("i32", (9,)), count=("i32", (1,)))


@pytest.mark.parametrize("change,block,want", [
    (None, 16, None), (("table", "f32", (4, 8)), 16, "UNSUPPORTED_DTYPE"),
    (("lens", "i32", (3,)), 16, "SHAPE_MISMATCH"), (("cu", "i32", (4,)), 16, "SHAPE_MISMATCH"),
    (("positions", "i32", (19,)), 16, "SHAPE_MISMATCH"), (("count", "i32", (2,)), 16, "SHAPE_MISMATCH"),
    (("slots", "i32", (5, 4)), 16, "UNSUPPORTED_RANK"), (None, 0, "INVALID_ARGUMENT"),
    (None, -1, "INVALID_ARGUMENT"), (None, 2 ** 31, "INVALID_ARGUMENT")])
def test_grow(lib, change, block, want):
    a = grow_args()
    if change:
        a.put(*change)
    code = lib.mcb_paged_grow_v1(*a.ref(GROW), block, None)
    assert ok(code) if want is None else name_of(code) == want


def test_grow_memory_and_aliases(lib):
    a = grow_args()
    a.put("lens", "i32", (4,), device=False)
    assert name_of(lib.mcb_paged_grow_v1(*a.ref(GROW), 16, None)) == "UNSUPPORTED_MEMORY_SPACE"
    for one, other in (("after", "lens"), ("left", "count"), ("slots", "positions"), ("table", "free")):
        a = grow_args()
        a.t[one].data = a.t[other].data
        assert name_of(lib.mcb_paged_grow_v1(*a.ref(GROW), 16, None)) == "ALIAS_VIOLATION"
    a = grow_args()
    del a.t["count"]
    assert name_of(lib.mcb_paged_grow_v1(*a.ref(GROW), 16, None)) == "INVALID_ARGUMENT"


def test_release(lib):
    names = "free left table lens new count"
    assert ok(lib.mcb_paged_release_v1(*grow_args().ref(names), 16, None))
    assert name_of(lib.mcb_paged_release_v1(*grow_args().ref(names), 0, None)) == "INVALID_ARGUMENT"
    a = grow_args()
    a.t["left"].data = a.t["count"].data
    assert name_of(lib.mcb_paged_release_v1(*a.ref(names), 16, None)) == "ALIAS_VIOLATION"


ROPE = "qo ko q k cs pos"
APPEND = "qo kc vc q k v cs pos slots"


def rope_args(t=6, h=4, hk=2, d=64, r=32, dtype="bf16"):
    return Args(qo=(dtype, (t, h, d)), ko=(dtype, (t, hk, d)), q=(dtype, (t, h, d)),
                k=(dtype, (t, hk, d)), v=(dtype, (t, hk, d)), cs=("f32", (50, 2 * r)),
                pos=("i32", (3, t)), slots=("i32", (t,)), kc=(dtype, (7, 16, hk, d)),
                vc=(dtype, (7, 16, hk, d)))


@pytest.mark.parametrize("change,flags,want", [
    (None, 3, None), (None, 4, "INVALID_ARGUMENT"), (("k", "bf16", (6, 2, 32)), 0, "SHAPE_MISMATCH"),
    (("qo", "f32", (6, 4, 64)), 0, "UNSUPPORTED_DTYPE"), (("cs", "f32", (50, 63)), 0, "INVALID_SHAPE"),
    (("cs", "f32", (50, 66)), 0, "INVALID_SHAPE"), (("cs", "bf16", (50, 64)), 0, "UNSUPPORTED_DTYPE"),
    (("pos", "i32", (5, 6)), 0, "INVALID_SHAPE"), (("pos", "i32", (3, 7)), 0, "SHAPE_MISMATCH"),
    (("q", "i8", (6, 4, 64)), 0, "UNSUPPORTED_DTYPE")])
def test_rope(lib, change, flags, want):
    a = rope_args()
    if change:
        a.put(*change)
    code = lib.mcb_rope_v1(*a.ref(ROPE), None, flags, None)
    assert ok(code) if want is None else name_of(code) == want


def test_rope_axes_and_aliases(lib):
    a = rope_args()
    assert ok(lib.mcb_rope_v1(*a.ref(ROPE), bytes([2] * 32), 0, None))
    assert name_of(lib.mcb_rope_v1(*a.ref(ROPE), bytes([0] * 31 + [3]), 0, None)) == "INVALID_ARGUMENT"
    a.t["qo"].data = a.t["q"].data
    assert ok(lib.mcb_rope_v1(*a.ref(ROPE), None, 0, None))  # in place
    a.t["qo"].data = a.t["q"].data + 2
    assert name_of(lib.mcb_rope_v1(*a.ref(ROPE), None, 0, None)) == "ALIAS_VIOLATION"
    # in place inside one packed row [q | k | v]: rows interleave without touching
    a = rope_args()
    base, row = 1 << 30, (4 + 2 + 2) * 64
    for name, at, heads in (("q", 0, 4), ("qo", 0, 4), ("k", 256, 2), ("ko", 256, 2)):
        a.put(name, "bf16", (6, heads, 64), [row, 64, 1], base + 2 * at)
    assert ok(lib.mcb_rope_v1(*a.ref(ROPE), None, 0, None))
    a.put("qo", "bf16", (6, 4, 64), [row, 64, 1], base + 2 * 64)  # reaches into k
    assert name_of(lib.mcb_rope_v1(*a.ref(ROPE), None, 0, None)) == "ALIAS_VIOLATION"


@pytest.mark.parametrize("change,want", [
    (None, None), (("slots", "i32", (5,)), "SHAPE_MISMATCH"), (("v", "f16", (6, 2, 64)), "UNSUPPORTED_DTYPE"),
    (("vc", "bf16", (7, 8, 2, 64)), "SHAPE_MISMATCH"), (("kc", "bf16", (7, 16, 4, 64)), "SHAPE_MISMATCH"),
    (("kc", "bf16", (7, 16, 128)), "UNSUPPORTED_RANK")])
def test_append(lib, change, want):
    a = rope_args()
    if change:
        a.put(*change)
    code = lib.mcb_rope_append_v1(*a.ref(APPEND), None, 0, None)
    assert ok(code) if want is None else name_of(code) == want


def test_append_aliases_and_sizes(lib):
    a = rope_args()
    a.t["vc"].data = a.t["kc"].data
    assert name_of(lib.mcb_rope_append_v1(*a.ref(APPEND), None, 0, None)) == "ALIAS_VIOLATION"
    a = rope_args()
    for n in ("kc", "vc"):  # slot numbers are 32-bit
        a.put(n, "bf16", (2 ** 20, 2 ** 12, 2, 64), data=(1 << 45) * (1 + (n == "vc")))
    assert name_of(lib.mcb_rope_append_v1(*a.ref(APPEND), None, 0, None)) == "INVALID_SHAPE"


TREE = "o lse q kc vc table cu kv mask"


def tree_args(dtype="bf16"):
    return Args(o=(dtype, (10, 8, 64)), lse=("f32", (10, 8)), q=(dtype, (10, 8, 64)),
                kc=(dtype, (30, 16, 2, 64)), vc=(dtype, (30, 16, 2, 64)), table=("i32", (3, 9)),
                cu=("i32", (4,)), kv=("i32", (3,)), mask=("i32", (10, 2)))


@pytest.mark.parametrize("change,scale,want", [
    (None, 0.1, None), (None, float("nan"), "INVALID_ARGUMENT"), (None, 1e300, "INVALID_ARGUMENT"),
    (("o", "bf16", (10, 8, 32)), 1, "SHAPE_MISMATCH"), (("o", "f32", (10, 8, 64)), 1, "UNSUPPORTED_DTYPE"),
    (("cu", "i32", (3,)), 1, "SHAPE_MISMATCH"), (("kv", "i32", (4,)), 1, "SHAPE_MISMATCH"),
    (("mask", "i32", (9, 2)), 1, "SHAPE_MISMATCH"), (("mask", "i8", (10, 2)), 1, "UNSUPPORTED_DTYPE"),
    (("lse", "f32", (10, 9)), 1, "SHAPE_MISMATCH"), (("lse", "bf16", (10, 8)), 1, "UNSUPPORTED_DTYPE"),
    (("vc", "bf16", (31, 16, 2, 64)), 1, "SHAPE_MISMATCH"), (("kc", "f16", (30, 16, 2, 64)), 1, "UNSUPPORTED_DTYPE"),
    (("table", "f32", (3, 9)), 1, "UNSUPPORTED_DTYPE")])
def test_tree_attention(lib, change, scale, want):
    a = tree_args()
    if change:
        a.put(*change)
    code = lib.mcb_tree_attention_v1(*a.ref(TREE), scale, None)
    assert ok(code) if want is None else name_of(code) == want


def test_tree_attention_heads_and_aliases(lib):
    a = tree_args()
    for n in ("kc", "vc"):
        a.put(n, "bf16", (30, 16, 3, 64))
    assert name_of(lib.mcb_tree_attention_v1(*a.ref(TREE), 1.0, None)) == "INVALID_SHAPE"
    a = tree_args()
    a.t["o"].data = a.t["q"].data
    assert name_of(lib.mcb_tree_attention_v1(*a.ref(TREE), 1.0, None)) == "ALIAS_VIOLATION"
    a = tree_args()
    del a.t["lse"], a.t["mask"]
    assert ok(lib.mcb_tree_attention_v1(*a.ref(TREE), 1.0, None))
    a.put("q", "bf16", (0, 8, 64))
    a.put("o", "bf16", (0, 8, 64))
    assert lib.mcb_tree_attention_v1(*a.ref(TREE), 1.0, None) == 0  # nothing to do


LOGITS = "out x ids cu prompt rep pre fre bi bv bc allowed"


def logits_args():
    return Args(out=("f32", (3, 100)), x=("bf16", (3, 100)), ids=("i32", (40,)), cu=("i32", (4,)),
                prompt=("i32", (3,)), rep=("f32", (3,)), pre=("f32", (3,)), fre=("f32", (3,)),
                bi=("i32", (7,)), bv=("f32", (7,)), bc=("i32", (4,)), allowed=("i32", (3, 4)))


@pytest.mark.parametrize("change,want", [
    (None, None), (("out", "f16", (3, 100)), "UNSUPPORTED_DTYPE"), (("out", "f32", (3, 99)), "SHAPE_MISMATCH"),
    (("x", "i32", (3, 100)), "UNSUPPORTED_DTYPE"), (("rep", "f32", (4,)), "SHAPE_MISMATCH"),
    (("pre", "bf16", (3,)), "UNSUPPORTED_DTYPE"), (("bv", "f32", (6,)), "SHAPE_MISMATCH"),
    (("bc", "i32", (3,)), "SHAPE_MISMATCH"), (("allowed", "i32", (3, 3)), "SHAPE_MISMATCH"),
    (("cu", "i32", (3,)), "SHAPE_MISMATCH"), (("ids", "i32", (4, 10)), "UNSUPPORTED_RANK")])
def test_logits(lib, change, want):
    a = logits_args()
    if change:
        a.put(*change)
    code = lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None)
    assert ok(code) if want is None else name_of(code) == want


def test_logits_optional_and_aliases(lib):
    a = logits_args()
    for n in "rep pre fre bi bv bc allowed".split():
        del a.t[n]
    assert ok(lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None))
    a = logits_args()
    del a.t["bc"]
    assert name_of(lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None)) == "INVALID_ARGUMENT"
    a = logits_args()
    a.put("x", "f32", (3, 100))
    a.t["out"].data = a.t["x"].data
    assert ok(lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None))  # in place
    a.t["out"].data = a.t["x"].data + 4
    assert name_of(lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None)) == "ALIAS_VIOLATION"
    a = logits_args()
    a.put("x", "bf16", (3, 100), device=False)
    assert name_of(lib.mcb_adjust_logits_v1(*a.ref(LOGITS), None)) == "UNSUPPORTED_MEMORY_SPACE"


def test_python_arguments(mcb):
    import numpy as np
    with pytest.raises(ValueError):
        mcb.paged_grow(np.zeros((1, 1), np.int32), *[np.zeros(1, np.int32)] * 4, 16)
    x = np.zeros((1, 1, 8), np.float32)
    with pytest.raises(ValueError):
        mcb.rope(x, x, np.zeros((4, 8), np.float32), np.zeros(1, np.int32), axis_map=[0], out=(x, x))
    with pytest.raises(ValueError):
        mcb.adjust_logits(np.zeros((1, 4), np.float32), *[np.zeros(1, np.int32)] * 3, out_dtype="i8")
