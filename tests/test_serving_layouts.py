"""CPU: cache pairs that are views of one tensor are taken wherever they share no element, and refused
wherever they do, before any device is touched (made-up addresses; nothing reads them)."""
import itertools

import numpy as np
import pytest

from tests.test_serving_arguments import APPEND, name_of, no_gpu, rope_args  # noqa: F401


@pytest.fixture
def lib(mcb):
    return mcb.load()


BASE = 1 << 40


def append(lib, shape, strides, apart, dtype="bf16"):
    """rope_append into caches of one shape, `apart` bytes from each other."""
    blocks, block, heads, dim = shape
    a = rope_args(t=6, h=2 * heads, hk=heads, d=dim, r=max(1, dim // 4), dtype=dtype)
    a.put("kc", dtype, shape, strides, BASE)
    a.put("vc", dtype, shape, strides, BASE + apart)
    return name_of(lib.mcb_rope_append_v1(*a.ref(APPEND), None, 0, None))


@pytest.mark.parametrize("strides,apart", [
    ([2 * 16 * 2 * 64, 2 * 64, 64, 1], 16 * 2 * 64),    # [blocks, 2, block, heads, dim]
    ([2 * 16 * 2 * 64, 2 * 2 * 64, 64, 1], 2 * 64),     # [blocks, block, 2, heads, dim]
    ([2 * 16 * 2 * 64, 2 * 2 * 64, 2 * 64, 1], 64),     # [blocks, block, heads, 2, dim]
    ([2 * 16 * 2 * 64, 64, 16 * 64, 1], 2 * 16 * 64),   # [blocks, 2, heads, block, dim]
    ([16 * 2 * 64, 2 * 64, 64, 1], 7 * 16 * 2 * 64)])   # [2, blocks, block, heads, dim]
def test_one_tensor_for_keys_and_values(lib, strides, apart):
    shape = (7, 16, 2, 64)
    for sign in (1, -1):
        assert append(lib, shape, strides, sign * 2 * apart) == "CANDIDATE_UNAVAILABLE"
        for off in (1, -1):  # a row that begins an element too early or too late
            touches = apart != 7 * 16 * 2 * 64 or off == -1
            want = "ALIAS_VIOLATION" if touches else "CANDIDATE_UNAVAILABLE"
            assert append(lib, shape, strides, sign * 2 * (apart + off)) == want


def test_the_answer_is_exact(lib):
    """Against the sets of elements, for small views of nested strides in any order."""
    rng = np.random.default_rng(3)
    seen = set()
    for _ in range(400):
        shape = [int(x) for x in rng.integers(1, 4, 4)]
        shape[3] = int(rng.choice([2, 4]))
        strides, span = [0, 0, 0, 1], shape[3]
        for i in rng.permutation(3):
            strides[i] = span + int(rng.integers(0, 2 * span))
            span = strides[i] * shape[i]
        off = int(rng.integers(-span, span))
        at = {sum(i * s for i, s in zip(x, strides)) for x in itertools.product(*map(range, shape))}
        touches = any(x + off in at for x in at)
        got = append(lib, tuple(shape), strides, 4 * off, "f32")
        assert got == ("ALIAS_VIOLATION" if touches else "CANDIDATE_UNAVAILABLE"), (shape, strides, off)
        seen.add((touches, abs(off) < max(at)))
    assert len(seen) >= 3  # apart and touching, interleaved and not
