"""CPU: the attention over a paged cache shares every unit's key tiles out once, whatever the lengths
say, and reads no length that is not there. The functions that the kernels run on the device are
compiled for the host (tests/native/tree_shares.cu)."""
import subprocess

import numpy as np
import pytest

from tests.native_util import compile_native

COST = {16: 1, 32: 1, 128: 3, 256: 3}


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    out = compile_native("tree_shares", tmp_path_factory.mktemp("native"))

    def run(rows, threads, grid, tokens, group, kv_heads, block, columns, masked, cu, kv):
        numbers = [rows, threads, grid, tokens, group, kv_heads, block, columns, int(masked), len(kv),
                   *cu, *kv]
        r = subprocess.run([out], input=" ".join(str(int(x)) for x in numbers), text=True,
                           capture_output=True, timeout=60)
        assert r.returncode == 0, r.returncode  # below 0: ended by a signal
        segments, parts = [], {}
        for line in r.stdout.splitlines():
            if line.startswith("part"):
                x = [int(y) for y in line.split()[1:]]
                parts[x[0]] = x[1:]
            else:
                segments.append([int(y) for y in line.split()])
        return segments, parts
    return run


def units(rows, tokens, group, kv_heads, block, columns, masked, cu, kv):
    """{(request, head, first row): (rows, first token, tiles)} by the definition."""
    out = {}
    for b, length in enumerate(kv):
        first, last = max(0, int(cu[b])), min(tokens, int(cu[b + 1]))
        n, length = int(cu[b + 1]) - int(cu[b]), max(0, int(length))
        keys = min(length, columns * block)
        total = max(0, last - first) * group
        for row0 in range(0, total, rows):
            nrows = min(rows, total - row0)
            end = keys
            if not masked:  # the last row's own key
                i = first - int(cu[b]) + (row0 + nrows - 1) // group
                end = min(keys, max(0, length - n + i + 1))
            for head in range(kv_heads):
                out[b, head, row0] = (nrows, first, max(1, -(-end // 128)))
    return out


def check(shares, rows, grid, tokens, group, kv_heads, block, columns, masked, cu, kv):
    args = (tokens, group, kv_heads, block, columns, masked, cu, kv)
    segments, parts = shares(rows, 512 if rows > 32 else 288, grid, *args)
    want = units(rows, *args)
    got, ctas = {}, {}
    for cta, kind, b, head, row0, nrows, tok0, _, _, tile0, ntiles in segments:
        nrows_w, first, tiles = want[b, head, row0]
        assert (nrows, tok0) == (nrows_w, first)
        at = got.get((b, head, row0), 0)
        assert tile0 == at and ntiles > 0  # the next tiles, in the order of the CTAs
        got[b, head, row0] = at + ntiles
        assert kind == (1 if tile0 else 0 if ntiles == tiles else 2)
        ctas.setdefault((b, head, row0), []).append(cta)
    assert got == {u: w[2] for u, w in want.items()}
    split = {u: c for u, c in ctas.items() if len(c) > 1}
    for u, c in split.items():
        assert c == list(range(c[0], c[0] + len(c)))
        assert parts[c[0]] == [len(c), want[u][1], u[1], u[2], want[u][0]]
    assert {c for c, x in parts.items() if x[0]} == {c[0] for c in split.values()}
    cost = sum(w[2] + COST[rows] for w in want.values())
    busy = min(grid, cost)
    for cta in range(grid):  # equal shares
        mine = sum(s[10] for s in segments if s[0] == cta)
        assert mine <= -(-cost // max(1, busy))


@pytest.mark.parametrize("rows", [16, 32, 128, 256])
@pytest.mark.parametrize("masked", [True, False])
def test_every_tile_is_taken_once(shares, rows, masked):
    rng = np.random.default_rng(rows)
    for requests in (1, 2, 7, 64, 700):
        new = rng.integers(0, 40 if requests < 700 else 4, requests)
        if requests == 2:
            new = np.array([1, 300])
        kv = new + rng.integers(0, 3000, requests) * rng.integers(0, 2, requests)
        cu = np.concatenate([[0], np.cumsum(new)])
        tokens = int(cu[-1])
        check(shares, rows, 148, tokens, 4, 2, 16, 100, masked, cu, kv)
        check(shares, rows, 5, tokens + 9, 3, 1, 24, 200, masked, cu + 4, kv)
        check(shares, rows, 148, max(1, tokens - 5), 4, 2, 16, 250, masked, cu, kv - 50)


@pytest.mark.parametrize("rows", [16, 128])
@pytest.mark.parametrize("masked", [True, False])
def test_requests_that_begin_before_the_first_token(shares, rows, masked):
    """Their tokens from the first one on are shared out like all others."""
    rng = np.random.default_rng(rows)
    for cut in (1, 3, 17, 70):
        new = rng.integers(0, 40, 7)
        kv = new + rng.integers(0, 3000, 7)
        cu = np.concatenate([[0], np.cumsum(new)])
        check(shares, rows, 148, int(cu[-1]) - cut, 4, 2, 16, 100, masked, cu - cut, kv)
    far = np.array([-2 ** 31, 5, 2 ** 31 - 1])
    for tokens in (3, 9):
        check(shares, rows, 148, tokens, 4, 2, 16, 100, masked, far, np.array([300, 1000]))


@pytest.mark.parametrize("rows", [16, 32, 128, 256])
@pytest.mark.parametrize("masked", [True, False])
def test_where_cu_new_descends_nothing_is_shared_out(shares, rows, masked):
    """Every second request would hold all tokens: some would be computed many times, and where the
    costs pass 32 bits others not at all."""
    threads = 512 if rows > 32 else 288
    for requests, tokens, columns in ((700, 4096, 65536), (3, 10, 20), (2000, 30000, 100000)):
        cu = np.tile([0, tokens], requests)[:requests + 1]
        kv = np.full(requests, columns * 16)
        segments, parts = shares(rows, threads, 148, tokens, 8, 8, 16, columns, masked, cu, kv)
        assert not segments
        assert len(parts) == 148 and all(x[0] == -1 for x in parts.values())
    cu = np.array([0, 5, 3, 8, 9])  # one step back is enough
    segments, parts = shares(rows, threads, 148, 9, 2, 2, 16, 20, masked, cu, np.full(4, 300))
    assert not segments and parts[0][0] == -1
