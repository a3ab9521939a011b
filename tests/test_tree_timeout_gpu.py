"""GPU: the attention of few rows leaves as a whole when one warp's wait runs out. The self-test lets
one warp of each CTA act as if it had (nothing stalls, nothing faults); the kernel must return, report
the status bit and leave the context usable."""
import pytest

from matcoredsl_b200 import _abi

pytestmark = pytest.mark.gpu

TIMEOUT_FULL = 1 << 0


def give_up(mcb, last):
    import torch
    lib = _abi.load()
    mcb.device_status(0, clear=True)
    for _ in range(2):
        code = lib.mcb_device_tree_timeout_selftest_v1(0, last)
        assert code == _abi.STATUS_CODE["DEVICE_TIMEOUT"], _abi.STATUS.get(code, code)
        assert mcb.device_status(0, clear=True) == TIMEOUT_FULL
    # an ordinary call afterwards: uniform weights over 300 keys
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.zeros(5, 64, 1, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.ones(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    o = mcb.tree_attention(q, k, torch.ones_like(k), i32(0, 1, 2, 3, 4)[None], i32(0, 1), i32(300))
    assert mcb.api.last_result.route == "tree_attention_few_rows"
    assert (o == 1).all() and mcb.device_status(0) == 0


def test_a_wait_that_runs_out_at_the_last_tile(mcb):
    """The other warps find the end of the work next."""
    give_up(mcb, 1)


def test_a_wait_that_runs_out_while_copies_are_on_their_way(mcb):
    """The keys and values of the next tiles are being copied: they land before the CTA ends."""
    give_up(mcb, 0)


def test_selftest_refuses_other_places(mcb):
    assert _abi.load().mcb_device_tree_timeout_selftest_v1(0, 2) == \
        _abi.STATUS_CODE["INVALID_ARGUMENT"]
