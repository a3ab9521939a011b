"""GPU: a bounded wait that has no abort flag to look at (the drains of work in flight at a kernel's
end) runs out with its own status bit, and the context stays usable. Nothing faults: the wait is on
a phase that nothing completes, with a limit of 10^6 cycles."""
import pytest

from matcoredsl_b200 import _abi

pytestmark = pytest.mark.gpu

TIMEOUT_FULL, TIMEOUT_DRAIN = 1 << 0, 1 << 3


def test_a_drain_that_never_ends_runs_out(mcb):
    import torch
    lib = _abi.load()
    mcb.device_status(0, clear=True)
    for _ in range(2):
        code = lib.mcb_device_timeout_selftest_v1(0, 1_000_000)
        assert code == _abi.STATUS_CODE["DEVICE_TIMEOUT"], _abi.STATUS.get(code, code)
        assert mcb.device_status(0, clear=True) == TIMEOUT_FULL | TIMEOUT_DRAIN
    x = torch.ones(128, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, 128, dtype=torch.bfloat16, device="cuda")
    y = mcb.gemm_epilogue(x, w, out_dtype="f32")
    assert (y == 64).all() and mcb.device_status(0) == 0
