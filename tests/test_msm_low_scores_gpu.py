"""GPU: matmul-softmax-matmul whose scores are all far below zero: the reference maximum of a row is one
of its scores and nothing else, or every weight would be 0."""
import numpy as np
import pytest

from tests import gpu_util as gu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,d", [(256, 256, 128), (128, 256, 128), (512, 1024, 64), (256, 200, 128)])
def test_all_scores_far_below_zero(mcb, orc, m, n, d):
    rng = np.random.default_rng(m + n + d)
    q = 1 + 0.1 * rng.standard_normal((1, 2, m, d), dtype=np.float32)
    k = -12 + 0.1 * rng.standard_normal((1, 2, n, d), dtype=np.float32)
    v = rng.standard_normal((1, 2, n, d), dtype=np.float32)
    (qh, qf), (kh, kf), (vh, vf) = (gu.bf16_pair(x) for x in (q, k, v))
    o = mcb.msm(gu.to_dev_bf16(qh), gu.to_dev_bf16(kh), gu.to_dev_bf16(vh), 1.0)
    assert mcb.api.last_result.route == "tcgen05_bf16_msm"
    got = gu.from_dev(o)
    for h in range(2):
        assert orc.rel_frobenius(got[0, h], orc.msm(qf[0, h], kf[0, h], vf[0, h], 1.0)) < 1e-2
