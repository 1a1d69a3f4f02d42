"""What the library cannot do is refused once, and not told of the calls after it."""
import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu


def test_failed_call_and_the_next(moehip):
    """Memory that is not there is refused once; the call after it is done."""
    M = moehip
    x, w = np.linspace(-1, 1, 64, dtype=np.float32), np.ones(64, np.float32)
    bufs = [M.DeviceBuffer.from_array(a) for a in (x, w, np.zeros(64, np.float32))]
    with pytest.raises(M.MoeError, match="emory"):
        M.DeviceBuffer(1 << 42)
    M.check(M.lib().moe_rmsnorm_dev(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, 1, 64, 1e-6), "rmsnorm")
    np.testing.assert_array_equal(bufs[2].download((64,), np.float32), O.rmsnorm(x.reshape(1, 64), w)[0])
