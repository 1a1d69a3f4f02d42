"""What the Python wrappers of the paged cache refuse before any device memory is made or read.  CPU only."""
import types

import numpy as np
import pytest

import moehip as M


def test_cache_of_another_number_of_layers():
    """The C call reads as many pages as the model has layers from the cache's array."""
    m = M.Model.__new__(M.Model)
    m.h, m.V = None, 10
    m.cfg = M.qwen_config(64, 3, 16, 4, 2, 32, 8, 8, 10)
    moved = []
    for n in (0, 2, 4):
        cache = types.SimpleNamespace(layers=(M.Pages * n)(), n_req=1, set_step=lambda *a: moved.append(a))
        with pytest.raises(M.MoeError, match="layers"):
            m.step_paged(cache, [1], np.zeros(1, np.int32))
    assert not moved


@pytest.mark.parametrize("side", ["k_scale", "v_scale"])
@pytest.mark.parametrize("shape", [(), (1,), (3,), (5,), (4, 1)])
def test_scales_of_another_number_of_heads(side, shape, monkeypatch):
    """The kernels read one scale for each key-value head."""
    def none(*a):
        raise AssertionError("device memory was made")

    monkeypatch.setattr(M.DeviceBuffer, "__init__", none)
    with pytest.raises(M.MoeError, match=side):
        M.PagedCache(2, 4, 64, 10, 16, 2, 4, 8, M.PAGE_E4M3, **{side: np.ones(shape, np.float32)})
