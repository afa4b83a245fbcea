"""Calls of the cache that are refused before any work on a device."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from tinyfa_b200 import _lib, api


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 15) & ~15
    del buf


def test_plan_lengths_that_overlap(p):
    """Slots follow from the lengths before and after: they cannot be one array."""
    f = _lib.load().tfa_b200_kv_cache_plan

    def call(before, after, batch=4):
        return f(p, before, p + 512, None, p + 1024, p + 1536, p + 1600, p + 2048, after, p + 2560, batch, 4, 4, 16, 4, None)

    for before, after in ((p + 3200, p + 3200), (p + 3200, p + 3212), (p + 3212, p + 3200)):
        assert call(before, after) == 3 and "overlap" in _lib.last_error()


def test_gradients_of_either_mode():
    x, y = torch.randn(3), torch.randn(3)
    api._check_no_grad(x, None, y)
    with pytest.raises(RuntimeError, match="forward only"):
        api._check_no_grad(x, y.clone().requires_grad_())
    with forward_ad.dual_level():
        api._check_no_grad(x, y)
        with pytest.raises(RuntimeError, match="forward only"):
            api._check_no_grad(x, forward_ad.make_dual(y, x))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward only"):
            api._check_no_grad(forward_ad.make_dual(x, y))
    api._check_no_grad(x, y)
