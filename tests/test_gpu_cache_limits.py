"""The paged 8-bit cache at the ends of what its calls allow: first use, many captured calls, the smallest scales, rows of a block in any order."""
import os
import subprocess
import sys

import pytest
import torch

import tinyfa_b200 as tfa
from test_gpu_cache import CODE, _cache, _expect, _store_by_hand, form  # noqa: F401

pytestmark = pytest.mark.gpu


def test_maxima_that_a_c_int_does_not_hold(form):  # noqa: F811
    cache = _cache("int8", [300], 2, 64, 16, 14)
    one, cu = torch.tensor([300], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    Q = torch.randn(2, 4, 64, device="cuda").half()
    want = tfa.flash_attn_cache_forward(Q, *cache, one, cu, 2, 300)
    _expect(want, Q, cache, [300], [2])
    for most in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 40):
        _expect(tfa.flash_attn_cache_forward(Q, *cache, one, cu, most, most), Q, cache, [300], [2])
