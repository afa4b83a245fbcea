"""flash_attn_scored_forward at the ends of its arguments' ranges: prefix lengths, document ids, positions and caps."""
import math

import pytest
import torch

import tinyfa_b200 as tfa
from plain64 import U, attend, check, visible
from test_gpu_scored import _compare, _inputs, _slopes

pytestmark = pytest.mark.gpu
LARGEST, SMALLEST = 2 ** 31 - 1, -(2 ** 31)
# tiles, tiles of one CTA, few rows with and without a merge, and fp32 on the CUDA cores and on the tensor cores
CALLS = [("fp16", 130, 300, 4, 2, 64, -1), ("bf16", 300, 300, 2, 1, 128, -1), ("bf16", 2, 500, 4, 2, 128, -1), ("fp16", 3, 4000, 2, 1, 64, -1),
         ("fp16", 140, 200, 2, 1, 256, -1), ("fp32", 130, 200, 2, 1, 64, 0), ("fp32", 130, 200, 2, 1, 64, 1), ("fp32", 140, 300, 1, 1, 192, 1)]


@pytest.fixture(params=CALLS, ids=lambda c: "-".join(map(str, c)))
def call(request):
    tfa.set_option("fp32_tc", request.param[6])
    yield request.param[:6]
    tfa.set_option("fp32_tc", -1)


@pytest.mark.parametrize("dtype,B,n,Skv,Hq,Hkv,D", [("fp16", 2, 3, 4000, 2, 1, 64), ("bf16", 9, 1, 700, 8, 2, 128), ("bf16", 40, 2, 300, 16, 16, 96), ("fp16", 5, 16, 1500, 1, 1, 256),
                                                     ("bf16", 3, 4, 9000, 4, 1, 32), ("fp16", 70, 1, 257, 32, 4, 192)])
@pytest.mark.parametrize("q_start", [0, 100])
def test_prefixes_of_entries_that_one_run_reads(dtype, B, n, Skv, Hq, Hkv, D, q_start):
    """A run of the decode kernel that goes on into the next batch entry goes on with that entry's prefix."""
    Q, K, V = _inputs(dtype, B, n, Skv, Hq, Hkv, D, 10)
    for turn in range(2):
        prefix = torch.tensor([[0, Skv, Skv // 2 + 1, 130][(b + turn) % 4] for b in range(B)], dtype=torch.int32, device="cuda")
        got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, prefix_lens=prefix, softcap=8.0, q_start=q_start)
        _compare(got, Q, K, V, True, 8.0, prefix=prefix, q_start=q_start)
