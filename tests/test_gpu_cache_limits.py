"""The paged 8-bit cache at the ends of what its calls allow: first use, many captured calls, the smallest scales, rows of a block in any order."""
import os
import subprocess
import sys

import pytest
import torch

import tinyfa_b200 as tfa
from test_gpu_cache import CODE, _cache, _expect, _store_by_hand, form  # noqa: F401

pytestmark = pytest.mark.gpu


FIRST_USE = """
import torch
import tinyfa_b200 as tfa
lens, new, Hq, Hkv, D, block = [9000, 2500, 40], [1, 1, 1], 8, 2, 128, 64
held = [-(-n // block) for n in lens]
g = torch.Generator(device="cuda").manual_seed(0)
kc, vc = (torch.randint(-127, 128, (sum(held), Hkv, block, D), device="cuda", generator=g).to(torch.int8) for _ in range(2))
ks, vs = (torch.rand(sum(held), Hkv, device="cuda", generator=g) * 0.02 for _ in range(2))
table, at = torch.full((3, max(held)), -1, dtype=torch.int32), 0
for b, h in enumerate(held):
    table[b, :h] = torch.arange(at, at + h)
    at += h
Q = torch.randn(3, Hq, D, device="cuda", generator=g).half()
args = (Q, kc, vc, ks, vs, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda"), 1, 9000)
side = torch.cuda.Stream()
torch.cuda.synchronize()
torch.cuda._sleep(20_000_000)  # some milliseconds on the default stream
with torch.cuda.stream(side):
    got = [tfa.flash_attn_cache_forward(*args) for _ in range(50)]
torch.cuda.synchronize()
want = tfa.flash_attn_cache_forward(*args)
assert want.abs().sum() > 0 and all(torch.equal(x, want) for x in got)
"""


def _run(code):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_first_call_of_a_process_on_a_side_stream():
    """The arrival counters are zero before any stream counts with them, whatever is queued on the default stream."""
    _run(FIRST_USE)


def test_first_attention_call_of_a_process_on_a_side_stream():
    """The same for the work counters of the tile kernel."""
    _run("""
import torch
import tinyfa_b200 as tfa
Q, K, V = (torch.randn(2, 600, 8, 64, device="cuda").half() for _ in range(3))
side = torch.cuda.Stream()
torch.cuda.synchronize()
torch.cuda._sleep(20_000_000)
with torch.cuda.stream(side):
    got = [tfa.flash_attn_forward(Q, K, V, True) for _ in range(50)]
torch.cuda.synchronize()
want = tfa.flash_attn_forward(Q, K, V, True)
assert all(torch.equal(x, want) for x in got)
tfa.device_status()
""")


@pytest.mark.parametrize("form", [0, 1])
def test_first_call_of_a_process_under_capture(form):  # noqa: F811
    _run(FIRST_USE.split("side = ")[0] + f"tfa.set_option('cache_tc', {form})" + """
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = tfa.flash_attn_cache_forward(*args)
for _ in range(3):
    got.zero_()
    graph.replay()
    want = tfa.flash_attn_cache_forward(*args)
    assert want.abs().sum() > 0 and torch.equal(got, want)
""")


def test_more_captured_calls_than_the_work_counters_have_room_for():
    """A decode graph for each batch size of a server and each layer of a model."""
    cache = _cache("int8", [2500, 40], 2, 64, 64, 11)
    lens, cu = torch.tensor([2500, 40], dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    Q = torch.randn(2, 8, 64, device="cuda").half()
    want = tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 1, 2500)
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append([tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 1, 2500) for _ in range(1700)])
        graphs.append(graph)
    for graph, outs in zip(graphs, held):
        for _ in range(2):
            graph.replay()
        assert all(torch.equal(x, want) for x in outs)
    assert torch.equal(tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 1, 2500), want)
    tfa.device_status()
