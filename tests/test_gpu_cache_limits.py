"""The paged 8-bit cache at the ends of what its calls allow: first use, many captured calls, the smallest scales, rows of a block in any order."""
import os
import subprocess
import sys

import pytest
import torch

import tinyfa_b200 as tfa
from test_gpu_cache import CODE, DT, _cache, _expect, _store_by_hand, form  # noqa: F401

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


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_smallest_scales(code, form):  # noqa: F811
    """Scales that kv_cache_store writes for the smallest values, alone, and beside blocks of zeros and of 2^-120."""
    lens, new = [400, 90, 300], [3, 1, 70]
    for kind in ("alone", "mixed"):
        cache = _cache(code, lens, 2, 64, 16, 12)
        vs = cache[3]
        vs.fill_(2.0 ** -126)
        if kind == "mixed":
            vs[::3] = 2.0 ** -120
            vs[1::5] = 0.0
        Q = torch.randn(sum(new), 4, 64, device="cuda").bfloat16()
        cu = torch.tensor([0, 3, 4, 74], dtype=torch.int32, device="cuda")
        got = tfa.flash_attn_cache_forward(Q, *cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, 70, 400)
        _expect(got, Q, cache, lens, new)
    tfa.device_status()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("what", ["begins", "grows"])
def test_rows_of_a_block_in_any_order(code, what):
    """Rows of a block follow one another, in whatever order of their cells: as if they came in ascending order."""
    g = torch.Generator().manual_seed(13)
    for block, D, dtype in ((16, 64, torch.float16), (128, 256, torch.float32), (64, 128, torch.bfloat16)):
        n, Hkv = 40, 2
        kc = torch.randint(-100, 101, (n, Hkv, block, D), device="cuda").float().to(CODE[code][0])
        ks = torch.full((n, Hkv), 50.0 if what == "begins" else 1e-3, device="cuda")
        runs = []
        for blk in torch.randperm(n, generator=g).tolist()[:30]:
            first = 0 if what == "begins" else int(torch.randint(1, block - 3, (1,), generator=g))
            cells = torch.arange(first, int(torch.randint(first + 1, block + 1, (1,), generator=g)))
            cells = cells[torch.randperm(len(cells), generator=g)]
            if what == "begins" and len(cells) > 1 and cells[0] == 0:
                cells = cells.flip(0)
            runs.append(blk * block + cells)
        slots = torch.cat(runs).cuda()
        rise = torch.cat([r.argsort() + sum(map(len, runs[:i])) for i, r in enumerate(runs)]).cuda()
        K = torch.randn(len(slots), Hkv, D, device="cuda").to(dtype)
        want = _store_by_hand(K[rise], kc, ks, slots[rise], code)
        vc, vs = kc.clone(), ks.clone()
        tfa.kv_cache_store(K, K.clone(), kc, vc, ks, vs, slots)
        assert torch.equal(ks.cpu(), want[1]) and torch.equal(kc.float().cpu(), want[0])
        assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8)) and torch.equal(ks, vs)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    cache = _cache("int8", [20], 1, 64, 16)
    one, cu = torch.tensor([20], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    Q, K = torch.randn(1, 2, 64, device="cuda").half(), torch.randn(1, 1, 64, device="cuda").half()
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="forward only"):
            tfa.flash_attn_cache_forward(fwd.make_dual(Q, Q), *cache, one, cu, 1, 20)
        with pytest.raises(RuntimeError, match="forward only"):
            tfa.kv_cache_store(K, fwd.make_dual(K.clone(), K), *cache[:4], torch.tensor([3], device="cuda"))


def test_maxima_that_a_c_int_does_not_hold(form):  # noqa: F811
    cache = _cache("int8", [300], 2, 64, 16, 14)
    one, cu = torch.tensor([300], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    Q = torch.randn(2, 4, 64, device="cuda").half()
    want = tfa.flash_attn_cache_forward(Q, *cache, one, cu, 2, 300)
    _expect(want, Q, cache, [300], [2])
    for most in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 40):
        _expect(tfa.flash_attn_cache_forward(Q, *cache, one, cu, most, most), Q, cache, [300], [2])


def test_caps_below_and_above_what_fp32_holds(form):  # noqa: F811
    cache = _cache("e4m3", [300], 2, 64, 16, 15)
    one, cu = torch.tensor([300], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    Q = torch.randn(2, 4, 64, device="cuda").half()
    got = tfa.flash_attn_cache_forward(Q, *cache, one, cu, 2, 300, softcap=1e-60)
    _expect(got, Q * 0, cache, [300], [2])
    got = tfa.flash_attn_cache_forward(Q * 0.1, *cache, one, cu, 2, 300, softcap=1e60)
    _expect(got, Q * 0.1, cache, [300], [2])


@pytest.mark.parametrize("dtype,code,D,block", [("fp16", "int8", 64, 16), ("bf16", "e4m3", 128, 64), ("fp16", "e4m3", 256, 32), ("bf16", "int8", 96, 128)])
@pytest.mark.parametrize("factor", [4, 40])
def test_scores_on_both_sides_of_half_a_cap(dtype, code, D, block, factor, form):  # noqa: F811
    """Some below half the cap, where the tanh is a polynomial, some far above, in the same blocks."""
    lens, new = [700, 90], [3, 70]
    cache = _cache(code, lens, 2, D, block, 16, spread=0.3)
    Q = (torch.randn(sum(new), 4, D, device="cuda") * factor).to(DT[dtype])
    cu = torch.tensor([0, 3, 73], dtype=torch.int32, device="cuda")
    got = tfa.flash_attn_cache_forward(Q, *cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, 70, 700, softcap=30.0)
    _expect(got, Q, cache, lens, new, True, 30.0)
