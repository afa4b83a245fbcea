"""The paged 8-bit cache on the GPU against its definition: tables and slots, rows written, attention, and a serving loop of all of them."""
import math
import random

import pytest
import torch

import tinyfa_b200 as tfa
from plain64 import U, attend, check

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODE = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


@pytest.fixture(params=[0, 1], ids=["stream", "tensor"])
def form(request):
    """Both forms of the attention kernel, whatever the sizes."""
    tfa.set_option("cache_tc", request.param)
    yield request.param
    tfa.set_option("cache_tc", -1)


# ---------------------------------------------------------------------------------------------------------- attention
def _cache(code, lens, Hkv, D, block, seed=0, spare=3, spread=1.0):
    """A cache of random codes and scales with a table in no order; cells behind a request's last token hold rubbish."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-n // block) for n in lens]
    n = sum(held) + spare
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(held + [1])
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-7] * (width - h))
        at += h
    out = []
    for _ in range(2):
        raw = torch.randint(-127, 128, (n, Hkv, block, D), device="cuda", generator=g)
        codes = raw.to(torch.int8) if code == "int8" else (raw.float() * 3.0).to(torch.float8_e4m3fn)
        scales = torch.exp(spread * torch.randn(n, Hkv, device="cuda", generator=g)) * (0.02 if code == "int8" else 0.01)
        out += [codes, scales]
    return out[0], out[2], out[1], out[3], torch.tensor(table, dtype=torch.int32, device="cuda").view(len(lens), width)


def _values(codes, scales, ids, length):
    x = codes.view(torch.uint8)[ids].view(codes.dtype).double() * scales[ids].double()[..., None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:length]


def _expect(got, Q, cache, lens, new, causal=True, cap=0.0, slopes=None):
    kc, vc, ks, vs, table = cache
    block, row = kc.shape[2], 0
    for b, (n, length) in enumerate(zip(new, lens)):
        if n == 0:
            continue
        ids = table[b, :-(-length // block)].long()
        k, v = _values(kc, ks, ids, length), _values(vc, vs, ids, length)
        i = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        see = (j <= i) if causal else (j >= 0) & (i == i)
        o, off, a = attend(Q[row:row + n].double(), k, v, see, cap, slopes, (i - j).abs().double())
        # Weights have 11 bits whatever the type of Q and are relative to a scale of V that is at most the largest; they are stored 2^3 larger
        # at least, so what falls below fp16's normal numbers is off by 2^-28 of the row's largest weight, times the largest code.
        floor = length * 2.0 ** -28 * 448.0 * vs[ids].max().item()
        check(got[row:row + n], o, off, a, U[torch.float16], floor)
        row += n
    assert (got[row:] == 0).all()


CASES = [  # dtype, code, lengths, new, Hq, Hkv, D, block
    ("fp16", "int8", [1], [1], 1, 1, 32, 16), ("bf16", "e4m3", [1, 2, 64, 65], [1, 1, 1, 1], 4, 2, 64, 64),
    ("bf16", "int8", [700, 1, 129], [1, 1, 1], 32, 8, 128, 16), ("fp16", "e4m3", [1000, 33], [3, 4], 4, 1, 96, 32),
    ("bf16", "e4m3", [500], [2], 6, 3, 192, 128), ("fp16", "int8", [300, 301], [1, 1], 4, 4, 256, 64),
    ("bf16", "int8", [90, 700], [90, 300], 8, 2, 128, 64), ("fp16", "e4m3", [200], [37], 5, 1, 64, 16),
    ("fp16", "int8", [5000], [1], 8, 1, 64, 32), ("bf16", "e4m3", [20000], [1], 16, 2, 128, 64),
    ("bf16", "e4m3", [17, 0, 40], [5, 0, 8], 4, 2, 32, 16), ("fp16", "int8", [250, 130], [40, 129], 12, 2, 256, 128),
    ("bf16", "int8", [257] * 40, [1] * 40, 4, 2, 96, 16), ("bf16", "e4m3", [3000, 10, 4000], [16, 2, 11], 24, 8, 128, 64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("what", ["plain", "cap", "bias", "all_keys"])
def test_attention_over_the_cache(case, what, form):
    dtype, code, lens, new, Hq, Hkv, D, block = case
    cache = _cache(code, lens, Hkv, D, block)
    g = torch.Generator(device="cuda").manual_seed(1)
    Q = (torch.randn(sum(new) + 2, Hq, D, device="cuda", generator=g) * 0.5).to(DT[dtype])  # two rows behind the last request
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cap = 3.0 if what == "cap" else 0.0
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device="cuda") if what == "bias" else None
    got = tfa.flash_attn_cache_forward(Q, *cache, n, cu, max(new), max(lens), is_causal=what != "all_keys", softcap=cap, alibi_slopes=slopes)
    _expect(got, Q, cache, lens, new, what != "all_keys", cap, slopes)
    # the maxima only size the launch
    again = tfa.flash_attn_cache_forward(Q, *cache, n, cu, 1, 1, is_causal=what != "all_keys", softcap=cap, alibi_slopes=slopes)
    _expect(again, Q, cache, lens, new, what != "all_keys", cap, slopes)
    tfa.device_status()


def test_block_scales_that_differ_by_orders_of_magnitude(form):
    """Weights are kept relative to the largest scale of V: rows that see small blocks only, and blocks of all sizes."""
    for code, dtype in (("int8", "bf16"), ("e4m3", "fp16")):
        cache = _cache(code, [400, 600], 2, 64, 16, 3, spread=1.0)
        cache[3].mul_(torch.logspace(-3, 1, cache[3].shape[0], device="cuda")[:, None])
        cache[2][5] = 0.0  # blocks of zeros
        cache[3][7] = 0.0
        Q = torch.randn(40, 4, 64, device="cuda").to(DT[dtype])
        cu, lens = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda"), torch.tensor([400, 600], dtype=torch.int32, device="cuda")
        got = tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 20, 600)
        _expect(got, Q, cache, [400, 600], [20, 20])


def test_caps_far_above_all_scores(form):
    """c tanh(s / c) is s within s^3 / 3 c^2 < 1e-7, and within 2.4e-6 |s| as it is computed, which the exponential's bound leaves room for."""
    for code, dtype, lens, new, cap in (("int8", "fp16", [400, 70], [1, 2], 1e5), ("e4m3", "bf16", [300], [90], 1e35)):
        cache = _cache(code, lens, 2, 64, 16, 6, spread=0.3)
        Q = (torch.randn(sum(new), 4, 64, device="cuda") * 0.3).to(DT[dtype])
        cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        got = tfa.flash_attn_cache_forward(Q, *cache, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, max(new), max(lens), softcap=cap)
        _expect(got, Q, cache, lens, new)


def test_nan_in_cells_and_blocks_that_no_request_has(form):
    cache = _cache("e4m3", [100, 37, 64], 2, 128, 16, 9)
    kc, vc, ks, vs, table = cache
    used = {int(i) for row, n in zip(table.tolist(), (100, 37, 64)) for i in row[:-(-n // 16)]}
    for c, s in ((kc, ks), (vc, vs)):
        raw = c.view(torch.uint8)
        for i in range(kc.shape[0]):
            if i not in used:
                raw[i] = 0x7F
                s[i] = math.nan
        raw[int(table[0, 6]), :, 4:] = 0x7F  # behind token 99
        raw[int(table[1, 2]), :, 5:] = 0xFF  # behind token 36
    cu = torch.tensor([0, 1, 20, 84], dtype=torch.int32, device="cuda")
    Q = torch.randn(84, 4, 128, device="cuda").half()
    got = tfa.flash_attn_cache_forward(Q, *cache, torch.tensor([100, 37, 64], dtype=torch.int32, device="cuda"), cu, 64, 100)
    _expect(got, Q, cache, [100, 37, 64], [1, 19, 64])


def test_calls_on_streams_and_graphs_at_once(form):
    """Arrival counters and parts belong to a stream or a captured call: eager calls on two streams and two graphs of one call side by side."""
    cache = _cache("int8", [9000, 2500, 40], 2, 128, 64, 10)
    lens = torch.tensor([9000, 2500, 40], dtype=torch.int32, device="cuda")
    jobs = []
    for n, new in enumerate(([1, 1, 1], [40, 3, 20])):
        cu = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32, device="cuda")
        Q = torch.randn(sum(new), 8, 128, device="cuda").half()
        jobs.append((Q, *cache, lens, cu, max(new), 9000))
    want = [tfa.flash_attn_cache_forward(*j) for j in jobs]
    torch.cuda.synchronize()
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append([tfa.flash_attn_cache_forward(*j) for j in jobs])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for k in range(10):
        for s, graph in zip(streams[:2], graphs):
            with torch.cuda.stream(s):
                graph.replay()
        for n, s in enumerate(streams[2:]):
            with torch.cuda.stream(s):
                got.append((n, tfa.flash_attn_cache_forward(*jobs[n])))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[n]) for n, x in got)
    for outs in held:
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
    tfa.device_status()


def test_queries_of_any_magnitude(form):
    """bf16 queries become fp16 with a power of two per row taken out."""
    cache = _cache("int8", [300], 1, 128, 16, 4)
    for scale in (2.0 ** -60, 2.0 ** -20, 2.0 ** -3):
        Q = (torch.randn(1, 4, 128, device="cuda") * scale).bfloat16()
        one = torch.tensor([300], dtype=torch.int32, device="cuda")
        got = tfa.flash_attn_cache_forward(Q, *cache, one, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, 300)
        _expect(got, Q, cache, [300], [1])
    Q = torch.zeros(1, 4, 128, device="cuda").bfloat16()
    got = tfa.flash_attn_cache_forward(Q, *cache, one, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, 300)
    _expect(got, Q, cache, [300], [1])


def test_rows_without_keys_and_blocks_that_do_not_exist(form):
    cache = _cache("e4m3", [100, 0, 64], 2, 64, 16, 5)
    kc, vc, ks, vs, table = cache
    cu, lens = torch.tensor([2, 5, 7, 75], dtype=torch.int32, device="cuda"), torch.tensor([100, 0, 64], dtype=torch.int32, device="cuda")
    Q = torch.randn(80, 4, 64, device="cuda").half()
    got = tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 68, 100)
    assert (got[:2] == 0).all() and (got[5:11] == 0).all() and (got[75:] == 0).all()  # 68 queries of 64 tokens: four have no position
    _expect(got[2:5], Q[2:5], (kc, vc, ks, vs, table), [100], [3])
    _expect(got[11:75], Q[11:75], (kc, vc, ks, vs, table[2:]), [64], [64])
    # a block id outside the cache: its keys are not seen
    bad = table.clone()
    bad[0, 1], bad[0, 3] = -5, kc.shape[0]
    got = tfa.flash_attn_cache_forward(Q[2:5], kc, vc, ks, vs, bad[:1], lens[:1], torch.tensor([0, 3], dtype=torch.int32, device="cuda"), 3, 100)
    ids = table[0, :7].long()
    k, v = _values(kc, ks, ids, 100), _values(vc, vs, ids, 100)
    j = torch.arange(100, device="cuda")[None]
    see = (j <= torch.arange(97, 100, device="cuda")[:, None]) & (j // 16 != 1) & (j // 16 != 3)
    o, off, a = attend(Q[2:5].double(), k, v, see)
    check(got, o, off, a, U[torch.float16], 100 * 2.0 ** -28 * 448.0 * vs[ids].max().item())


def test_calls_are_repeatable_on_streams_and_in_graphs(form):
    cache = _cache("int8", [3000, 70, 900, 1], 8, 128, 64, 6)
    lens = torch.tensor([3000, 70, 900, 1], dtype=torch.int32, device="cuda")
    cu = torch.arange(5, dtype=torch.int32, device="cuda")
    Q = torch.randn(4, 32, 128, device="cuda").bfloat16()
    call = lambda: tfa.flash_attn_cache_forward(Q, *cache, lens, cu, 1, 3000)  # noqa: E731
    want = call()
    for _ in range(20):
        assert torch.equal(call(), want)
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for s in streams * 5:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for n in ([3000, 70, 900, 1], [1, 2000 % 64, 100, 1]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        assert torch.equal(got, call())


def test_cache_past_32_bits():
    """Blocks past 2^31 bytes and 2^31 elements of the cache."""
    n, Hkv, block, D = 2200, 8, 128, 128  # 2.3e9 codes
    raw = torch.zeros(n, Hkv, block, D, dtype=torch.int8, device="cuda")
    ids = torch.tensor([2199, 0, 2100, 2150], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    raw[ids] = torch.randint(-127, 128, (4, Hkv, block, D), device="cuda", generator=g).to(torch.int8)
    scales = torch.full((n, Hkv), 0.02, device="cuda")
    cache = (raw, raw, scales, scales, ids.int().view(1, 4))
    Q = torch.randn(1, 8, D, device="cuda").half()
    got = tfa.flash_attn_cache_forward(Q, *cache, torch.tensor([500], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                       1, 500)
    _expect(got, Q, cache, [500], [1])
    K = torch.randn(1, Hkv, D, device="cuda").half()
    tfa.kv_cache_store(K, K, raw, raw.clone(), scales, scales.clone(), torch.tensor([2180 * block], device="cuda"))
    assert raw[2180, :, 0].abs().amax() == 127 and (raw[2180, :, 1:] == 0).all()


# -------------------------------------------------------------------------------------------------------------- store
def _store_by_hand(x, codes, scales, slots, code):
    """One row after the other, block by block, in fp32 with the roundings that the definition names: a new scale max |x| / top is stored
    rounded, codes are those of x top / max |x|."""
    dtype, top = CODE[code]
    block = codes.shape[2]
    codes, scales = codes.float().cpu(), scales.cpu().clone()
    x, slots = x.float().cpu(), slots.tolist()
    to = lambda y: (y.round() if code == "int8" else y).clamp(-top, top).to(dtype).float()  # noqa: E731
    r = 0
    while r < len(slots):
        if not 0 <= slots[r] < codes.shape[0] * block:
            r += 1
            continue
        blk, first, n = slots[r] // block, slots[r] % block, 1
        while r + n < len(slots) and slots[r + n] >= 0 and slots[r + n] // block == blk:
            n += 1
        part = x[r:r + n]
        finite = torch.where(part.isfinite(), part, 0.0).abs().amax((0, 2))
        need = torch.where(finite > 0, (finite / top).clamp(min=2.0 ** -126), 0.0)
        old = scales[blk] if first else torch.zeros_like(scales[blk])
        new = torch.maximum(old, need)
        run = (need >= old) & (need > 2.0 ** -126) & (finite <= 1e35)
        num, den = torch.where(run, top, 1.0)[:, None], torch.where(run, finite, torch.where(new > 0, new, 1.0))[:, None]
        for h in range(codes.shape[1]):
            if new[h] != old[h]:
                codes[blk, h, :first] = to(codes[blk, h, :first] * old[h] * num[h] / den[h])
        for i in range(n):
            y = part[i] * num / den
            codes[blk, :, slots[r + i] % block] = to(torch.where(y.isnan() | (new == 0)[:, None], 0.0, y))
        scales[blk] = new
        r += n
    return codes, scales


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("D,Hkv,block", [(32, 1, 16), (64, 3, 64), (96, 2, 32), (128, 8, 128), (256, 1, 16), (192, 2, 64)])
def test_store(dtype, code, D, Hkv, block):
    g = torch.Generator(device="cuda").manual_seed(D + block)
    n = 9
    kc, vc = (torch.randint(-100, 101, (n, Hkv, block, D), device="cuda", generator=g).float().to(CODE[code][0]) for _ in range(2))
    ks, vs = (torch.rand(n, Hkv, device="cuda", generator=g) * 0.02 for _ in range(2))
    # a run over three blocks, single rows in the middle of blocks (growing and not), padding, a slot past the cache
    slots = list(range(2 * block + 5, 2 * block + 5 + block)) + [7 * block + block - 1, -1, 4 * block + 3, 9 * block, 5 * block, 5 * block + 1, 0]
    T = len(slots)
    K, V = (torch.randn(T, Hkv, D, device="cuda", generator=g) * torch.logspace(-2, 1, T, device="cuda")[:, None, None] for _ in range(2))
    K, V = K.to(DT[dtype]), V.to(DT[dtype])
    V[-1] = 0.0
    slots = torch.tensor(slots, device="cuda")
    want = [_store_by_hand(x, c, s, slots, code) for x, c, s in ((K, kc, ks), (V, vc, vs))]
    tfa.kv_cache_store(K, V, kc, vc, ks, vs, slots)
    for (codes, scales), c, s in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(s.cpu(), scales)
        assert torch.equal(c.float().cpu(), codes)
    again = [x.clone() for x in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    tfa.kv_cache_store(K, V, kc, vc, ks, vs, slots)  # the same rows once more change nothing
    assert all(torch.equal(x, y) for x, y in zip(again, (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)))


def test_store_many_rows_and_specials():
    """Enough rows for the form with sixteen rows a CTA; infinities, NaN and denormals."""
    code, Hkv, D, block = "e4m3", 2, 64, 32
    n = 40
    kc = torch.zeros(n, Hkv, block, D, device="cuda").to(torch.float8_e4m3fn)
    vc, ks, vs = kc.clone(), torch.zeros(n, Hkv, device="cuda"), torch.zeros(n, Hkv, device="cuda")
    slots = torch.cat([torch.arange(100, 700), torch.arange(800, 1170)]).cuda()
    K = torch.randn(970, Hkv, D, device="cuda")
    K[5, 0, 3], K[6, 1, 4], K[40, 0, 0], K[50:90] = math.inf, math.nan, -math.inf, 1e-41
    K[500:600] = 0.0
    K[700:800] *= 3e37
    want = _store_by_hand(K, kc, ks, slots, code)
    tfa.kv_cache_store(K, K.clone(), kc, vc, ks, vs, slots)
    assert torch.equal(ks.cpu(), want[1]) and torch.equal(kc.float().cpu(), want[0])
    assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8)) and torch.equal(ks, vs)


def test_stored_rows_come_back_within_half_a_step():
    for code, step in (("int8", lambda x, s: s / 2), ("e4m3", lambda x, s: torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10))):
        dt, top = CODE[code]
        K = torch.randn(64, 4, 128, device="cuda")
        kc, ks = torch.zeros(2, 4, 64, 128, device="cuda").to(dt), torch.zeros(2, 4, device="cuda")
        tfa.kv_cache_store(K, K, kc, kc.clone(), ks, ks.clone(), torch.arange(64, 128, device="cuda"))
        got = (kc[1].float() * ks[1][:, None, None]).permute(1, 0, 2)
        assert ((got - K).abs() <= step(K, ks[1][None, :, None]) * (1 + 1e-5)).all()


# --------------------------------------------------------------------------------------------------------------- plan
def _plan_by_hand(table, lens, new, free, num_free, block, total, finished):
    table, lens, free, B, width = [r[:] for r in table], lens[:], free[:], len(lens), len(table[0])
    top = num_free
    for b in range(B):
        if finished[b]:
            for i in range(-(-lens[b] // block)):
                free[top] = table[b][i]
                top += 1
            lens[b] = 0
    have, asked, taken, after, slots, cu = top, 0, 0, [], [], [0]
    for b in range(B):
        n, held = max(new[b], 0), -(-lens[b] // block)
        fits = lens[b] + n <= width * block
        need = -(-(lens[b] + n) // block) - held if fits else 0
        asked += need
        served = fits and (need == 0 or asked <= have)
        if served:
            for i in range(need):
                table[b][held + i] = free[have - 1 - (asked - need) - i]
            taken += need
        slots += [table[b][t // block] * block + t % block if served else -1 for t in range(lens[b], lens[b] + n)]
        cu.append(cu[-1] + n)
        after.append(lens[b] + (n if served else 0))
    slots = (slots + [-1] * total)[:total]
    return slots, cu, after, have - taken, table, free


@pytest.mark.parametrize("B,most,block,spare,done", [(1, 1, 16, 5, 0.0), (3, 40, 16, 50, 0.3), (70, 1, 64, 100, 0.1), (70, 90, 32, 60, 0.2), (1500, 3, 16, 2000, 0.1),
                                                     (40, 700, 128, 400, 0.1), (2100, 1, 64, 900, 0.0), (5, 0, 16, 3, 1.0)])
def test_plan(B, most, block, spare, done):
    rng = random.Random(B + most)
    width = 12 if most < 100 else 16
    lens = [rng.randint(0, width * block) for _ in range(B)]
    new = [rng.randint(-1, most) for _ in range(B)]
    held = [-(-n // block) for n in lens]
    ids = list(range(sum(held) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    free = ids[at:] + [-1] * at
    finished = [rng.random() < done for _ in range(B)]
    total = sum(max(n, 0) for n in new) + 3
    want = _plan_by_hand(table, lens, new, free, spare, block, total, finished)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    t, f, held_lens = i32(table), i32(free), i32(lens)
    slots, cu, after, left = tfa.kv_cache_plan(t, held_lens, i32(new), f, i32([spare]), block, total, torch.tensor(finished, device="cuda") if done else None)
    assert slots.dtype == torch.int64 and slots.tolist() == want[0]
    assert cu.tolist() == want[1] and after.tolist() == want[2] and left.tolist() == [want[3]]
    assert t.tolist() == want[4] and f.tolist() == want[5]
    assert held_lens.tolist() == lens


# --------------------------------------------------------------------------------------------------------------- loop
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "fp16")])
def test_serving_loop(code, dtype, form):
    """Prompts, chunks and single tokens through tables, store and attention; requests end and their places are taken again.  The cache's
    contents after every step are those of a store by hand, and the attention that of the cache's contents."""
    Hq, Hkv, D, block, B, pool = 8, 2, 64, 16, 5, 60
    rng = random.Random(3)
    dt = CODE[code][0]
    kc = torch.zeros(pool, Hkv, block, D, device="cuda").to(dt)
    vc, ks, vs = kc.clone(), torch.zeros(pool, Hkv, device="cuda"), torch.zeros(pool, Hkv, device="cuda")
    table = torch.full((B, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    free, num_free = torch.arange(pool, dtype=torch.int32, device="cuda"), torch.tensor([pool], dtype=torch.int32, device="cuda")
    for step in range(12):
        done = [step > 3 and rng.random() < 0.2 for _ in range(B)]
        held = [0 if d else n for n, d in zip(lens.tolist(), done)]
        new = [rng.choice([1, 1, 1, 7, 40]) if n < 140 else 1 for n in held]
        total = sum(new)
        slots, cu, lens, num_free = tfa.kv_cache_plan(table, lens, torch.tensor(new, dtype=torch.int32, device="cuda"), free, num_free, block, total,
                                                      finished=torch.tensor(done, device="cuda"))
        assert lens.tolist() == [h + n for h, n in zip(held, new)] and (slots >= 0).all() and slots.unique().numel() == total
        K, V = (torch.randn(total, Hkv, D, device="cuda").to(DT[dtype]) for _ in range(2))
        want = [_store_by_hand(x, c, s, slots, code) for x, c, s in ((K, kc, ks), (V, vc, vs))]
        tfa.kv_cache_store(K, V, kc, vc, ks, vs, slots)
        assert torch.equal(kc.float().cpu(), want[0][0]) and torch.equal(vc.float().cpu(), want[1][0])
        assert torch.equal(ks.cpu(), want[0][1]) and torch.equal(vs.cpu(), want[1][1])
        Q = torch.randn(total, Hq, D, device="cuda").to(DT[dtype])
        got = tfa.flash_attn_cache_forward(Q, kc, vc, ks, vs, table, lens, cu, max(new), 192, softcap=30.0)
        _expect(got, Q, (kc, vc, ks, vs, table), lens.tolist(), new, True, 30.0)
    in_use = sum(-(-n // block) for n in lens.tolist())
    assert num_free.item() == pool - in_use
    live = [table[b, :-(-n // block)] for b, n in enumerate(lens.tolist())] + [free[:num_free.item()]]
    assert torch.cat(live).sort().values.tolist() == list(range(pool))
