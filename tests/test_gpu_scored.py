"""flash_attn_scored_forward on the GPU against 64 bits: caps, distance bias, prefix and document masks, first positions."""
import math

import pytest
import torch

import tinyfa_b200 as tfa
from plain64 import U, attend, check, visible

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _inputs(dtype, B, Sq, Skv, Hq, Hkv, D, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(B, s, h, D, device="cuda", generator=g).to(DT[dtype]) for s, h in ((Sq, Hq), (Skv, Hkv), (Skv, Hkv)))


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")


def _compare(got, Q, K, V, causal, cap=0.0, slopes=None, prefix=None, dq=None, dk=None, q_start=0, fp32_error=2.0 ** -21):
    for b in range(Q.shape[0]):
        see, dist = visible(Q.shape[1], K.shape[1], causal, q_start, None if prefix is None else int(prefix[b]), None if dq is None else dq[b],
                            None if dk is None else dk[b])
        o, off, a = attend(Q[b].double(), K[b].double(), V[b].double(), see, cap, slopes, dist,
                            fp32_error if Q.dtype == torch.float32 else 8.6e-5)
        check(got[b], o, off, a, U[Q.dtype], K.shape[1] * 2.0 ** -25 * V[b].abs().max().item() if Q.dtype == torch.float16 else 0.0)


SHAPES = [  # dtype, B, Sq, Skv, Hq, Hkv, D
    ("fp16", 1, 1, 1, 1, 1, 32), ("bf16", 2, 7, 9, 3, 1, 64), ("fp16", 2, 130, 257, 4, 2, 96), ("bf16", 1, 300, 300, 8, 2, 128),
    ("fp16", 1, 200, 461, 2, 2, 192), ("bf16", 1, 131, 300, 4, 1, 256), ("bf16", 2, 517, 333, 6, 3, 32), ("fp16", 3, 257, 129, 4, 4, 64),
    ("fp32", 1, 1, 3, 2, 1, 32), ("fp32", 2, 65, 130, 4, 2, 64), ("fp32", 1, 130, 67, 2, 2, 96), ("fp32", 1, 100, 129, 2, 1, 128),
    ("fp32", 1, 66, 66, 1, 1, 192), ("fp32", 1, 70, 140, 2, 1, 256),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("what", ["mask", "cap", "bias", "both"])
@pytest.mark.parametrize("causal", [False, True])
def test_cap_and_bias(shape, what, causal):
    dtype, B, Sq, Skv, Hq, Hkv, D = shape
    Q, K, V = _inputs(dtype, B, Sq, Skv, Hq, Hkv, D)
    cap = 2.5 if what in ("cap", "both") else 0.0
    slopes = _slopes(Hq) if what in ("bias", "both") else None
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=causal, softcap=cap, alibi_slopes=slopes)
    _compare(got, Q, K, V, causal, cap, slopes)
    tfa.device_status()


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_prefix(shape):
    dtype, B, Sq, Skv, Hq, Hkv, D = shape
    Q, K, V = _inputs(dtype, B, Sq, Skv, Hq, Hkv, D, 1)
    prefix = torch.tensor([[0, Skv // 3 + 1, Skv + 500][b % 3] for b in range(B)], dtype=torch.int32, device="cuda")
    slopes = _slopes(Hq)
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, prefix_lens=prefix, alibi_slopes=slopes)
    _compare(got, Q, K, V, True, slopes=slopes, prefix=prefix)


def _documents(B, S, mean, seed, pad=True, shuffle=False):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b in range(B):
        row, d = [], 3 * b
        while len(row) < S:
            row += [d] * (1 + int(torch.empty(1).exponential_(1.0 / mean, generator=g)))
            d += 1
        row = row[:S]
        if pad:
            row[S - S // 5:] = [-1] * (S // 5)
        if shuffle:
            row = [row[i] for i in torch.randperm(S, generator=g).tolist()]
        rows.append(row)
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,B,S,Hq,Hkv,D", [("fp16", 2, 700, 4, 2, 64), ("bf16", 1, 1100, 8, 2, 128), ("bf16", 3, 130, 2, 2, 32), ("fp16", 1, 600, 2, 1, 256),
                                                ("fp32", 2, 300, 4, 2, 64), ("fp32", 1, 200, 1, 1, 256), ("bf16", 1, 20, 4, 1, 96), ("fp16", 1, 500, 2, 2, 192)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["ascending", "shuffled", "all_padding", "one"])
def test_documents(dtype, B, S, Hq, Hkv, D, causal, kind):
    Q, K, V = _inputs(dtype, B, S, S, Hq, Hkv, D, 2)
    if kind == "all_padding":
        docs = torch.full((B, S), -1, dtype=torch.int32, device="cuda")
    elif kind == "one":
        docs = torch.full((B, S), 7, dtype=torch.int32, device="cuda")
    else:
        docs = _documents(B, S, 90, 5, shuffle=kind == "shuffled")
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=causal, softcap=4.0, doc_ids_q=docs, doc_ids_kv=docs)
    _compare(got, Q, K, V, causal, 4.0, dq=docs, dk=docs)
    assert (got[docs < 0] == 0).all()


def test_documents_of_other_keys_with_prefix_and_start():
    Q, K, V = _inputs("bf16", 2, 150, 900, 4, 2, 128, 3)
    dk = _documents(2, 900, 200, 8, pad=False)
    dq = dk[:, 400:550].contiguous()
    prefix = torch.tensor([450, 0], dtype=torch.int32, device="cuda")
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, prefix_lens=prefix, doc_ids_q=dq, doc_ids_kv=dk, q_start=400)
    _compare(got, Q, K, V, True, prefix=prefix, dq=dq, dk=dk, q_start=400)


@pytest.mark.parametrize("dtype,B,n,L,Hq,Hkv,D", [("bf16", 3, 1, 1000, 8, 2, 128), ("fp16", 2, 4, 5000, 4, 1, 64), ("bf16", 1, 1, 9001, 32, 8, 96), ("fp16", 5, 3, 300, 5, 1, 32),
                                                  ("bf16", 1, 2, 3000, 4, 2, 192), ("fp16", 1, 1, 2049, 2, 1, 256), ("fp32", 2, 3, 700, 4, 2, 128),
                                                  ("bf16", 2, 40, 6000, 8, 2, 128), ("fp16", 3, 5, 6455, 4, 1, 96), ("bf16", 1, 60, 9000, 2, 1, 32), ("fp16", 1, 50, 5000, 4, 1, 192), ("fp16", 1, 17, 12000, 4, 4, 64), ("bf16", 1, 100, 4000, 2, 1, 256)])
@pytest.mark.parametrize("extra", [0, 77])
def test_tokens_and_chunks_behind_keys(dtype, B, n, L, Hq, Hkv, D, extra):
    """Single tokens, draft tokens and chunks at the end of the keys (or with keys behind them that they do not see)."""
    Q, K, V = _inputs(dtype, B, n, L + n + extra, Hq, Hkv, D, 4)
    slopes = _slopes(Hq)
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, softcap=20.0, alibi_slopes=slopes, q_start=L)
    _compare(got, Q, K, V, True, 20.0, slopes, q_start=L)
    if n > 1:  # without the mask
        _compare(tfa.flash_attn_scored_forward(Q, K, V, softcap=20.0), Q, K, V, False, 20.0)
    tfa.device_status()


def test_matches_the_plain_call_without_options():
    for dtype, D in (("bf16", 128), ("fp16", 64)):
        Q, K, V = _inputs(dtype, 2, 500, 500, 4, 2, D, 6)
        for causal in (False, True):
            want = tfa.flash_attn_forward(Q, K, V, causal)
            assert torch.equal(tfa.flash_attn_scored_forward(Q, K, V, causal), want)


def test_scores_far_past_the_cap():
    """Scores of hundreds against a cap of 1 and 30: all weights are within e^2c of each other, nothing overflows."""
    for dtype in ("fp16", "bf16", "fp32"):
        Q, K, V = _inputs(dtype, 1, 200, 300, 2, 1, 64, 7)
        for cap in (1.0, 30.0):
            got = tfa.flash_attn_scored_forward(Q * 30, K * 30, V, softcap=cap)
            assert torch.isfinite(got).all()
            if cap == 1.0:
                # a score of hundreds is +-1 after the cap, but the few near zero follow their error: 900 D 2^-24 sum |q k|
                _compare(got, Q * 30, K * 30, V, False, cap)


def test_large_q_start_keeps_distances():
    Q, K, V = _inputs("bf16", 1, 1, 4000, 4, 1, 64, 8)
    slopes = _slopes(4) * 0.01
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, alibi_slopes=slopes, q_start=5000)
    _compare(got, Q, K, V, True, slopes=slopes, q_start=5000)


def test_replayed_graph_and_side_stream():
    Q, K, V = _inputs("bf16", 2, 300, 300, 8, 2, 128, 9)
    docs = _documents(2, 300, 70, 1)
    args = dict(is_causal=True, softcap=30.0, doc_ids_q=docs, doc_ids_kv=docs)
    want = tfa.flash_attn_scored_forward(Q, K, V, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tfa.flash_attn_scored_forward(Q, K, V, **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = tfa.flash_attn_scored_forward(Q, K, V, **args)
    for seed in (10, 11):
        q2, k2, v2 = _inputs("bf16", 2, 300, 300, 8, 2, 128, seed)
        Q.copy_(q2), K.copy_(k2), V.copy_(v2)
        graph.replay()
        assert torch.equal(captured, tfa.flash_attn_scored_forward(Q, K, V, **args))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_nan_keys_and_values_in_places_nobody_sees(dtype):
    """Padding of a batch may hold anything; keys that a row masks may be NaN."""
    Q, K, V = _inputs(dtype, 2, 260, 260, 4, 2, 64, 12)
    docs = _documents(2, 260, 60, 3)
    want = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, doc_ids_q=docs, doc_ids_kv=docs)
    pad = docs < 0
    Q[pad], K[pad] = math.nan, math.inf
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, doc_ids_q=docs, doc_ids_kv=docs)
    assert torch.equal(got, want)
    K[:, 200:] = math.nan  # the causal mask hides them from the rows before
    got = tfa.flash_attn_scored_forward(Q[:, :200].contiguous(), K, V, is_causal=True, doc_ids_q=docs[:, :200].contiguous(), doc_ids_kv=docs)
    assert torch.equal(got, want[:, :200])


@pytest.mark.parametrize("dtype,B,Sq,Skv,Hq,Hkv,D", [("fp16", 1, 200, 300, 2, 1, 64), ("bf16", 1, 150, 150, 2, 2, 128), ("fp16", 2, 2, 900, 4, 2, 64),
                                                      ("bf16", 1, 1, 5000, 8, 2, 128), ("fp32", 1, 150, 200, 2, 1, 64), ("fp32", 1, 40, 50, 2, 1, 128)])
@pytest.mark.parametrize("cap", [1e5, 1e35])
def test_caps_far_above_all_scores(dtype, B, Sq, Skv, Hq, Hkv, D, cap):
    """c tanh(s / c) is s within s^3 / 3 c^2 < 1e-8, and within 2.4e-6 |s| as it is computed: 2 x 2.4e-6 x 8 < 4e-5 of A, inside the
    exponential's 8.6e-5, of which these calls use a part; fp32 has an exact tanh."""
    Q, K, V = _inputs(dtype, B, Sq, Skv, Hq, Hkv, D, 40)
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, softcap=cap, q_start=Skv - Sq)
    _compare(got, Q, K, V, True, q_start=Skv - Sq, fp32_error=2.0 ** -19)
    tiny = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, softcap=1e-36, q_start=Skv - Sq)  # all scores are zero: means of V
    _compare(tiny, Q * 0, K, V, True, q_start=Skv - Sq, fp32_error=2.0 ** -19)


def test_calls_on_streams_and_threads_at_once():
    """Partial results, document tables and work counters belong to a call, whatever runs beside it."""
    import threading

    shapes = [("bf16", 1, 3, 6000, 8, 2, 128), ("fp16", 1, 100, 4000, 2, 1, 64), ("bf16", 2, 600, 600, 4, 2, 96), ("fp32", 1, 300, 900, 2, 1, 64)]
    jobs = []
    for n, shape in enumerate(shapes):
        Q, K, V = _inputs(*shape, 50 + n)
        kw = dict(is_causal=True, softcap=5.0, q_start=shape[3] - shape[2])
        if n == 2:
            docs = _documents(2, 600, 100, 8)
            kw.update(doc_ids_q=docs, doc_ids_kv=docs)
        jobs.append((Q, K, V, kw, tfa.flash_attn_scored_forward(Q, K, V, **kw)))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(12):
                Q, K, V, kw, want = jobs[(i + k) % len(jobs)]
                got = tfa.flash_attn_scored_forward(Q, K, V, **kw)
                if not torch.equal(got, want):
                    wrong.append((i, k))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    tfa.device_status()


FP32_SHAPES = [  # B, Sq, Skv, Hq, Hkv: one key, tile edges, heads in one tile, several key ranges, more than one batch entry
    (1, 1, 1, 1, 1), (2, 3, 1300, 8, 2), (1, 127, 129, 3, 1), (2, 129, 300, 4, 4), (1, 300, 1500, 2, 1), (3, 140, 131, 6, 2),
]


@pytest.mark.parametrize("D", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("shape", FP32_SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_both_fp32_forms(shape, D):
    """CUDA cores and three bf16 parts per float.  The latter's scores: six passes of D/16 steps, each truncating once (2^-23 of the sum), and
    the two products of 2^-24 that are left out: 0.75 D + 2 units of 2^-24, within plain64's D.  P V: the last pass of a block of 128 keys
    truncates 8 times at full magnitude, 2^-20 A (the five before it at 2^-8 of that), blocks are added with 2^-24 each, and the parts
    left out are 2^-23: with plain64's 2^-21 for the exponential together below 2^-19."""
    B, Sq, Skv, Hq, Hkv = shape
    Q, K, V = _inputs("fp32", *shape, D, 20)
    prefix = torch.tensor([[0, Skv // 3 + 1, Skv + 500][b % 3] for b in range(B)], dtype=torch.int32, device="cuda")
    docs = _documents(B, max(Sq, Skv), 70, 5)
    mixed = _documents(B, max(Sq, Skv), 70, 5, shuffle=True)
    slopes = _slopes(Hq)
    calls = [
        (dict(is_causal=True, softcap=2.5, alibi_slopes=slopes), dict(cap=2.5, slopes=slopes)),
        (dict(is_causal=False, alibi_slopes=slopes), dict(slopes=slopes)),
        (dict(is_causal=True, softcap=0.7, prefix_lens=prefix), dict(cap=0.7, prefix=prefix)),
        (dict(is_causal=True, q_start=max(Skv - Sq, 0), alibi_slopes=slopes), dict(q_start=max(Skv - Sq, 0), slopes=slopes)),
        (dict(is_causal=True, doc_ids_q=docs[:, :Sq].contiguous(), doc_ids_kv=docs[:, :Skv].contiguous()), dict(dq=docs[:, :Sq], dk=docs[:, :Skv])),
        (dict(is_causal=False, doc_ids_q=docs[:, :Sq].contiguous(), doc_ids_kv=mixed[:, :Skv].contiguous(), alibi_slopes=slopes),
         dict(dq=docs[:, :Sq], dk=mixed[:, :Skv], slopes=slopes)),
    ]
    for form, error in ((0, 2.0 ** -21), (1, 2.0 ** -19)):
        tfa.set_option("fp32_tc", form)
        try:
            for args, plain in calls:
                got = tfa.flash_attn_scored_forward(Q, K, V, **args)
                _compare(got, Q, K, V, args["is_causal"], fp32_error=error, **plain)
            tfa.device_status()
        finally:
            tfa.set_option("fp32_tc", -1)


def test_fp32_call_in_pieces():
    """A workspace beyond what the pool keeps: fewer batch entries at a time, each with its part of the tables, slopes and prefixes."""
    B, S, H, D = 260, 520, 16, 64
    g = torch.Generator(device="cuda").manual_seed(60)
    Q, K, V = (torch.randn(B, S, H, D, device="cuda", generator=g) for _ in range(3))
    docs, slopes = _documents(B, S, 200, 9), _slopes(H)
    prefix = torch.arange(B, dtype=torch.int32, device="cuda")
    for kw in (dict(doc_ids_q=docs, doc_ids_kv=docs), dict(prefix_lens=prefix)):
        got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, softcap=4.0, alibi_slopes=slopes, **kw)
        for b in (0, B // 2 - 1, B // 2, B - 1):
            one = slice(b, b + 1)
            more = dict(dq=docs[one], dk=docs[one]) if "doc_ids_q" in kw else dict(prefix=prefix[one])
            _compare(got[one], Q[one], K[one], V[one], True, 4.0, slopes, fp32_error=2.0 ** -19, **more)
    tfa.device_status()


def test_fp32_values_outside_the_exact_range():
    """Such calls are left to the CUDA cores, to the last bit; the document tables are then those of the other kernel's blocks."""
    Q, K, V = _inputs("fp32", 2, 400, 400, 4, 2, 64, 21)
    docs = _documents(2, 400, 90, 6)
    K[0, 17, 1, 3] = 2.0 ** -110
    args = dict(is_causal=True, softcap=3.0, alibi_slopes=_slopes(4), doc_ids_q=docs, doc_ids_kv=docs)
    got = []
    for form in (0, 1):
        tfa.set_option("fp32_tc", form)
        got.append(tfa.flash_attn_scored_forward(Q, K, V, **args))
        tfa.set_option("fp32_tc", -1)
    assert torch.equal(*got)
    tfa.device_status()


@pytest.mark.parametrize("dtype,B,Sq,Skv,Hq,Hkv,D", [
    ("fp16", 2, 260, 260, 4, 2, 64), ("bf16", 1, 300, 300, 2, 1, 128), ("fp16", 1, 200, 200, 2, 2, 32), ("bf16", 1, 150, 150, 1, 1, 96), ("fp16", 1, 140, 140, 2, 1, 192),
    ("bf16", 1, 140, 140, 2, 1, 256),  # tiles
    ("fp16", 1, 64, 6000, 2, 1, 64), ("bf16", 1, 100, 4000, 2, 1, 256), ("bf16", 1, 40, 6000, 4, 1, 96), ("fp16", 1, 70, 6000, 4, 1, 128),  # key ranges
    ("fp16", 3, 4, 700, 4, 1, 64), ("bf16", 1, 4, 9000, 8, 2, 128), ("bf16", 9, 2, 300, 16, 16, 96), ("fp16", 1, 3, 8000, 1, 1, 256),  # few rows
    ("fp32", 2, 100, 130, 4, 2, 64), ("fp32", 1, 200, 260, 2, 1, 128), ("fp32", 1, 70, 200, 2, 1, 256),
])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_that_a_mask_hides(dtype, B, Sq, Skv, Hq, Hkv, D, bad):
    """V behind a row's own position may be anything: the row is as without it.  Rows that see it are what 0 x NaN and sums make of them."""
    Q, K, V = _inputs(dtype, B, Sq, Skv, Hq, Hkv, D, 30)
    q_start = Skv - Sq
    slopes = _slopes(Hq)
    first = q_start + Sq // 2  # the first key with a bad value
    V2 = V.clone()
    V2[:, first, :, 5] = bad
    V2[:, first + 3:] = -bad
    got = tfa.flash_attn_scored_forward(Q, K, V2, is_causal=True, softcap=3.0, alibi_slopes=slopes, q_start=q_start)
    n = first - q_start  # rows before it
    clean = V.clone()
    clean[:, first:] = 0
    _compare(got[:, :n], Q[:, :n], K, clean, True, 3.0, slopes, q_start=q_start, fp32_error=2.0 ** -19)
    assert not torch.isfinite(got[:, n:, :, 5]).any()
    if n + 3 <= Sq:
        assert torch.isfinite(got[:, n:n + 3, :, 6:]).all()
    tfa.device_status()


@pytest.mark.parametrize("dtype,Sq,Hq,Hkv,D", [("fp16", 1, 4, 1, 64), ("bf16", 3, 8, 4, 128), ("fp16", 200, 2, 2, 64), ("fp32", 150, 2, 1, 64)])
def test_values_far_behind_a_prefix(dtype, Sq, Hq, Hkv, D):
    """With a prefix the decode kernel reads every key, however far behind the rows."""
    B, Skv, q_start = 2, 3000, 500
    Q, K, V = _inputs(dtype, B, Sq, Skv, Hq, Hkv, D, 32)
    prefix = torch.tensor([400, 900], dtype=torch.int32, device="cuda")
    V2, K2 = V.clone(), K.clone()
    V2[:, 1500:] = math.nan
    K2[:, 2000:] = math.inf
    got = tfa.flash_attn_scored_forward(Q, K2, V2, is_causal=True, prefix_lens=prefix, q_start=q_start)
    _compare(got, Q, K, V, True, prefix=prefix, q_start=q_start, fp32_error=2.0 ** -19)
    tfa.device_status()


@pytest.mark.parametrize("dtype,S,D", [("fp16", 300, 64), ("bf16", 500, 128), ("fp32", 300, 64), ("fp16", 200, 256)])
@pytest.mark.parametrize("shuffle", [False, True])
def test_values_of_other_documents_and_padding(dtype, S, D, shuffle):
    Q, K, V = _inputs(dtype, 2, S, S, 2, 1, D, 31)
    docs = _documents(2, S, 40, 7, shuffle=shuffle)
    V2, K2 = V.clone(), K.clone()
    V2[docs < 0] = math.nan
    K2[docs < 0] = math.nan
    V2[docs == 4] = math.inf
    got = tfa.flash_attn_scored_forward(Q, K2, V2, is_causal=False, doc_ids_q=docs, doc_ids_kv=docs)
    want = tfa.flash_attn_scored_forward(Q, K, V, is_causal=False, doc_ids_q=docs, doc_ids_kv=docs)
    assert (docs == 4).any() and not torch.isfinite(got[docs == 4]).any()
    got[docs == 4] = want[docs == 4]
    _compare(got, Q, K, V, False, dq=docs, dk=docs, fp32_error=2.0 ** -19)
    tfa.device_status()


def test_refusals():
    Q, K, V = _inputs("fp16", 1, 8, 8, 2, 1, 64)
    ids = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    f = tfa.flash_attn_scored_forward
    for kw, text in ((dict(softcap=-1.0), "softcap"), (dict(softcap=math.inf), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(q_start=-1), "q_start"),
                     (dict(q_start=1.5), "q_start"), (dict(prefix_lens=ids[:, 0]), "causal"), (dict(doc_ids_q=ids), "together"),
                     (dict(doc_ids_q=ids.long(), doc_ids_kv=ids), "int32"), (dict(doc_ids_q=ids[:, :4], doc_ids_kv=ids), "contiguous|shape"),
                     (dict(alibi_slopes=torch.ones(1, device="cuda")), "shape"), (dict(alibi_slopes=torch.ones(2)), "CUDA"),
                     (dict(alibi_slopes=torch.ones(2, device="cuda", dtype=torch.float64)), "float32")):
        with pytest.raises(RuntimeError, match=text):
            f(Q, K, V, **kw)
    with pytest.raises(RuntimeError, match="forward only"):
        f(Q.requires_grad_(), K, V)
    with torch.no_grad():
        f(Q, K, V)
    with pytest.raises(RuntimeError, match="contiguous"):
        f(Q.detach().transpose(1, 2), K, V)
    empty = f(Q.detach(), K[:, :0], V[:, :0])
    assert (empty == 0).all()
