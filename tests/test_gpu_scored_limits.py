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


def test_prefixes_at_the_ends_of_their_type(call):
    dtype, Sq, Skv, Hq, Hkv, D = call
    values = [LARGEST, LARGEST - 62, LARGEST - 63, SMALLEST, SMALLEST + 1, -1]
    Q, K, V = _inputs(dtype, len(values), Sq, Skv, Hq, Hkv, D, 1)
    prefix = torch.tensor(values, dtype=torch.int32, device="cuda")
    for slopes in (None, _slopes(Hq)):
        got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=True, prefix_lens=prefix, alibi_slopes=slopes)
        _compare(got, Q, K, V, True, slopes=slopes, prefix=prefix, fp32_error=2.0 ** -19)
    tfa.device_status()


def test_lowest_prefix_and_values_that_the_mask_hides(call):
    """A row that is computed again from what it sees: no key of a prefix below zero."""
    dtype, Sq, Skv, Hq, Hkv, D = call
    Q, K, V = _inputs(dtype, 2, Sq, Skv, Hq, Hkv, D, 2)
    prefix = torch.tensor([SMALLEST, LARGEST], dtype=torch.int32, device="cuda")
    V2 = V.clone()
    first = Sq // 2
    V2[0, first:] = math.nan
    got = tfa.flash_attn_scored_forward(Q, K, V2, is_causal=True, prefix_lens=prefix)
    _compare(got[:1, :first], Q[:1, :first], K[:1], V[:1], True, prefix=prefix[:1], fp32_error=2.0 ** -19)
    _compare(got[1:], Q[1:], K[1:], V[1:], True, prefix=prefix[1:], fp32_error=2.0 ** -19)
    tfa.device_status()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,S,Hq,Hkv,D,fp32_tc", [("fp16", 300, 4, 2, 64, -1), ("bf16", 200, 2, 1, 128, -1), ("bf16", 140, 2, 1, 256, -1), ("fp32", 200, 2, 1, 64, 0),
                                                       ("fp32", 200, 2, 1, 64, 1), ("fp32", 200, 1, 1, 256, 1)])
def test_largest_document_id_beside_padding(dtype, S, Hq, Hkv, D, fp32_tc, causal):
    """Padding belongs to no document, to the one with the largest id as little as to another."""
    Q, K, V = _inputs(dtype, 3, S, S, Hq, Hkv, D, 3)
    docs = torch.full((3, S), -1, dtype=torch.int32, device="cuda")
    docs[0, : S // 2], docs[1, : S // 3], docs[1, S // 3: S // 2] = LARGEST, LARGEST - 1, LARGEST
    docs[2, : S // 2], docs[2, S // 2 + 9:] = LARGEST, SMALLEST
    tfa.set_option("fp32_tc", fp32_tc)
    try:
        got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=causal, doc_ids_q=docs, doc_ids_kv=docs)
    finally:
        tfa.set_option("fp32_tc", -1)
    _compare(got, Q, K, V, causal, dq=docs, dk=docs, fp32_error=2.0 ** -19)
    assert (got[docs < 0] == 0).all()
    tfa.device_status()


@pytest.mark.parametrize("q_start", [5000, 2 ** 24 + 3, 2 ** 30 + 1])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_distances_from_far_positions(call, q_start, causal, cap):
    """All keys lie to the left of every row: |p - j| is (p - Skv + 1) + (Skv - 1 - j), and what all scores of a row share is nothing to its weights.
    So the rows are those of position Skv - 1 with every key visible, in 64 bits too, and distances are as exact as there."""
    dtype, Sq, Skv, Hq, Hkv, D = call
    Q, K, V = _inputs(dtype, 2, Sq, Skv, Hq, Hkv, D, 4)
    slopes = _slopes(Hq)
    got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=causal, softcap=cap, alibi_slopes=slopes, q_start=q_start)
    see = torch.ones(Sq, Skv, dtype=torch.bool, device="cuda")
    distance = (Skv - 1 - torch.arange(Skv, device="cuda", dtype=torch.float64)).expand(Sq, Skv)
    for b in range(2):
        o, off, a = attend(Q[b].double(), K[b].double(), V[b].double(), see, cap, slopes, distance, 2.0 ** -19 if dtype == "fp32" else 8.6e-5)
        check(got[b], o, off, a, U[Q.dtype], Skv * 2.0 ** -25 * V[b].abs().max().item() if dtype == "fp16" else 0.0)
    tfa.device_status()


def test_positions_that_a_c_int_does_not_hold():
    Q, K, V = _inputs("fp16", 1, 8, 20, 2, 1, 64, 5)
    f = tfa.flash_attn_scored_forward
    for q_start in (2 ** 31, 2 ** 32 + 5, 2 ** 64 + 3):
        with pytest.raises(RuntimeError, match="q_start"):
            f(Q, K, V, is_causal=True, q_start=q_start)


def test_caps_below_and_above_what_fp32_holds(call):
    """A cap of next to nothing leaves all scores equal, one far above them leaves them as they are."""
    dtype, Sq, Skv, Hq, Hkv, D = call
    Q, K, V = _inputs(dtype, 2, Sq, Skv, Hq, Hkv, D, 6)
    got = tfa.flash_attn_scored_forward(Q, K, V, softcap=1e-60)
    _compare(got, Q * 0, K, V, False, fp32_error=2.0 ** -19)
    got = tfa.flash_attn_scored_forward(Q, K, V, softcap=1e60)
    _compare(got, Q, K, V, False, fp32_error=2.0 ** -19)


@pytest.mark.parametrize("cap,factor", [(30.0, 3.0), (30.0, 12.0), (5.0, 2.0)])
def test_scores_on_both_sides_of_half_a_cap(call, cap, factor):
    """Scores of factor^2 standard normals: some below half the cap, where the tanh is a polynomial, some far above, in the same blocks."""
    dtype, Sq, Skv, Hq, Hkv, D = call
    Q, K, V = _inputs(dtype, 1, Sq, Skv, Hq, Hkv, D, 7)
    Q, K = Q * factor, K * factor
    for causal, q_start in ((False, 0), (True, Skv - Sq)):
        got = tfa.flash_attn_scored_forward(Q, K, V, is_causal=causal, softcap=cap, q_start=q_start)
        _compare(got, Q, K, V, causal, cap, q_start=q_start, fp32_error=2.0 ** -19)
    # Q in a block of small scores only, and in one of large ones only
    Q[:, : Sq // 2] /= 64
    got = tfa.flash_attn_scored_forward(Q, K, V, softcap=cap, alibi_slopes=_slopes(Hq))
    _compare(got, Q, K, V, False, cap, _slopes(Hq), fp32_error=2.0 ** -19)
    tfa.device_status()


def test_tangents_are_refused():
    """Forward-mode gradients are not dropped either."""
    import torch.autograd.forward_ad as fwd

    Q, K, V = _inputs("fp16", 1, 8, 8, 2, 1, 64, 8)
    with fwd.dual_level():
        dual = fwd.make_dual(Q, torch.ones_like(Q))
        with pytest.raises(RuntimeError, match="forward only"):
            tfa.flash_attn_scored_forward(dual, K, V)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward only"):
            tfa.flash_attn_scored_forward(Q, K, fwd.make_dual(V, torch.ones_like(V)))
        want = tfa.flash_attn_scored_forward(Q, K, V)
        assert torch.equal(tfa.flash_attn_scored_forward(fwd.unpack_dual(dual).primal, K, V), want)


def test_rows_that_take_long_to_compute_again():
    """A value that the mask hides from rows with very many keys: the other warps wait for as long as the rows take, which is more than a
    wait without any progress may last."""
    Sq, Skv, D = 40000, 6_000_000, 32
    g = torch.Generator(device="cuda").manual_seed(9)
    Q, K, V = (torch.randn(1, n, 1, D, device="cuda", generator=g).bfloat16() for n in (Sq, Skv, Skv))
    V += 1
    q_start = Skv - Sq
    bad = q_start + 20 * 128 + 100  # hidden from the hundred rows before it in its block
    V2 = V.clone()
    V2[0, bad, 0, 5] = math.nan
    got = tfa.flash_attn_scored_forward(Q, K, V2, is_causal=True, softcap=2.0, q_start=q_start)
    tfa.device_status()
    n = bad - q_start
    assert torch.isfinite(got[:, :n]).all() and not torch.isfinite(got[:, n:, :, 5]).any()
    for r in (0, n - 100, n - 50, n - 1):
        i = q_start + r
        see, dist = visible(1, i + 1, True, i)
        o, off, a = attend(Q[0, r:r + 1].double(), K[0, :i + 1].double(), V[0, :i + 1].double(), see, 2.0, None, dist)
        check(got[0, r:r + 1], o, off, a, U[torch.bfloat16])
