"""CTAs with two query tiles whose items differ in what the tiles have to do: items without a second tile, and tiles of which one has more key
blocks than the other.  The two tiles' MMAs are issued by two threads that walk one ring of K/V loads; repeated calls are equal to the
last bit, and the first is the attention of its definition."""
import random

import pytest
import torch

import tinyfa_b200 as tfa
from plain64 import U, attend, check, visible

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _inputs(dtype, B, Sq, Skv, Hq, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(Sq + D)
    return tuple(torch.randn(B, s, h, D, device="cuda", generator=g).to(DT[dtype]) for s, h in ((Sq, Hq), (Skv, Hkv), (Skv, Hkv)))


def _same(call, times):
    want = call()
    for _ in range(times):
        assert torch.equal(call(), want)
    tfa.device_status()
    return want


CASES = [  # dtype, B, Sq, Skv, Hq, Hkv, D: an odd number of tiles, and key blocks that are one, two and three rounds of the ring
    ("fp16", 130, 71, 468, 24, 3, 96), ("bf16", 130, 300, 468, 6, 3, 128), ("fp16", 200, 257, 256, 4, 4, 128), ("bf16", 60, 600, 700, 8, 8, 128),
    ("fp16", 40, 1150, 1024, 4, 2, 96), ("bf16", 300, 129, 129, 4, 1, 128), ("fp16", 130, 224, 1142, 4, 1, 128), ("fp16", 130, 300, 468, 6, 3, 64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("causal", [False, True])
def test_fixed_length(case, causal):
    Q, K, V = _inputs(*case)
    got = _same(lambda: tfa.flash_attn_forward(Q, K, V, causal), 150)
    see, _ = visible(Q.shape[1], K.shape[1], causal)
    for b in range(0, Q.shape[0], 13):
        o, off, a = attend(Q[b].double(), K[b].double(), V[b].double(), see)
        check(got[b], o, off, a, U[Q.dtype], K.shape[1] * 2.0 ** -25 * V[b].abs().max().item() if Q.dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("what", ["cap", "chunk", "prefix", "documents"])
def test_scored(case, what):
    Q, K, V = _inputs(*case)
    B, Sq, Skv, Hq = Q.shape[0], Q.shape[1], K.shape[1], Q.shape[2]
    rng, kw, plain = random.Random(Sq), {}, {}
    if what == "cap":
        kw, plain = dict(softcap=3.0), dict(cap=3.0)
    elif what == "chunk":
        kw = dict(is_causal=True, q_start=max(Skv - Sq, 0))
    elif what == "prefix":
        kw = dict(is_causal=True, prefix_lens=torch.tensor([rng.randint(0, Skv) for _ in range(B)], dtype=torch.int32, device="cuda"))
    else:  # tiles of one item see from one to all key blocks
        ids = lambda n: sorted(rng.randint(0, 6) for _ in range(n))  # noqa: E731
        kw = dict(doc_ids_q=torch.tensor([ids(Sq) for _ in range(B)], dtype=torch.int32, device="cuda"),
                  doc_ids_kv=torch.tensor([ids(Skv) for _ in range(B)], dtype=torch.int32, device="cuda"))
    got = _same(lambda: tfa.flash_attn_scored_forward(Q, K, V, **kw), 100)
    for b in range(0, B, 13):
        prefix, docs = kw.get("prefix_lens"), kw.get("doc_ids_q")
        see, _ = visible(Sq, Skv, kw.get("is_causal", False), kw.get("q_start", 0), None if prefix is None else int(prefix[b]), None if docs is None else docs[b],
                         None if docs is None else kw["doc_ids_kv"][b])
        o, off, a = attend(Q[b].double(), K[b].double(), V[b].double(), see, plain.get("cap", 0.0))
        check(got[b], o, off, a, U[Q.dtype], Skv * 2.0 ** -25 * V[b].abs().max().item() if Q.dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_packed(causal, D):
    rng = random.Random(D)
    lens = [rng.choice([rng.randint(1, 2100), 129, 257, 700]) for _ in range(40)]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    Q = torch.randn(sum(lens), 8, D, device="cuda", generator=g).bfloat16()
    K, V = (torch.randn(sum(lens), 2, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    got = _same(lambda: tfa.flash_attn_varlen_forward(Q, K, V, cu, cu, max(lens), max(lens), causal), 300)
    for b in range(0, 40, 7):
        one = slice(int(cu[b]), int(cu[b + 1]))
        see, _ = visible(lens[b], lens[b], causal)
        o, off, a = attend(Q[one].double(), K[one].double(), V[one].double(), see)
        check(got[one], o, off, a, U[torch.bfloat16])


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 96), ("bf16", 192), ("fp16", 256), ("bf16", 64)])
@pytest.mark.parametrize("Skv", [100, 200, 300])
def test_items_of_few_key_blocks_behind_a_slow_output(dtype, D, Skv):
    """The warps that write a tile's output compute rows again, because a masked value is NaN; meanwhile the softmax of the next items, of one to
    three key blocks each, is done."""
    B, Sq = 700, 256
    Q, K, V = _inputs(dtype, B, Sq, Skv, 2, 1, D)
    V2 = V.clone()
    V2[:, 50:, :, 5] = float("nan")
    got = tfa.flash_attn_scored_forward(Q, K, V2, is_causal=True)
    tfa.device_status()
    see, _ = visible(50, Skv, True)
    for b in range(0, B, 31):
        o, off, a = attend(Q[b, :50].double(), K[b].double(), V[b].double(), see)
        check(got[b, :50], o, off, a, U[Q.dtype], Skv * 2.0 ** -25 * V[b].abs().max().item() if Q.dtype == torch.float16 else 0.0)
        assert not torch.isfinite(got[b, 50:, :, 5]).any() and torch.isfinite(got[b, 50:, :, 6:]).all()


@pytest.mark.parametrize("D", [96, 128, 192, 256])
@pytest.mark.parametrize("Skv", [1, 77, 128, 250])
def test_items_of_one_and_two_key_blocks(D, Skv):
    Q, K, V = _inputs("bf16", 300, 400, Skv, 4, 2, D)
    got = _same(lambda: tfa.flash_attn_forward(Q, K, V), 60)
    see, _ = visible(400, Skv, False)
    for b in range(0, 300, 37):
        o, off, a = attend(Q[b].double(), K[b].double(), V[b].double(), see)
        check(got[b], o, off, a, U[torch.bfloat16])
