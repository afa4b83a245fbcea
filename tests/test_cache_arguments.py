"""The cache's and the scored attention's refusals without a GPU: status codes of the C entries, checks of the Python functions."""
import ctypes

import pytest
import torch

import tinyfa_b200 as tfa
from tinyfa_b200 import _lib


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096)
    test_at = (ctypes.addressof(buf) + 15) & ~15
    yield test_at
    del buf


def test_scored_status_codes(p):
    f = _lib.load().tfa_b200_fwd_scored
    ok = dict(dtype=1, B=1, Sq=16, Skv=16, Hq=2, Hkv=1, D=64, causal=1, q_start=0, cap=0.0, slopes=None, prefix=None, dq=None, dk=None)

    def call(q=p, **kw):
        a = {**ok, **kw}
        return f(q, p, p, p, a["dtype"], a["B"], a["Sq"], a["Skv"], a["Hq"], a["Hkv"], a["D"], a["causal"], a["q_start"], a["cap"], a["slopes"], a["prefix"],
                 a["dq"], a["dk"], None)

    assert call(dtype=9) == 1 and call(D=80) == 2 and call(Hq=3, Hkv=2) == 3 and call(Sq=-1) == 3
    assert call(q=None) == 3 and call(q=p + 4) == 3
    assert call(q_start=-1) == 3 and call(cap=-1.0) == 3 and call(cap=float("inf")) == 3 and call(cap=float("nan")) == 3
    assert call(prefix=p, causal=0) == 3 and "isCausal" in _lib.last_error()
    assert call(dq=p) == 3 and call(dk=p) == 3 and "document" in _lib.last_error()
    assert call(q_start=0x7FFFFFFF) == 6 and call(B=60000, Sq=60000) == 6
    assert call(B=0) == 0 and call(Sq=0) == 0 and call(Skv=0) == 0


def test_plan_status_codes(p):
    f = _lib.load().tfa_b200_kv_cache_plan

    def call(table=p, lens=p, free=p, num=p, slots=p, cu=p, B=1, width=4, cap=4, block=16, total=4):
        return f(table, lens, p, None, free, num, slots, cu, p, p, B, width, cap, block, total, None)

    assert call(block=8) == 3 and call(block=48) == 3 and call(block=256) == 3 and "16, 32, 64 or 128" in _lib.last_error()
    assert call(B=-1) == 3 and call(width=-1) == 3 and call(cap=-1) == 3 and call(total=-1) == 3
    assert call(table=None) == 3 and call(lens=None) == 3 and call(free=None) == 3 and call(num=None) == 3 and call(slots=None) == 3 and call(cu=None) == 3
    assert call(total=1 << 31) == 6 and call(width=1 << 28) == 6


def test_store_status_codes(p):
    f = _lib.load().tfa_b200_kv_cache_store

    def call(k=p, vc=p, scales=p, slots=p, dtype=2, kind=1, total=4, blocks=4, heads=2, D=64, block=16):
        return f(k, p, p, vc, scales, p, slots, dtype, kind, total, blocks, heads, D, block, None)

    assert call(dtype=0) == 1 and call(kind=0) == 1 and call(kind=3) == 1 and call(D=48) == 2
    assert call(block=17) == 3 and call(total=-1) == 3 and call(blocks=-1) == 3 and call(heads=0) == 3
    assert call(k=None) == 3 and call(k=p + 8) == 3 and call(vc=None) == 3 and call(vc=p + 2) == 3 and call(scales=None) == 3 and call(slots=None) == 3
    assert call(total=1 << 31) == 6
    assert call(total=0) == 0 and call(blocks=0) == 0


def test_cache_attention_status_codes(p):
    f = _lib.load().tfa_b200_fwd_cache

    def call(q=p, kc=p, ks=p, table=p, lens=p, cu=p, dtype=2, kind=1, B=1, mq=1, mkv=64, total=1, blocks=4, width=4, block=16, Hq=4, Hkv=2, D=64, cap=0.0):
        return f(q, p, kc, p, ks, p, table, lens, cu, dtype, kind, B, mq, mkv, total, blocks, width, block, Hq, Hkv, D, 1, cap, None, None)

    assert call(dtype=3) == 1 and "fp16 and bf16" in _lib.last_error()
    assert call(dtype=7) == 1 and call(kind=5) == 1 and call(D=40) == 2
    assert call(block=0) == 3 and call(block=100) == 3 and call(block=256) == 3
    assert call(total=-1) == 3 and call(blocks=-2) == 3 and call(width=-2) == 3 and call(cap=-0.5) == 3 and call(cap=float("nan")) == 3
    assert call(Hq=5) == 3 and call(mq=-1) == 3 and call(mkv=-1) == 3 and call(B=-1) == 3
    assert call(q=None) == 3 and call(kc=None) == 3 and call(ks=None) == 3 and call(table=None) == 3 and call(lens=None) == 3 and call(cu=None) == 3
    assert call(q=p + 8) == 3 and call(kc=p + 1) == 3
    assert call(total=1 << 31) == 6 and call(width=1 << 28) == 6 and call(B=70000) == 6
    assert call(total=0) == 0


def test_python_checks_before_any_device_work():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tfa.flash_attn_scored_forward(q, q, q)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tfa.kv_cache_store(q[0], q[0], q, q, q, q, i)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tfa.flash_attn_cache_forward(q[0], q, q, q, q, i, i, i, 1, 1)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        tfa.kv_cache_plan(i[None], i, i, i, i, 16, 0)
    with pytest.raises(RuntimeError, match="must be a torch.Tensor"):
        tfa.kv_cache_plan(None, i, i, i, i, 16, 0)
