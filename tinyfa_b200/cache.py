"""The paged 8-bit K/V cache: its tables, rows written into it, attention over it.

K and V of a layer each are codes [numBlocks, Hkv, blockTokens, D] (torch.int8 or torch.float8_e4m3fn) and one float32 scale per block and
head [numBlocks, Hkv]: value = code * scale.  blockTokens is 16, 32, 64 or 128.  A step of a serving loop is

    slots, cu_seqlens, seq_lens, num_free = kv_cache_plan(block_table, seq_lens, new_lens, free_blocks, num_free, blockTokens, total_new)
    kv_cache_store(K, V, k_cache, v_cache, k_scales, v_scales, slots)                                   # each layer
    O = flash_attn_cache_forward(Q, k_cache, v_cache, k_scales, v_scales, block_table, seq_lens, cu_seqlens, max_new, max_len)

Checks, streams, devices and errors as in api.py; nothing is copied to the host.
"""
import torch

from . import _lib
from .api import _DTYPE_CODE, _check, _check_aux, _check_input, _check_no_grad, _check_softcap, _current_device, _dtype_code, _raw_stream

_CACHE_CODE = {torch.int8: 1, torch.float8_e4m3fn: 2}
_BLOCK_TOKENS = (16, 32, 64, 128)


def _on_device(device, call):
    if _current_device() == device:
        return call()
    with torch.cuda.device(device):
        return call()


def _check_cache(k_cache, v_cache, k_scales, v_scales, device):
    for x, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_scales, "k_scales"), (v_scales, "v_scales")):
        _check_input(x, name)
        _check(x.get_device() == device, f"{name} must be on the device of the other tensors")
    _check(k_cache.dim() == 4, "k_cache must be 4D [numBlocks, numHeadsKV, blockTokens, headDim]")
    _check(k_cache.dtype in _CACHE_CODE, f"caches are int8 or float8_e4m3fn, got {k_cache.dtype}")
    _check(v_cache.dtype == k_cache.dtype and v_cache.shape == k_cache.shape, "k_cache and v_cache must have the same dtype and shape")
    _check(k_cache.shape[2] in _BLOCK_TOKENS, f"blocks hold 16, 32, 64 or 128 tokens, got {k_cache.shape[2]}")
    for x, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
        _check(x.dtype == torch.float32 and x.shape == k_cache.shape[:2], f"{name} must be float32 [numBlocks, numHeadsKV]")


def kv_cache_plan(block_table, seq_lens, new_lens, free_blocks, num_free, block_tokens, total_new, finished=None):
    """Block tables and slot maps from request lengths, on the GPU.

    block_table int32 [B, maxBlocks]; seq_lens, new_lens int32 [B]: tokens that each request holds and gets; free_blocks int32 [F]: stack of
    free block ids with its top at num_free - 1; num_free int32 [1]; total_new: rows of the packed tensors, the sum of new_lens (rows behind
    it get slot -1); finished bool [B]: requests that give their blocks back and start anew from length zero.  block_table and free_blocks
    are updated in place, the other arguments are left as they are.  Returns
      slots int64 [total_new], cu_seqlens int32 [B + 1], seq_lens int32 [B] with the new tokens, num_free int32 [1].
    A request that finds too few free blocks (counting what every request ahead of it asks for), or that would need more than maxBlocks,
    gets none: its length stays and its rows have slot -1.
    """
    _check_input(block_table, "block_table")
    _check(block_table.dtype == torch.int32 and block_table.dim() == 2, "block_table must be int32 [batch, maxBlocks]")
    _check(block_tokens in _BLOCK_TOKENS, f"blocks hold 16, 32, 64 or 128 tokens, got {block_tokens}")
    _check(isinstance(total_new, int) and total_new >= 0, "total_new must be an integer >= 0")
    device, (batch, width) = block_table.get_device(), block_table.shape
    _check_input(free_blocks, "free_blocks")
    _check(seq_lens is not None and new_lens is not None and num_free is not None, "seq_lens, new_lens and num_free must be tensors")
    lens = _check_aux(seq_lens, "seq_lens", torch.int32, (batch,), device)
    new = _check_aux(new_lens, "new_lens", torch.int32, (batch,), device)
    free = _check_aux(free_blocks, "free_blocks", torch.int32, (free_blocks.numel(),), device)
    have = _check_aux(num_free, "num_free", torch.int32, (1,), device)
    done = _check_aux(finished, "finished", torch.bool, (batch,), device)

    def call():
        # one allocation for the four results; slots first, so that they are aligned
        out = torch.empty(2 * total_new + 2 * batch + 2, dtype=torch.int32, device=block_table.device)
        slots, cu, after, left = out[:2 * total_new].view(torch.int64), out[2 * total_new:-batch - 1], out[-batch - 1:-1], out[-1:]
        rc = _lib.load().tfa_b200_kv_cache_plan(block_table.data_ptr(), lens, new, done, free, have, slots.data_ptr(), cu.data_ptr(), after.data_ptr(),
                                                left.data_ptr(), batch, width, free_blocks.numel(), block_tokens, total_new, _raw_stream(device))
        if rc != 0:
            _lib.check(rc, "kv_cache_plan")
        return slots, cu, after, left

    return _on_device(device, call)


def kv_cache_store(K, V, k_cache, v_cache, k_scales, v_scales, slots):
    """Writes rows of K and V [total, Hkv, D] (fp16, bf16, fp32) into their slots (int64 [total], -1: nowhere) of the cache, in place.

    The scale of a block and head grows to what its new rows need, max |x| / 127 (int8) or / 448 (e4m3); when it grows, codes that were in the
    block before are rounded anew.  Rows that begin at a block's first cell begin the block, whatever its scale was.  Infinities become the
    largest code and NaN zero.  The rows of one block follow one another and no slot comes twice, as kv_cache_plan gives them.
    """
    _check_input(K, "K")
    _check_input(V, "V")
    _check(K.dim() == 3 and V.shape == K.shape, "K and V must be 3D [total, numHeadsKV, headDim] of the same shape")
    _check(K.dtype == V.dtype, "K and V must have the same dtype")
    code, device = _dtype_code(K, "kv_cache_store"), K.get_device()
    _check(V.get_device() == device, "K and V must be on the same device")
    _check_cache(k_cache, v_cache, k_scales, v_scales, device)
    _check(k_cache.shape[1] == K.shape[1] and k_cache.shape[3] == K.shape[2], "cache and K must have the same heads and head dim")
    _check(slots is not None, "slots must be a tensor")
    _check_no_grad(K, V)
    where = _check_aux(slots, "slots", torch.int64, (K.shape[0],), device)

    def call():
        rc = _lib.load().tfa_b200_kv_cache_store(K.data_ptr(), V.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(),
                                                 v_scales.data_ptr(), where, code, _CACHE_CODE[k_cache.dtype], K.shape[0], k_cache.shape[0],
                                                 K.shape[1], K.shape[2], k_cache.shape[2], _raw_stream(device))
        if rc != 0:
            _lib.check(rc, "kv_cache_store")

    _on_device(device, call)


def flash_attn_cache_forward(Q, k_cache, v_cache, k_scales, v_scales, block_table, seq_lens, cu_seqlens_q, max_seqlen_q, max_seqlen_kv,
                             is_causal=True, softcap=0.0, alibi_slopes=None):
    """Attention of packed queries over the paged 8-bit cache.  Q [totalQ, Hq, D] fp16 / bf16; returns O like Q.

    block_table int32 [B, maxBlocks]; seq_lens int32 [B]: tokens of each request with those of its queries, which are its last positions;
    cu_seqlens_q int32 [B + 1]; max_seqlen_q / max_seqlen_kv only size the launch.  is_causal: a query sees keys up to its own position, else
    all of its request's.  softcap and alibi_slopes as in flash_attn_scored_forward.  Rows of no request and rows that see no key are zero.
    """
    _check_input(Q, "Q")
    _check(Q.dim() == 3, "Q must be 3D [totalQ, numHeadsQ, headDim]")
    _check(Q.dtype in (torch.float16, torch.bfloat16), f"flash_attn_cache_forward only supports fp16 and bf16, got {Q.dtype}")
    device = Q.get_device()
    _check_cache(k_cache, v_cache, k_scales, v_scales, device)
    total, heads_q, head_dim = Q.shape
    blocks, heads_kv, block_tokens, _ = k_cache.shape
    _check(k_cache.shape[3] == head_dim, "Head dims must match")
    _check(heads_kv > 0 and heads_q % heads_kv == 0, "numHeadsQ must be divisible by numHeadsKV (GQA)")
    _check_input(block_table, "block_table")
    _check(block_table.dim() == 2, "block_table must be int32 [batch, maxBlocks]")
    _check(seq_lens is not None and cu_seqlens_q is not None, "seq_lens and cu_seqlens_q must be tensors")
    batch, width = block_table.shape
    table = _check_aux(block_table, "block_table", torch.int32, (batch, width), device)
    lens = _check_aux(seq_lens, "seq_lens", torch.int32, (batch,), device)
    cu = _check_aux(cu_seqlens_q, "cu_seqlens_q", torch.int32, (batch + 1,), device)
    slopes = _check_aux(alibi_slopes, "alibi_slopes", torch.float32, (heads_q,), device)
    max_q, max_kv, softcap = int(max_seqlen_q), int(max_seqlen_kv), _check_softcap(softcap)
    _check_no_grad(Q, alibi_slopes)

    def call():
        O = torch.empty_like(Q)
        rc = _lib.load().tfa_b200_fwd_cache(Q.data_ptr(), O.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(),
                                            v_scales.data_ptr(), table, lens, cu, _DTYPE_CODE[Q.dtype], _CACHE_CODE[k_cache.dtype], batch, max_q,
                                            max_kv, total, blocks, width, block_tokens, heads_q, heads_kv, head_dim, 1 if is_causal else 0,
                                            softcap, slopes, _raw_stream(device))
        if rc != 0:
            _lib.check(rc, "flash_attn_cache_forward")
        return O

    return _on_device(device, call)
