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
from .api import (_aux, _check, _check_input, _check_no_grad, _current_device, _dtype_code, _fits, _raw_stream, _usable_softcap)

_CACHE_CODE = {torch.int8: 1, torch.float8_e4m3fn: 2}
_BLOCK_TOKENS = (16, 32, 64, 128)
_QUERY_CODE = {torch.float16: 1, torch.bfloat16: 2}


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


def _table_shape(block_table):
    if isinstance(block_table, torch.Tensor):
        shape = block_table.shape
        if len(shape) == 2 and _fits(block_table, torch.int32, shape, block_table.get_device()):
            return shape
    _check_input(block_table, "block_table")
    raise RuntimeError("block_table must be int32 [batch, maxBlocks]")


def _rows_shape(x, name, what):
    """Shape, type and device of packed rows."""
    if isinstance(x, torch.Tensor):
        shape, dtype, device = x.shape, x.dtype, x.get_device()
        if len(shape) == 3 and _fits(x, dtype, shape, device):
            return shape, dtype, device
    _check_input(x, name)
    raise RuntimeError(f"{name} must be 3D {what}")


def _cache_shape(k_cache, v_cache, k_scales, v_scales, device):
    """[numBlocks, numHeadsKV, blockTokens, headDim] and the type code of a cache whose four tensors belong together."""
    if isinstance(k_cache, torch.Tensor):
        shape, dtype = k_cache.shape, k_cache.dtype
        code, tiles = _CACHE_CODE.get(dtype), shape[:2]
        if (code is not None and len(shape) == 4 and shape[2] in _BLOCK_TOKENS and _fits(k_cache, dtype, shape, device)
                and _fits(v_cache, dtype, shape, device) and _fits(k_scales, torch.float32, tiles, device)
                and _fits(v_scales, torch.float32, tiles, device)):
            return shape, code
    _check_cache(k_cache, v_cache, k_scales, v_scales, device)
    raise RuntimeError("unsupported cache")


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
    table_shape = _table_shape(block_table)
    if block_tokens not in _BLOCK_TOKENS:
        raise RuntimeError(f"blocks hold 16, 32, 64 or 128 tokens, got {block_tokens}")
    _check(isinstance(total_new, int) and total_new >= 0, "total_new must be an integer >= 0")
    (batch, width), device = table_shape, block_table.get_device()
    _check(isinstance(free_blocks, torch.Tensor) and free_blocks.dim() == 1, "free_blocks must be an int32 tensor of one dimension")
    capacity = free_blocks.numel()
    lens = _aux(seq_lens, "seq_lens", torch.int32, (batch,), device)
    new = _aux(new_lens, "new_lens", torch.int32, (batch,), device)
    free = _aux(free_blocks, "free_blocks", torch.int32, (capacity,), device)
    have = _aux(num_free, "num_free", torch.int32, (1,), device)
    done = _aux(finished, "finished", torch.bool, (batch,), device) if finished is not None else None
    if _current_device() == device:
        return _run_plan(block_table, lens, new, done, free, have, batch, width, capacity, block_tokens, total_new, device)
    with torch.cuda.device(device):
        return _run_plan(block_table, lens, new, done, free, have, batch, width, capacity, block_tokens, total_new, device)


def _run_plan(block_table, lens, new, done, free, have, batch, width, capacity, block_tokens, total_new, device):
    where = block_table.device
    slots = torch.empty(total_new, dtype=torch.int64, device=where)
    cu = torch.empty(batch + 1, dtype=torch.int32, device=where)
    after = torch.empty(batch, dtype=torch.int32, device=where)
    left = torch.empty(1, dtype=torch.int32, device=where)
    rc = _lib.load().tfa_b200_kv_cache_plan(block_table.data_ptr(), lens, new, done, free, have, slots.data_ptr(), cu.data_ptr(), after.data_ptr(),
                                            left.data_ptr(), batch, width, capacity, block_tokens, total_new, _raw_stream(device))
    if rc != 0:
        _lib.check(rc, "kv_cache_plan")
    return slots, cu, after, left


def kv_cache_store(K, V, k_cache, v_cache, k_scales, v_scales, slots):
    """Writes rows of K and V [total, Hkv, D] (fp16, bf16, fp32) into their slots (int64 [total], -1: nowhere) of the cache, in place.

    The scale of a block and head grows to what its new rows need, max |x| / 127 (int8) or / 448 (e4m3); when it grows, codes that were in the
    block before - in front of the first cell that the call writes - are rounded anew.  Rows of which one goes to a block's first cell begin the
    block, whatever its scale was.  Infinities become the largest code and NaN zero.  The rows of one block follow one another, in any order
    of their cells, and no slot comes twice, as kv_cache_plan gives them.
    """
    shape, dtype, device = _rows_shape(K, "K", "[total, numHeadsKV, headDim]")
    code = _dtype_code(K, "kv_cache_store")
    v = _aux(V, "V", dtype, shape, device)
    cache, kind = _cache_shape(k_cache, v_cache, k_scales, v_scales, device)
    _check(cache[1] == shape[1] and cache[3] == shape[2], "cache and K must have the same heads and head dim")
    _check_no_grad(K, V)
    where = _aux(slots, "slots", torch.int64, (shape[0],), device)
    if _current_device() == device:
        return _run_store(K, v, k_cache, v_cache, k_scales, v_scales, where, code, kind, shape, cache, device)
    with torch.cuda.device(device):
        return _run_store(K, v, k_cache, v_cache, k_scales, v_scales, where, code, kind, shape, cache, device)


def _run_store(K, v, k_cache, v_cache, k_scales, v_scales, where, code, kind, shape, cache, device):
    rc = _lib.load().tfa_b200_kv_cache_store(K.data_ptr(), v, k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), where, code,
                                             kind, shape[0], cache[0], shape[1], shape[2], cache[2], _raw_stream(device))
    if rc != 0:
        _lib.check(rc, "kv_cache_store")


def flash_attn_cache_forward(Q, k_cache, v_cache, k_scales, v_scales, block_table, seq_lens, cu_seqlens_q, max_seqlen_q, max_seqlen_kv,
                             is_causal=True, softcap=0.0, alibi_slopes=None):
    """Attention of packed queries over the paged 8-bit cache.  Q [totalQ, Hq, D] fp16 / bf16; returns O like Q.

    block_table int32 [B, maxBlocks]; seq_lens int32 [B]: tokens of each request with those of its queries, which are its last positions;
    cu_seqlens_q int32 [B + 1]; max_seqlen_q / max_seqlen_kv only size the launch.  is_causal: a query sees keys up to its own position, else
    all of its request's.  softcap and alibi_slopes as in flash_attn_scored_forward.  Rows of no request and rows that see no key are zero.
    """
    shape, dtype, device = _rows_shape(Q, "Q", "[totalQ, numHeadsQ, headDim]")
    code = _QUERY_CODE.get(dtype)
    if code is None:
        raise RuntimeError(f"flash_attn_cache_forward only supports fp16 and bf16, got {dtype}")
    cache, kind = _cache_shape(k_cache, v_cache, k_scales, v_scales, device)
    _check(cache[3] == shape[2], "Head dims must match")
    _check(cache[1] > 0 and shape[1] % cache[1] == 0, "numHeadsQ must be divisible by numHeadsKV (GQA)")
    batch, width = table_shape = _table_shape(block_table)
    table = _aux(block_table, "block_table", torch.int32, table_shape, device)
    lens = _aux(seq_lens, "seq_lens", torch.int32, (batch,), device)
    cu = _aux(cu_seqlens_q, "cu_seqlens_q", torch.int32, (batch + 1,), device)
    slopes = _aux(alibi_slopes, "alibi_slopes", torch.float32, (shape[1],), device) if alibi_slopes is not None else None
    softcap = _usable_softcap(softcap)
    _check_no_grad(Q, alibi_slopes)
    most_q, most_kv = min(int(max_seqlen_q), 2 ** 31 - 1), min(int(max_seqlen_kv), 2 ** 31 - 1)  # (a C int would keep their low bits)
    sizes = (batch, most_q, most_kv, shape[0], cache[0], width, cache[2], shape[1], cache[1], shape[2])
    if _current_device() == device:
        return _run_cache(Q, k_cache, v_cache, k_scales, v_scales, table, lens, cu, code, kind, sizes, is_causal, softcap, slopes, device)
    with torch.cuda.device(device):
        return _run_cache(Q, k_cache, v_cache, k_scales, v_scales, table, lens, cu, code, kind, sizes, is_causal, softcap, slopes, device)


def _run_cache(Q, k_cache, v_cache, k_scales, v_scales, table, lens, cu, code, kind, sizes, is_causal, softcap, slopes, device):
    O = torch.empty_like(Q)
    rc = _lib.load().tfa_b200_fwd_cache(Q.data_ptr(), O.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), table,
                                        lens, cu, code, kind, *sizes, 1 if is_causal else 0, softcap, slopes, _raw_stream(device))
    if rc != 0:
        _lib.check(rc, "flash_attn_cache_forward")
    return O
