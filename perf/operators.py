"""What attention with scores of other kinds and the paged 8-bit K/V cache are timed and compared on.

Every case is one call of a public entry point: flash_attn_scored_forward, kv_cache_plan, kv_cache_store or
flash_attn_cache_forward.  Inputs live on the GPU; queries, keys and values are independent standard normals, as in this
repository's benchmark, and sizes those of its workloads and tests and odd ones between them.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
TINY = 2.0 ** -126  # smallest scale of a block that holds anything but zeros


# ------------------------------------------------------------------------------------------------------------ cases
def _scored(name, dtype, causal, B, Sq, Skv, Hq, Hkv, D, cap=0.0, alibi=False, prefix=0, docs=0, q_start=0, lens_seed=0):
    return {"name": name, "op": "scored", "dtype": dtype, "causal": causal, "B": B, "Sq": Sq, "Skv": Skv, "Hq": Hq, "Hkv": Hkv, "D": D,
            "cap": cap, "alibi": alibi, "prefix": prefix, "docs": docs, "q_start": q_start, "lens_seed": lens_seed}


def _cache(name, dtype, code, B, new_lo, new_hi, lo, hi, Hq, Hkv, D, block, cap=0.0, alibi=False, lens_seed=0):
    return {"name": name, "op": "cache", "dtype": dtype, "code": code, "B": B, "new_lo": new_lo, "new_hi": new_hi, "lo": lo, "hi": hi,
            "Hq": Hq, "Hkv": Hkv, "D": D, "block": block, "cap": cap, "alibi": alibi, "lens_seed": lens_seed}


def _store(name, dtype, code, B, new_lo, new_hi, lo, hi, Hkv, D, block, lens_seed=0):
    return {"name": name, "op": "store", "dtype": dtype, "code": code, "B": B, "new_lo": new_lo, "new_hi": new_hi, "lo": lo, "hi": hi,
            "Hkv": Hkv, "D": D, "block": block, "lens_seed": lens_seed}


def _plan(name, B, new_lo, new_hi, lo, hi, block, done, lens_seed=0):
    return {"name": name, "op": "plan", "B": B, "new_lo": new_lo, "new_hi": new_hi, "lo": lo, "hi": hi, "block": block, "done": done,
            "lens_seed": lens_seed}


def listed():
    return [
        # a prompt batch of a model with capped scores, at the shape this repository's throughput is quoted on, grouped heads: the largest call
        _scored("cap_prefill_bf16", "bf16", True, 2, 4096, 4096, 32, 8, 128, cap=50.0),
        # several documents packed into each row (padding behind the last), distance bias: evaluation of packed text
        _scored("documents_fp16", "fp16", True, 4, 4096, 4096, 16, 16, 64, alibi=True, docs=700, lens_seed=1),
        # encoder-decoder attention of a short batch, odd lengths, capped, no mask: latency
        _scored("cross_cap_fp16", "fp16", False, 3, 333, 517, 12, 12, 96, cap=30.0),
        # full-precision evaluation with a prefix that all tokens see, odd length
        _scored("prefix_fp32", "fp32", True, 1, 999, 999, 8, 2, 64, alibi=True, prefix=300, lens_seed=2),
        # one new token per sequence against long keys, capped and biased: decode without a paged cache
        _scored("token_bf16", "bf16", True, 8, 1, 20011, 32, 8, 128, cap=50.0, alibi=True, q_start=20010),
        # one decode step of a serving batch, ragged caches from one block to 8192 tokens
        _cache("decode_e4m3", "bf16", "e4m3", 64, 1, 1, 1, 8192, 32, 8, 128, 64, lens_seed=3),
        # one request with a long cache, capped scores: the smallest batch, bound by latency and the split over keys
        _cache("decode_one_int8", "fp16", "int8", 1, 1, 1, 32768, 32768, 32, 8, 128, 16, cap=50.0, lens_seed=4),
        # chunks of prompts of different progress against their caches, distance bias
        _cache("chunk_e4m3", "bf16", "e4m3", 4, 200, 512, 1000, 8192, 32, 8, 128, 64, alibi=True, lens_seed=5),
        # prompts written into the cache
        _store("store_prompts", "bf16", "e4m3", 8, 100, 2000, 100, 2500, 8, 128, 64, lens_seed=6),
        # one token per request written into the cache: latency
        _store("store_step", "fp16", "e4m3", 64, 1, 1, 1, 8192, 8, 128, 64, lens_seed=7),
        # the tables of a decode step
        _plan("plan_step", 256, 1, 1, 1, 8192, 64, 0.02, lens_seed=8),
        # the tables of a step that takes in prompts
        _plan("plan_prompts", 64, 1, 2000, 1, 8192, 16, 0.2, lens_seed=9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice([1, 2, 3, 4, 8, 16])
    return hkv * rng.choice([1, 1, 2, 4, 6, 8] if hkv <= 4 else [1, 2, 4]), hkv


def draw(rng):
    """Bounds: below the largest listed case of the same operator, in operations, in bytes and in the plain form's score matrix."""
    while True:
        op = rng.choice(["scored", "scored", "token", "fp32", "decode", "decode", "chunk", "store", "plan"])
        D = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
        dtype, code = rng.choice(["fp16", "bf16"]), rng.choice(["e4m3", "int8"])
        cap = rng.choice([0.0, 20.0, 30.0, 50.0])
        alibi, seed = rng.random() < 0.5, rng.randrange(1 << 30)
        Hq, Hkv = _heads(rng)
        block = rng.choice([16, 32, 64, 128])
        if op in ("scored", "fp32"):
            S = _log_int(rng, 16, 1500 if op == "fp32" else 6000)
            kind = rng.choice(["plain", "prefix", "docs", "cross", "chunk"])
            Skv = _log_int(rng, 16, 6000) if kind == "cross" else S
            causal = kind in ("prefix", "chunk") or (kind != "cross" and rng.random() < 0.7)
            q_start = 0
            if kind == "chunk":
                q_start = _log_int(rng, 1, 4000)
                Skv = q_start + S
            case = _scored("", "fp32" if op == "fp32" else dtype, causal, _log_int(rng, 1, 8), S, Skv, Hq, Hkv, D, cap, alibi,
                           _log_int(rng, 1, S) if kind == "prefix" else 0, _log_int(rng, 10, S) if kind == "docs" else 0, q_start, seed)
        elif op == "token":
            n, L = _log_int(rng, 1, 16), _log_int(rng, 300, 40000)
            case = _scored("", dtype, True, _log_int(rng, 1, 32), n, L + n, Hq, Hkv, D, cap, alibi, q_start=L)
        elif op in ("decode", "chunk"):
            n = 1 if op == "decode" and rng.random() < 0.7 else _log_int(rng, 1, 8) if op == "decode" else _log_int(rng, 10, 600)
            hi = _log_int(rng, 100, 30000)
            case = _cache("", dtype, code, _log_int(rng, 1, 128 if op == "decode" else 8), max(1, n // 3), n, _log_int(rng, 1, hi), hi, Hq, Hkv, D, block, cap,
                          alibi, seed)
        elif op == "store":
            n = rng.choice([1, 1, _log_int(rng, 2, 2000)])
            case = _store("", rng.choice(["fp16", "bf16", "fp32"]), "e4m3", _log_int(rng, 1, 128), max(1, n // 4), n, 1, _log_int(rng, 100, 8000), Hkv, D, block,
                          seed)
        else:
            n = rng.choice([1, _log_int(rng, 2, 2000)])
            case = _plan("", _log_int(rng, 1, 1000), 1, n, 1, _log_int(rng, 100, 8000), block, rng.choice([0.0, 0.1]), seed)
        del case["name"]
        w = work(case)
        if case["op"] == "scored" and (w["flops"] > (2e10 if case["dtype"] == "fp32" else 2.5e11) or w["bytes"] > 6.4e8 or
                                       case["B"] * case["Hq"] * case["Sq"] * case["Skv"] > 1.0e9):
            continue
        if case["op"] == "cache":
            new, lens = _lengths(case)
            if (w["flops"] > 4e10 or w["bytes"] > 5e8 or case["B"] * max(lens) * case["Hkv"] * case["D"] > 5e8 or
                    case["B"] * max(new) * max(lens) * case["Hq"] > 4e8):
                continue
        if case["op"] == "store" and (w["bytes"] > 4e7 or case["B"] * case["hi"] * case["Hkv"] * case["D"] > 4e8):
            continue
        if case["op"] == "plan" and w["bytes"] > 6e5:
            continue
        return case


def _lengths(case):
    """New tokens of every request, and its length with them."""
    rng = random.Random(case["lens_seed"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    lens = [max(n, rng.randint(case["lo"], case["hi"])) for n in new]
    return [0 if d else n for n, d in zip(new, _done(case))], lens


def _done(case):
    """Requests of a plan that have just finished: they give their blocks back and get no new tokens."""
    rng = random.Random(case["lens_seed"] + 1)
    return [case["op"] == "plan" and rng.random() < case["done"] for _ in range(case["B"])]


def _documents(case):
    """Document lengths of every batch entry; the rest of the entry is padding."""
    rng, rows = random.Random(case["lens_seed"]), []
    for _ in range(case["B"]):
        left, row = case["Sq"] - rng.randint(0, case["Sq"] // 16), []
        while left > 0:
            row.append(min(left, 1 + int(rng.expovariate(1.0 / case["docs"]))))
            left -= row[-1]
        rows.append(row)
    return rows


def _prefixes(case):
    rng = random.Random(case["lens_seed"])
    return [rng.randint(1, case["prefix"]) for _ in range(case["B"])]


def _triangle(first, rows, keys):
    """Pairs (i, j) with j <= first + i, i < rows, j < keys."""
    full = min(rows, max(0, keys - first))  # rows that do not see all keys
    return full * first + full * (full + 1) // 2 + (rows - full) * keys


def _visible(case):
    if case["docs"]:
        return sum(n * (n + 1) // 2 if case["causal"] else n * n for row in _documents(case) for n in row)
    if not case["causal"]:
        return case["B"] * case["Sq"] * case["Skv"]
    per = _triangle(case["q_start"], case["Sq"], case["Skv"])
    if not case["prefix"]:
        return case["B"] * per
    return sum(per + p * (p - 1) // 2 for p in _prefixes(case))


def work(case):
    if case["op"] == "plan":
        new, lens = _lengths(case)
        b = case["block"]
        touched = sum(-(-l // b) - (l - n) // b for n, l in zip(new, lens))
        return {"bytes": 8 * sum(new) + 4 * (6 * case["B"] + 2 * touched), "flops": 4 * (sum(new) + case["B"])}
    if case["op"] == "store":
        new, lens = _lengths(case)
        row, b = case["Hkv"] * case["D"], case["block"]
        old = sum((l - n) % b for n, l in zip(new, lens))  # tokens of blocks begun earlier, which a new scale rewrites
        blocks = sum(-(-l // b) - (l - n) // b for n, l in zip(new, lens))
        return {"bytes": 2 * (sum(new) * row * (ESIZE[case["dtype"]] + 1) + 2 * old * row + 8 * blocks * case["Hkv"]) + 8 * sum(new),
                "flops": 2 * 4 * sum(new) * row}
    e, D, Hq, Hkv = ESIZE[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
    if case["op"] == "cache":
        new, lens = _lengths(case)
        pairs = sum(_triangle(l - n, n, l) for n, l in zip(new, lens))
        blocks = sum(-(-l // case["block"]) for l in lens)
        return {"bytes": 2 * e * sum(new) * Hq * D + 2 * Hkv * (sum(lens) * D + 4 * blocks) + 4 * (blocks + 2 * case["B"] + 1),
                "flops": 4 * D * Hq * pairs}
    seen = case["Skv"] if not case["causal"] else min(case["Skv"], case["q_start"] + case["Sq"])
    return {"bytes": e * case["B"] * D * (2 * case["Sq"] * Hq + 2 * seen * Hkv) + (8 * case["B"] * case["Sq"] if case["docs"] else 0),
            "flops": 4 * D * Hq * _visible(case)}


# ----------------------------------------------------------------------------------------------------------- inputs
def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantised(x, code):
    """[blocks, heads, tokens, D] -> codes of the same shape and a scale for each block and head."""
    dtype, top = CODES[code]
    scale = x.abs().amax((2, 3)).div(top)
    x = x / scale[:, :, None, None]
    return (x.round().clamp(-top, top) if code == "int8" else x).to(dtype), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    state = {"case": case}
    if case["op"] == "scored":
        dt, B = DTYPES[case["dtype"]], case["B"]
        state["q"] = normal(B, case["Sq"], case["Hq"], case["D"]).to(dt)
        state["k"] = normal(B, case["Skv"], case["Hkv"], case["D"]).to(dt)
        state["v"] = normal(B, case["Skv"], case["Hkv"], case["D"]).to(dt)
        state["slopes"] = _slopes(case["Hq"]) if case["alibi"] else None
        state["prefix"] = _int32(_prefixes(case)) if case["prefix"] else None
        state["docs"] = None
        if case["docs"]:
            rows = [[d for d, n in enumerate(row) for _ in range(n)] for row in _documents(case)]
            state["docs"] = _int32([row + [-1] * (case["Sq"] - len(row)) for row in rows])
        return state
    new, lens = _lengths(case)
    b, B = case["block"], case["B"]
    if case["op"] == "plan":
        # a pool of blocks in no order; requests hold theirs, `done` of them have just finished
        rng, done = random.Random(seed), _done(case)
        before = [l - n for n, l in zip(new, lens)]
        held = [-(-m // b) for m in before]
        pool = list(range(sum(-(-l // b) for l in lens) + sum(-(-n // b) for n in new)))
        rng.shuffle(pool)
        width, at, table = max(-(-l // b) for l in lens), 0, []
        for h in held:
            table.append(pool[at:at + h] + [-1] * (width - h))
            at += h
        free = pool[at:]
        state.update(table=_int32(table), lens=_int32(before), new=_int32(new), total=sum(new), done=torch.tensor(done, device="cuda"),
                     free=_int32(free + [-1] * at), num_free=_int32([len(free)]))
        return state
    dt = DTYPES[case["dtype"]]
    held = [-(-l // b) for l in lens]
    blocks = sum(held) + 3
    order = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)
    starts = [sum(held[:i]) for i in range(B)]
    cells = torch.arange(max(held), device="cuda")[None]
    where = torch.tensor(starts, device="cuda")[:, None] + cells
    table = torch.where(cells < torch.tensor(held, device="cuda")[:, None], order[where.clamp(max=blocks - 1)], -1).to(torch.int32).contiguous()
    shape = (blocks, case["Hkv"], b, case["D"])
    (kc, ks), (vc, vs) = _quantised(normal(*shape), case["code"]), _quantised(normal(*shape), case["code"])
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    state.update(k_cache=kc, k_scales=ks, v_cache=vc, v_scales=vs, table=table)
    if case["op"] == "cache":
        state.update(q=normal(cu[-1], case["Hq"], case["D"]).to(dt), lens=_int32(lens), cu=_int32(cu), max_new=max(new), max_len=max(lens),
                     slopes=_slopes(case["Hq"]) if case["alibi"] else None)
        return state
    # rows of the packed K and V in the order of the requests, and the cell of the cache that each goes to
    request = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
    place = torch.arange(cu[-1], device="cuda") - torch.tensor(cu[:-1], device="cuda")[request] + torch.tensor(lens, device="cuda")[request] - \
        torch.tensor(new, device="cuda")[request]
    state["slots"] = table[request, place // b].long() * b + place % b
    state["k"] = normal(cu[-1], case["Hkv"], case["D"]).to(dt)
    state["v"] = normal(cu[-1], case["Hkv"], case["D"]).to(dt)
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _weights(s, vis):
    """Softmax over the last axis of the scores that the mask leaves, zero in a row that it leaves empty; as exponentials and their sum."""
    s = torch.where(vis, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    return p, p.sum(-1, keepdim=True)


def _plain_scored(st):
    c = st["case"]
    B, Sq, Skv, Hq, Hkv, D = (c[n] for n in ("B", "Sq", "Skv", "Hq", "Hkv", "D"))
    q = st["q"].float().view(B, Sq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    k, v = st["k"].float().permute(0, 2, 1, 3)[:, :, None], st["v"].float().permute(0, 2, 1, 3)[:, :, None]
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    i = c["q_start"] + torch.arange(Sq, device="cuda")[:, None]
    j = torch.arange(Skv, device="cuda")[None]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hkv, Hq // Hkv, 1, 1) * (i - j).abs().float()
    vis = torch.ones(B, Sq, Skv, dtype=torch.bool, device="cuda")
    if c["causal"]:
        vis = vis & (j <= i)
        if st["prefix"] is not None:
            vis = vis | (j[None] < st["prefix"][:, None, None])
    if st["docs"] is not None:
        vis = vis & (st["docs"][:, :, None] == st["docs"][:, None]) & (st["docs"][:, :, None] >= 0)
    p, total = _weights(s, vis[:, None, None])
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(st["q"].dtype)


def _plain_cache(st):
    c = st["case"]
    B, Hq, Hkv, D = (c[n] for n in ("B", "Hq", "Hkv", "D"))
    table = st["table"].long().clamp(min=0)
    read = lambda codes, scales: (codes.view(torch.uint8)[table].view(codes.dtype).float() * scales[table][..., None, None]).transpose(1, 2).reshape(  # noqa: E731
        B, Hkv, 1, -1, D)
    k, v = read(st["k_cache"], st["k_scales"]), read(st["v_cache"], st["v_scales"])
    cu, lens, rows = st["cu"].long(), st["lens"].long(), st["q"].shape[0]
    new = cu[1:] - cu[:-1]
    at = cu[:-1, None] + torch.arange(st["max_new"], device="cuda")[None]
    q = st["q"][at.clamp(max=rows - 1)].float().view(B, -1, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    i = (lens - new)[:, None, None] + torch.arange(st["max_new"], device="cuda")[None, :, None]
    j = torch.arange(k.shape[-2], device="cuda")[None, None]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hkv, Hq // Hkv, 1, 1) * (i - j).abs().float()[:, None, None]
    p, total = _weights(s, ((j <= i) & (j < lens[:, None, None]))[:, None, None])
    o = torch.matmul(p, torch.where((j < lens[:, None, None]).transpose(-1, -2)[:, None, None], v, 0.0)) / torch.where(total > 0, total, 1.0)
    request = torch.bucketize(torch.arange(rows, device="cuda"), cu[1:], right=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, -1, Hq, D)
    return o[request, torch.arange(rows, device="cuda") - cu[request]].to(st["q"].dtype)


def _plain_store(st, x, codes, scales):
    """The blocks that get rows: the scale grows to what the new rows need, and codes from before are rounded anew."""
    b, (dtype, top) = st["case"]["block"], CODES[st["case"]["code"]]
    block, cell = st["slots"] // b, st["slots"] % b
    ids, at = torch.unique(block, return_inverse=True)
    raw, x = codes.view(torch.uint8), x.float()
    need = x.abs().amax(-1) / top
    need = torch.where(need > 0, need.clamp(min=TINY), 0.0)
    first = torch.full_like(ids, b).scatter_reduce(0, at, cell, "amin")
    old = torch.where((first == 0)[:, None], 0.0, scales[ids])
    scale = old.scatter_reduce(0, at[:, None].expand_as(need), need, "amax")
    some = torch.where(scale > 0, scale, 1.0)
    to_codes = lambda y: (y.round().clamp(-top, top) if dtype == torch.int8 else y.clamp(-top, top)).to(dtype)  # noqa: E731
    held = raw[ids].view(dtype).float()
    again = (torch.arange(b, device="cuda") < first[:, None])[:, None, :, None] & (scale != old)[..., None, None]
    raw[ids] = to_codes(torch.where(again, held * old[..., None, None] / some[..., None, None], held)).view(torch.uint8)
    raw[block, :, cell] = to_codes(x / some[at][..., None]).view(torch.uint8)
    scales[ids] = scale


def _plain_plan(st):
    c = st["case"]
    b, (B, width) = c["block"], st["table"].shape
    lens, done, room = st["lens"].long(), st["done"], st["free"].shape[0]
    cells = torch.arange(width, device="cuda")[None]
    # blocks of finished requests go on top of the stack, in the order of the requests
    held = -(-lens // b)
    back = torch.where(done, held, 0)
    at = st["num_free"].long() + back.cumsum(0) - back
    free = torch.cat([st["free"], st["free"].new_zeros(1)])
    put = torch.where(done[:, None] & (cells < held[:, None]), at[:, None] + cells, room)
    free = free.scatter(0, put.reshape(-1), st["table"].reshape(-1))[:room]
    have = st["num_free"].long() + back.sum()
    lens = torch.where(done, 0, lens)
    # each request takes its new blocks from the top; one that finds too few keeps its length
    held, after = -(-lens // b), lens + st["new"].long()
    need = -(-after // b) - held
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= have)
    after = torch.where(served, after, lens)
    pick = have[:, None] - 1 - (upto - need)[:, None] - (cells - held[:, None])
    fresh = served[:, None] & (cells >= held[:, None]) & (cells < (held + need)[:, None])
    table = torch.where(fresh, free[pick.clamp(0, room - 1)], st["table"])
    left = have - torch.where(served, need, 0).sum()
    cu = torch.cat([lens.new_zeros(1), st["new"].long().cumsum(0)])
    rows = torch.arange(st["total"], device="cuda")
    request = torch.bucketize(rows, cu[1:], right=True)
    place = lens[request] + rows - cu[request]
    slots = torch.where(served[request], table[request, (place // b).clamp(max=width - 1)].long() * b + place % b, -1)
    st["table"].copy_(table)
    st["free"].copy_(free)
    return slots, cu.int(), after.int(), left.int().view(1)


def run(state):
    c = state["case"]
    if own:
        import tinyfa_b200 as tfa
    if c["op"] == "scored":
        if own:
            return tfa.flash_attn_scored_forward(state["q"], state["k"], state["v"], is_causal=c["causal"], softcap=c["cap"], alibi_slopes=state["slopes"],
                                                 prefix_lens=state["prefix"], doc_ids_q=state["docs"], doc_ids_kv=state["docs"], q_start=c["q_start"])
        return _plain_scored(state)
    if c["op"] == "cache":
        if own:
            return tfa.flash_attn_cache_forward(state["q"], state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"], state["table"],
                                                state["lens"], state["cu"], state["max_new"], state["max_len"], softcap=c["cap"],
                                                alibi_slopes=state["slopes"])
        return _plain_cache(state)
    if c["op"] == "store":
        if own:
            tfa.kv_cache_store(state["k"], state["v"], state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"], state["slots"])
        else:
            _plain_store(state, state["k"], state["k_cache"], state["k_scales"])
            _plain_store(state, state["v"], state["v_cache"], state["v_scales"])
        return state["k_cache"], state["v_cache"], state["k_scales"], state["v_scales"]
    if own:
        slots, cu, lens, left = tfa.kv_cache_plan(state["table"], state["lens"], state["new"], state["free"], state["num_free"], c["block"], state["total"],
                                                  finished=state["done"])
    else:
        slots, cu, lens, left = _plain_plan(state)
    return slots, cu, lens, left, state["table"], state["free"]


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _attend(q, k, v, see, cap, slope, distance):
    """One head: rows of q against the keys that each may see."""
    s = (q @ k.T) / math.sqrt(q.shape[1])
    if cap:
        s = cap * torch.tanh(s / cap)
    s = s - slope * distance
    s[~see] = -math.inf
    some = see.any(1)
    o = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    o[some] = torch.softmax(s[some], 1) @ v
    return o


def exact(case, seed):
    if case["op"] == "plan":
        return None
    st = prepare(case, seed)
    if case["op"] == "store":
        b, top, out = case["block"], CODES[case["code"]][1], []
        new, lens = _lengths(case)
        for x, codes, scales in ((st["k"], st["k_cache"], st["k_scales"]), (st["v"], st["v_cache"], st["v_scales"])):
            x, codes, scales, row = x.double(), codes.double(), scales.double(), 0
            table = st["table"].tolist()
            for r in range(case["B"]):
                pos, end = lens[r] - new[r], lens[r]
                while pos < end:
                    first, n, blk = pos % b, min(end, (pos // b + 1) * b) - pos, table[r][pos // b]
                    part = x[row:row + n].transpose(0, 1)
                    before = scales[blk].clone() if first else torch.zeros_like(scales[blk])
                    s = torch.maximum(before, part.abs().amax((1, 2)) / top)
                    codes[blk, :, :first] = (codes[blk, :, :first] * (before / s)[:, None, None]).to(CODES[case["code"]][0]).double()
                    codes[blk, :, first:first + n] = (part / s[:, None, None]).to(CODES[case["code"]][0]).double()
                    scales[blk] = s
                    row, pos = row + n, pos + n
            out.append((codes, scales))
        return out[0][0], out[1][0], out[0][1], out[1][1]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    slope = [2.0 ** (-8.0 * (h + 1) / Hq) if case["alibi"] else 0.0 for h in range(Hq)]
    if case["op"] == "cache":
        (new, lens), row, o = _lengths(case), 0, torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        if sum(n * l for n, l in zip(new, lens)) * Hq > 3e9 or case["B"] * Hq > 8192:
            return None
        for r in range(case["B"]):
            n, length = new[r], lens[r]
            ids = st["table"][r, :-(-length // case["block"])].long()
            k, v = ((st[x + "_cache"].view(torch.uint8)[ids].view(st[x + "_cache"].dtype).double() * st[x + "_scales"][ids].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :length]
                    for x in "kv")
            i = torch.arange(length - n, length, device="cuda", dtype=torch.float64)[:, None]
            j = torch.arange(length, device="cuda", dtype=torch.float64)[None]
            for h in range(Hq):
                kv = h // (Hq // Hkv)
                o[row:row + n, h] = _attend(st["q"][row:row + n, h].double(), k[kv], v[kv], j <= i, case["cap"], slope[h], (i - j).abs())
            row += n
        return o
    o = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    if case["B"] * Hq > 4096:
        return None
    i = torch.arange(case["q_start"], case["q_start"] + case["Sq"], device="cuda", dtype=torch.float64)[:, None]
    j = torch.arange(case["Skv"], device="cuda", dtype=torch.float64)[None]
    for r in range(case["B"]):
        see = torch.ones(case["Sq"], case["Skv"], dtype=torch.bool, device="cuda")
        if case["causal"]:
            see = j <= i
            if case["prefix"]:
                see = see | (j < _prefixes(case)[r])
        if case["docs"]:
            ids = st["docs"][r]
            see = see & (ids[:, None] == ids[None, :]) & (ids[:, None] != -1)
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            o[r, :, h] = _attend(st["q"][r, :, h].double(), st["k"][r, :, kv].double(), st["v"][r, :, kv].double(), see, case["cap"], slope[h], (i - j).abs())
    return o
