"""Attention with capped, biased and masked scores, and the paged 8-bit cache, in 64 bits from their definitions; error bounds.

With u the largest relative rounding error of a type (half a step: fp16 2^-11, bf16 2^-8), A = sum p |v| / sum p:
  * weights rounded to a type with u_p are each off by u_p relative: u_p A in the output;
  * a score that is off by e changes its weight by e relative, in numerator and denominator: 2 e A.  Scores are fp32 sums of D products,
    e <= D 2^-24 sum |q k| / sqrt(D); the cap adds c - 2 c / (e^2x + 1) in fp32 (4 roundings of at most c: c 2^-22), the bias one
    rounding of the score it leaves (2^-24 |S|), the exponential 8.6e-5 at most (one value in sixteen is a cubic);
  * a weight that falls below fp16's smallest normal number is rounded to a multiple of its smallest step 2^-24, i.e. off by 2^-25 of the
    row's largest weight (2^-35 where weights are stored 2^10 larger): for n keys n 2^-25 max |v| (`floor`);
  * the output is rounded to its type, after all that: u (|O| + the sum of the above).
"""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attend(q, k, v, see, cap=0.0, slopes=None, distance=None, exp_error=8.6e-5):
    """q [Sq,Hq,D], k and v [Skv,Hkv,D], see [Sq,Skv]; returns O and what it may be off before it is rounded, for weights without rounding,
    and A, all [Sq,Hq,D] in 64 bits."""
    sq, hq, d = q.shape
    group = hq // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    k = torch.where(see.any(0)[:, None, None], k, 0.0)  # what nobody sees says nothing
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(d)
    size = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) / math.sqrt(d)
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * distance
    s = torch.where(see, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    each = torch.where(see[None], d * 2.0 ** -24 * size + 2.0 ** -22 * (cap + s.abs()), 0.0).nan_to_num(posinf=0.0).amax(-1)  # [Hq,Sq]
    seen = torch.where(see.any(0)[:, None, None], v, 0.0)
    o = torch.einsum("hij,jhd->ihd", p, seen)
    a = torch.einsum("hij,jhd->ihd", p, seen.abs())
    return o, (2 * each.T[:, :, None] + exp_error) * a, a


def check(got, o, off, a, u_weights, floor=0.0):
    """got within the bound: off, and roundings of weights and output; denormal outputs to their step."""
    before = off + u_weights * a + floor
    tol = before + U[got.dtype] * (o.abs() + before) + torch.finfo(got.dtype).smallest_normal * 2.0 ** -7
    far = (got.double() - o).abs() - tol
    assert torch.isfinite(got).all()
    assert (far <= 0).all(), f"{(far > 0).sum().item()} of {far.numel()} values, worst {far.max().item():.3g} past the bound"


def visible(sq, skv, causal, q_start=0, prefix=None, doc_q=None, doc_kv=None, device="cuda"):
    i = torch.arange(sq, device=device)[:, None] + q_start
    j = torch.arange(skv, device=device)[None]
    see = torch.ones(sq, skv, dtype=torch.bool, device=device)
    if causal:
        see = j <= i
        if prefix is not None:
            see = see | (j < prefix)
    if doc_q is not None:
        see = see & (doc_q[:, None] == doc_kv[None]) & (doc_q[:, None] >= 0)
    return see, (i - j).abs().double()
