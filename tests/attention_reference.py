"""Attention in 64 bits from its formulas, with bounds of what rounding may do to each output.

The bounds count roundings.  A rounding to a type is off by at most u = finfo.eps / 2 of the value
(bf16 2^-8, fp32 2^-24).  With
    d_s  error of a score in fp32: (D + 8) 2^-24 scale |q||k| for the product, 8 roundings of what is
         added to it and of the exponential's argument, 2^-21 for exp2 and the divisions of tanh
    d    relative error of a probability: 2 d_s (its own score and the row's sum), and as much again
         where the backward rebuilds it from lse, plus (Sk / 32 + 32) 2^-24 for the sum
the outputs obey, with w = u of the storage type where probabilities or score gradients pass through
the tensor cores in it (else w = 0), entry by entry:
    |o'  - o|  <= (d + w) (P|V| + |o|) + u |o|: weights p(1 + e), |e| <= d + w, in the product and in the
         sum behind the quotient give sum p e (v - o), and |v - o| <= |v| + |o|
    |dv' - dv| <= (d + w) P^T|dO| + u |dv|
    |dS' - dS| <= (d + w) |dS| + P (e_dp + e_delta) =: b, e_dp = (D + 8) 2^-24 |dO||V|,
         e_delta = |dO| . bound(o) + (D + 8) 2^-24 |dO| . |o|
         or, where delta is told by the row's own sum of score gradients (exact_delta), which is off by their
         errors: e_delta = d (P.|dP| + |delta| + f) + P.e_dp + w f, f being the e_delta above, which a row's
         share of keys times that sum takes off again, rounded to w
    |dx' - dx| <= scale (c b + 4 d_s (|dS| + b)) =: bx for dx = scale c dS, c = 1 - tanh^2 off by at most
         4 d_s (twice the tanh's error and a rounding): (c + e1)(dS + e2) - c dS = c e2 + e1 dS + e1 e2
    |dq' - dq| <= bx |K| + u |dq|, |dk' - dk| <= bx^T |Q| + u |dk|
    dtable: sums of d |dS| + d P (|dP| + |delta|) + P e_dp, doubled: the rows' common error is taken off.
         With bf16, room for taking it off in proportion to sums of P in fp16 times 2^15 (no kernel needs it
         any more): off by 2^-11 of the sum, or by 2^-40 (half a step of the smallest fp16, 2^-24, over
         2^15), an addition, at most Sk / 128 + 2 of them by each of four threads; and the error taken off
         is at most e_delta + e_dp.
         With exact_delta, or where the keys are shared out over several calls (shares), nothing is taken
         off: sums of 2 (d |dS| + P e_dp) + P e_delta without its term in w, and of (Sq / 4 + 32) 2^-24 |dS|
         for a thread's own additions (a quarter of a key's queries), its warp's and its row's
"""
import math

import torch

F64 = torch.float64


def reference(q, k, v, dout=None, scale=None, cap=0.0, causal=False, kv_lens=None, q_start=None, prefix=None,
              q_docs=None, kv_docs=None, slopes=None, table=None, bucket_of=None, tensor_cores=None, exact_delta=False,
              shares=False):
    """(values, bounds): dicts of o, lse and, with dout, dq, dk, dv, dtable in float64 on the inputs' device."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    dev = q.device
    scale = D ** -0.5 if scale is None else scale
    u = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -24
    w = u if q.dtype == torch.bfloat16 else 0.0
    start = (q_start if q_start is not None else torch.zeros(B, device=dev)).long().clamp(-2 ** 30, 2 ** 30)
    lens = (kv_lens if kv_lens is not None else torch.full((B,), Sk, device=dev)).long().clamp(0, Sk)
    pre = (prefix if prefix is not None else torch.zeros(B, device=dev)).long().clamp(0, Sk)
    j = torch.arange(Sk, device=dev)
    p_at = start[:, None] + torch.arange(Sq, device=dev)[None, :]
    rel = j[None, None, :] - p_at[:, :, None]  # [B, Sq, Sk]
    seen = (j[None, None, :] < lens[:, None, None]).expand(B, Sq, Sk).clone()
    end = lens.clone()
    if causal:
        seen &= (rel <= 0) | (j[None, None, :] < pre[:, None, None])
        end = torch.minimum(lens, torch.maximum((start + Sq).clamp(min=0), pre))
    if q_docs is not None:
        seen &= q_docs[:, :, None] == kv_docs[:, None, :]
    # keys that no query reaches may hold anything
    live = (j[None, :] < end[:, None])[:, :, None, None]
    kd = torch.where(live, k.to(F64), 0.0).repeat_interleave(G, 2).permute(0, 2, 1, 3)
    vd = torch.where(live, v.to(F64), 0.0).repeat_interleave(G, 2).permute(0, 2, 1, 3)
    qd = q.to(F64).permute(0, 2, 1, 3)
    x = qd @ kd.transpose(-1, -2) * scale
    t = torch.tanh(x / cap) if cap else None
    s = cap * t if cap else x.clone()
    moved = s.abs()
    if slopes is not None:
        add = slopes.to(F64)[None, :, None, None] * rel.abs()[:, None].to(F64)
        s, moved = s - add, moved + add.abs()
    if table is not None:
        M = bucket_of.numel() // 2
        bucket = bucket_of.long()[rel.clamp(-M, M) + M].clamp(0, table.shape[1] - 1)  # [B, Sq, Sk]
        entry = torch.where(table < -1e30, -math.inf, table.to(F64))
        add = entry[:, bucket].transpose(0, 1)
        s, moved = s + add, moved + torch.where(add.isinf(), 0.0, add.abs())
    s = torch.where(seen[:, None], s, -math.inf)
    m = s.amax(-1, keepdim=True) if Sk else torch.full(s.shape[:-1] + (1,), -math.inf, dtype=F64, device=dev)
    m = torch.where(m.isinf(), 0.0, m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    P = e / torch.where(total == 0, 1.0, total)
    o = P @ vd
    lse = torch.where(total == 0, -math.inf, m + torch.log(torch.where(total == 0, 1.0, total)))[..., 0]

    size = scale * qd.norm(dim=-1)[..., None] * kd.norm(dim=-1)[..., None, :]
    reach = torch.where(seen[:, None], moved + size, 0.0).amax(-1, keepdim=True) if Sk else torch.zeros_like(m)
    d_s = 2.0 ** -24 * ((D + 8) * (size.amax(-1, keepdim=True) if Sk else 0.0) + 8 * reach) + 2.0 ** -21
    d = 4 * d_s + (Sk / 32 + 32) * 2.0 ** -24
    tiny = 1e-30

    def tokens(y):
        return y.permute(0, 2, 1, 3)

    b_o = (d + w) * (P @ vd.abs() + o.abs()) + u * o.abs()
    values, bounds = dict(o=tokens(o), lse=lse), dict(o=tokens(b_o) + tiny)
    bounds["lse"] = (2 * d_s)[..., 0] + 2.0 ** -23 * torch.where(lse.isinf(), 0.0, lse.abs()) + (Sk / 32 + 32) * 2.0 ** -24
    if dout is None:
        return values, bounds
    g = dout.to(F64).permute(0, 2, 1, 3)
    dP = g @ vd.transpose(-1, -2)
    delta = (P * dP).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    e_dp = (D + 8) * 2.0 ** -24 * (g.abs() @ vd.abs().transpose(-1, -2))
    e_delta = (g.abs() * b_o).sum(-1, keepdim=True) + (D + 8) * 2.0 ** -24 * (g.abs() * o.abs()).sum(-1, keepdim=True)
    from_output = e_delta
    if exact_delta:
        e_delta = d * ((P * dP.abs()).sum(-1, keepdim=True) + delta.abs() + from_output) + (P * e_dp).sum(-1, keepdim=True) \
            + w * from_output
    b_s = (d + w) * dS.abs() + P * (e_dp + e_delta)
    if table is not None:
        n = table.shape[1]
        one = torch.nn.functional.one_hot(bucket, n).to(F64)  # [B, Sq, Sk, n]
        values["dtable"] = torch.einsum("bhij,bijn->hn", dS, one)
        b_t = 2 * (d * dS.abs() + d * P * (dP.abs() + delta.abs()) + P * e_dp)
        bounds["dtable"] = torch.einsum("bhij,bijn->hn", b_t, one) + tiny
        if exact_delta or shares:
            b_t = 2 * (d * dS.abs() + P * e_dp) + P * (e_delta - (w * from_output if exact_delta else 0.0)) + (Sq / 4 + 32) * 2.0 ** -24 * dS.abs()
            bounds["dtable"] = torch.einsum("bhij,bijn->hn", b_t, one) + tiny
        elif w:
            most = from_output + (e_dp.amax(-1, keepdim=True) if Sk else 0.0)
            bounds["dtable"] += (Sk / 128 + 2) * (2.0 ** -11 * torch.einsum("bhij,bijn->hn", P * most, one)
                                                  + 4 * 2.0 ** -40 * most.sum((0, 2, 3))[:, None])
    dcap = (1 - t * t) if cap else torch.ones_like(x)
    dx, b_x = dS * dcap * scale, (b_s * dcap.abs() + 4 * d_s * (dS.abs() + b_s)) * scale

    def shared(y):  # sum over the query heads of a key/value head
        return y.unflatten(1, (Hk, G)).sum(2)

    dq, dk, dv = dx @ kd, shared(dx.transpose(-1, -2) @ qd), shared(P.transpose(-1, -2) @ g)
    values.update(dq=tokens(dq), dk=tokens(dk), dv=tokens(dv))
    grow = 1 + 2.0 ** -10  # second order: a bound on an already rounded factor
    bounds["dq"] = grow * tokens(b_x @ kd.abs() + u * dq.abs()) + 2.0 ** -24 * Sk * tokens(dx.abs() @ kd.abs()) + tiny
    bounds["dk"] = grow * tokens(shared(b_x.transpose(-1, -2) @ qd.abs()) + u * dk.abs()) \
        + 2.0 ** -24 * Sq * tokens(shared(dx.abs().transpose(-1, -2) @ qd.abs())) + tiny
    row = (d + w) * P
    bounds["dv"] = grow * tokens(shared(row.transpose(-1, -2) @ g.abs()) + u * dv.abs()) \
        + 2.0 ** -24 * Sq * tokens(shared(P.transpose(-1, -2) @ g.abs())) + tiny
    return values, bounds


def check(got, values, bounds):
    """got: dict of the same names; every entry inside its bound, infinities equal."""
    for name, want in values.items():
        if got.get(name) is None:
            continue
        a = got[name].to(F64)
        assert a.shape == want.shape, (name, a.shape, want.shape)
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(a), fine), f"{name}: not finite where it should be, or the other way round"
        assert torch.equal(a[~fine], want[~fine]), name
        off = torch.where(fine, (a - torch.where(fine, want, 0.0)).abs(), 0.0)
        ratio = (off / bounds[name].expand_as(want)).max().item() if want.numel() else 0.0
        assert ratio <= 1.0, f"{name}: {ratio:.3g} times its bound"
