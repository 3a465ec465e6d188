"""The attention operators as they are measured: cases, inputs, plain forms and 64-bit results.

Four kinds of case.  "forward" is one attention call over whole sequences, "train" a forward and a
backward pass, "step" one new token per sequence against a cache, "bias" the bucketed relative
position bias added to scores that a program holds as a matrix, with the gradient of its table.

Scores of query i (at position p = start + i) and key j:
    s = scale * <q_i, k_j>;  cap: s = cap * tanh(s / cap);  slope: s -= slope_h * |p - j|;
    buckets: s += table[h, bucket(j - p)]
and j is visible when j < kv_len, (not causal, or j <= p, or j < prefix), and the documents of i and
j are the same.
"""
import math
import random

import torch

own = False


def listed():
    """The real work these stand for, smallest calls first."""
    return [
        # the character model of this repository: 32 sequences of 64 characters, width 64
        dict(name="forward_char", kind="forward", dtype="fp32", batch=32, q_len=64, kv_len=64, heads=4, kv_heads=4, dim=16,
             causal=True, slopes=True),
        # evaluating a mid-sized fp32 model on packed documents, lengths that fit no tile
        dict(name="forward_fp32_docs", kind="forward", dtype="fp32", batch=2, q_len=1000, kv_len=1000, heads=16, kv_heads=16,
             dim=64, causal=True, docs=300, cap=30.0),
        # an encoder-decoder prompt: the prefix is seen by all, odd length, distance bias
        dict(name="forward_prefix_odd", kind="forward", dtype="bf16", batch=3, q_len=1531, kv_len=1531, heads=16, kv_heads=16,
             dim=64, causal=True, prefix=True, slopes=True),
        # prompts of width 4096 (32 heads of 128, 8 shared key/value heads), packed documents, capped scores
        dict(name="forward_docs_8192", kind="forward", dtype="bf16", batch=1, q_len=8192, kv_len=8192, heads=32, kv_heads=8,
             dim=128, causal=True, docs=2500, cap=50.0),
        # one training step of the character model's attention with a learned position bias
        dict(name="train_char", kind="train", dtype="fp32", batch=32, q_len=64, kv_len=64, heads=4, kv_heads=4, dim=16,
             causal=True, buckets=16, max_distance=64),
        # an fp32 model with an odd length and a head width that is no power of two
        dict(name="train_fp32_odd", kind="train", dtype="fp32", batch=2, q_len=777, kv_len=777, heads=8, kv_heads=4, dim=80,
             causal=True, prefix=True, slopes=True),
        # an encoder over padded sequences with the usual 32 buckets, both directions
        dict(name="train_buckets", kind="train", dtype="bf16", batch=4, q_len=2048, kv_len=2048, heads=16, kv_heads=16, dim=64,
             ragged=True, buckets=32, max_distance=128, both=True),
        # pre-training at width 4096 and 4096 tokens, capped scores, shared key/value heads
        dict(name="train_cap_4096", kind="train", dtype="bf16", batch=1, q_len=4096, kv_len=4096, heads=32, kv_heads=8, dim=128,
             causal=True, cap=50.0),
        # answering 64 users at once from caches of different lengths
        dict(name="step_batch", kind="step", dtype="bf16", batch=64, q_len=1, kv_len=8192, heads=32, kv_heads=8, dim=128,
             causal=True, ragged=True, slopes=True),
        # one user, one long cache
        dict(name="step_long", kind="step", dtype="bf16", batch=1, q_len=1, kv_len=65536, heads=32, kv_heads=8, dim=128,
             causal=True, cap=30.0),
        # scores held as a matrix, fp32, as the unfused path of this repository has them
        dict(name="bias_fp32", kind="bias", dtype="fp32", batch=2, q_len=2048, kv_len=2048, heads=16, kv_heads=16, dim=1,
             buckets=32, max_distance=128, both=True),
        # the same in bf16, cross lengths that fit no tile
        dict(name="bias_bf16_odd", kind="bias", dtype="bf16", batch=3, q_len=515, kv_len=1027, heads=12, kv_heads=12, dim=1,
             buckets=32, max_distance=100),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["forward", "forward", "train", "train", "step", "step", "bias"])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "bias":
        case.update(batch=rng.randint(1, 4), heads=rng.choice([4, 8, 12, 16]), q_len=_log_int(rng, 32, 2048),
                    kv_len=_log_int(rng, 32, 2048), dim=1)
        case["kv_heads"] = case["heads"]
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        case.update(kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 1, 2, 4, 8]))
        case["dim"] = rng.choice([16, 32, 64, 64, 80, 128, 128] if case["dtype"] == "bf16" else [16, 20, 32, 64, 80, 128])
    if kind == "step":
        case.update(batch=_log_int(rng, 1, 64), q_len=1, kv_len=_log_int(rng, 16, 32768), causal=True)
        while case["batch"] * case["kv_len"] * case["kv_heads"] * case["dim"] > 2 ** 28:
            case["kv_len"] = case["kv_len"] // 2 + 1
        case["ragged"] = rng.random() < 0.5
    elif kind in ("forward", "train"):
        case.update(batch=_log_int(rng, 1, 8), kv_len=_log_int(rng, 16, 4096), causal=rng.random() < 0.6)
        limit = 6e9 if case["dtype"] == "bf16" else 1.5e9
        while case["batch"] * case["heads"] * case["dim"] * case["kv_len"] ** 2 > limit:
            case["kv_len"] = case["kv_len"] // 2 + 1
        case["q_len"] = case["kv_len"]
        shape = rng.choice(["plain", "docs", "prefix", "ragged"])
        if shape == "docs":
            case["docs"] = _log_int(rng, 16, 2048)
        elif shape == "prefix" and case["causal"]:
            case["prefix"] = True
        elif shape == "ragged":
            case["ragged"] = True
    change = "buckets" if kind == "bias" else rng.choice(["none", "cap", "slopes", "buckets", "both"])
    if change in ("cap", "both") and kind != "bias":
        case["cap"] = rng.choice([20.0, 30.0, 50.0])
    if change == "slopes":
        case["slopes"] = True
    if change in ("buckets", "both"):
        case["both"] = not case.get("causal", False) and rng.random() < 0.7
        case["buckets"] = rng.choice([8, 16, 32])
        case["max_distance"] = rng.choice([32, 64, 100, 128])
    return case


# ---- what a case holds besides its tensors: the same for every seed ----------------------------
def _kv_lens(case):
    """Valid keys of every sequence of a padded batch, at least one."""
    rng = random.Random(case["batch"] * 7919 + case["kv_len"])
    return [rng.randint((case["kv_len"] + 1) // 2, case["kv_len"]) for _ in range(case["batch"])]


def _prefixes(case):
    rng = random.Random(case["batch"] * 104729 + case["kv_len"])
    return [rng.randint(0, case["kv_len"] // 2) for _ in range(case["batch"])]


def _documents(case):
    """Document numbers of the positions, ascending, lengths around the mean that the case gives."""
    rng = random.Random(case["docs"] * 15485863 + case["kv_len"])
    rows = []
    for b in range(case["batch"]):
        row, number = [], 0
        while len(row) < case["kv_len"]:
            row += [number] * rng.randint(max(1, case["docs"] // 2), case["docs"] * 3 // 2)
            number += 1
        rows.append(row[:case["kv_len"]])
    return rows


def _starts(case):
    """Position of the first query of every sequence."""
    if case["kind"] != "step":
        return [0] * case["batch"]
    lens = _kv_lens(case) if case.get("ragged") else [case["kv_len"]] * case["batch"]
    return [n - case["q_len"] for n in lens]


def _bucket_of(case):
    """bucket of j - p for j - p = -max_distance .. max_distance: exact up to half of the buckets of a direction, then
    logarithmic; a border that falls on a whole distance belongs to the upper bucket (hence the comparison of integers)."""
    n, top = case["buckets"], case["max_distance"]
    each = n // 2 if case.get("both") else n
    exact_up_to = each // 2
    wide = each - exact_up_to

    def of(distance):
        if distance < exact_up_to:
            return distance
        k = 0
        while k + 1 < wide and distance ** wide * exact_up_to ** (k + 1) >= top ** (k + 1) * exact_up_to ** wide:
            k += 1
        return exact_up_to + k

    if case.get("both"):
        return [of(-r) if r <= 0 else each + of(r) for r in range(-top, top + 1)]
    return [of(max(-r, 0)) for r in range(-top, top + 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    B, Sq, Sk, H, Hk, D = (case[x] for x in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(to)

    ints = dict(dtype=torch.int32, device="cuda")
    st = dict(case=case, scale=1.0 / math.sqrt(D), cap=case.get("cap", 0.0), causal=case.get("causal", False),
              kv_lens=None, q_start=None, prefix=None, docs=None, slopes=None, table=None, bucket_of=None)
    if case.get("buckets"):
        st["table"] = normal(H, case["buckets"], std=0.5, to=torch.float32)
        st["bucket_of"] = torch.tensor(_bucket_of(case), **ints)
    if case["kind"] == "bias":
        st["scores"] = normal(B, H, Sq, Sk)
        st["dscores"] = normal(B, H, Sq, Sk, std=0.1)
        return st
    if case["kind"] == "step":
        st["q"] = normal(B, Sq, H, D, std=1.5)
        st["k"], st["v"] = normal(B, Sk, Hk, D), normal(B, Sk, Hk, D)
    else:  # one projection makes queries, keys and values side by side
        qkv = normal(B, Sq, H + 2 * Hk, D)
        st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    if case["kind"] == "train":
        st["dout"] = normal(B, Sq, H, D)
    if case.get("ragged"):
        st["kv_lens"] = torch.tensor(_kv_lens(case), **ints)
        if case["kind"] == "train":  # no loss is taken on padding
            pad = torch.arange(Sq, device="cuda")[None, :] >= st["kv_lens"][:, None]
            st["dout"].masked_fill_(pad[:, :, None, None], 0.0)
    if case["kind"] == "step":
        st["q_start"] = torch.tensor(_starts(case), **ints)
    if case.get("prefix"):
        st["prefix"] = torch.tensor(_prefixes(case), **ints)
    if case.get("docs"):
        st["docs"] = torch.tensor(_documents(case), **ints)
    if case.get("slopes"):
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")
    return st


# ---- plain forms --------------------------------------------------------------------------------
def _distance(st):
    """j - p, [batch or 1, 1, 1, q_len, kv_len]."""
    case = st["case"]
    i = torch.arange(case["q_len"], device="cuda")[None, :]
    p = i + (st["q_start"][:, None].long() if st["q_start"] is not None else 0)
    return (torch.arange(case["kv_len"], device="cuda")[None, None, :] - p[:, :, None])[:, None, None]


def _buckets(st, rel):
    top = st["case"]["max_distance"]
    return st["bucket_of"].long()[rel.clamp(-top, top) + top]


def _hidden(st, rel):
    j = torch.arange(st["case"]["kv_len"], device="cuda")
    hide = torch.zeros_like(rel, dtype=torch.bool)
    if st["causal"]:
        hide = rel > 0
        if st["prefix"] is not None:
            hide = hide & (j >= st["prefix"][:, None, None, None, None])
    if st["kv_lens"] is not None:
        hide = hide | (j >= st["kv_lens"][:, None, None, None, None])
    if st["docs"] is not None:
        hide = hide | (st["docs"][:, None, None, :, None] != st["docs"][:, None, None, None, :])
    return hide


def _heads(x, groups):
    """[batch, token, head, dim] -> fp32 [batch, head / groups, groups, token, dim]."""
    b, t, h, d = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(b, h // groups, groups, t, d)


def _tokens(x, dtype):
    b, hk, g, t, d = x.shape
    return x.reshape(b, hk * g, t, d).permute(0, 2, 1, 3).contiguous().to(dtype)


def _plain_attention(st):
    case = st["case"]
    G = case["heads"] // case["kv_heads"]
    B, H, Hk, Sq = case["batch"], case["heads"], case["kv_heads"], case["q_len"]
    dtype = st["q"].dtype
    q, k, v = _heads(st["q"], G), _heads(st["k"], 1), _heads(st["v"], 1)
    rel = _distance(st)
    s = (q @ k.transpose(-1, -2)) * st["scale"]
    t = None
    if st["cap"]:
        t = torch.tanh(s / st["cap"])
        s = t * st["cap"]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hk, G, 1, 1) * rel.abs().float()
    if st["table"] is not None:
        bucket = _buckets(st, rel[:, 0, 0])  # [batch or 1, q, kv]
        s = s + st["table"][:, bucket].transpose(0, 1).unflatten(1, (Hk, G))
    hide = _hidden(st, rel)
    s = s.masked_fill(hide, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = p @ v
    lse = (m + torch.log(total)).reshape(B, H, Sq)
    if case["kind"] == "step":
        return _tokens(o, dtype)
    if case["kind"] == "forward":
        return _tokens(o, dtype), lse
    do = _heads(st["dout"], G)
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    out = {"o": _tokens(o, dtype), "lse": lse}
    if st["table"] is not None:  # a sum over batch and positions: 64 bits, as a product with the 0/1 matrix of the buckets
        one = (bucket[0].flatten()[:, None] == torch.arange(case["buckets"], device="cuda")).double()
        out["dtable"] = (ds.double().sum(0).reshape(H, -1) @ one).float()
    if t is not None:
        ds = ds * (1 - t * t)
    ds = ds * st["scale"]
    out["dq"] = _tokens(ds @ k, dtype)
    out["dk"] = _tokens((ds.transpose(-1, -2) @ q).sum(2, keepdim=True), dtype)
    out["dv"] = _tokens(dv, dtype)
    return out


def _plain_bias(st):
    case = st["case"]
    bucket = _buckets(st, _distance(st)[0, 0, 0])
    out = (st["scores"].float() + st["table"][:, bucket]).to(st["scores"].dtype)
    one = (bucket.flatten()[:, None] == torch.arange(case["buckets"], device="cuda")).double()
    return out, (st["dscores"].double().sum(0).reshape(case["heads"], -1) @ one).float()


def run(st):
    case = st["case"]
    if not own:
        return _plain_bias(st) if case["kind"] == "bias" else _plain_attention(st)
    from dl_cuda_b200 import ops
    if case["kind"] == "bias":
        out = ops.rel_bias_fwd(st["table"], st["bucket_of"], scores=st["scores"])
        return out, ops.rel_bias_bwd(st["dscores"], st["bucket_of"], case["buckets"])
    how = dict(scale=st["scale"], cap=st["cap"], causal=st["causal"], kv_lens=st["kv_lens"], q_start=st["q_start"],
               prefix=st["prefix"], q_docs=st["docs"], kv_docs=st["docs"], slopes=st["slopes"], table=st["table"],
               bucket_of=st["bucket_of"])
    if case["kind"] == "step":
        return ops.attn_fwd(st["q"], st["k"], st["v"], want_lse=False, **how)[0]
    o, lse = ops.attn_fwd(st["q"], st["k"], st["v"], **how)
    if case["kind"] == "forward":
        return o, lse
    dq, dk, dv, dtable = ops.attn_bwd(st["dout"], st["q"], st["k"], st["v"], o, lse, **how)
    out = {"o": o, "lse": lse}
    if dtable is not None:
        out["dtable"] = dtable
    out.update(dq=dq, dk=dk, dv=dv)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------
def _visible_pairs(case):
    """Visible (query, key) pairs of all sequences, one head, and the keys that any query of a sequence sees."""
    Sq, Sk = case["q_len"], case["kv_len"]
    lens = _kv_lens(case) if case.get("ragged") else [Sk] * case["batch"]
    starts = _starts(case)
    prefixes = _prefixes(case) if case.get("prefix") else [0] * case["batch"]
    docs = _documents(case) if case.get("docs") else None
    pairs = 0
    i = torch.arange(Sq)
    for b in range(case["batch"]):
        low, high = torch.zeros(Sq, dtype=torch.long), torch.full((Sq,), lens[b], dtype=torch.long)
        if case.get("causal"):
            high = torch.maximum(i + starts[b] + 1, torch.tensor(prefixes[b])).clamp(max=lens[b])
        if docs is not None:
            row = torch.tensor(docs[b])
            low = torch.searchsorted(row, row)
            high = torch.minimum(high, torch.searchsorted(row, row, right=True))
        pairs += int((high - low).clamp(min=0).sum())
    return pairs, sum(lens)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B, Sq, Sk, H, Hk, D = (case[x] for x in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
    if case["kind"] == "bias":
        n = B * H * Sq * Sk
        return {"bytes": 3 * n * e, "flops": 2 * n}
    pairs, keys = _visible_pairs(case)
    q_bytes, kv_bytes = B * Sq * H * D * e, keys * Hk * D * e
    if case["kind"] == "train":  # q, k, v, dout in; o, dq, dk, dv and lse out; seven products of 2 * dim per pair
        return {"bytes": 4 * q_bytes + 2 * kv_bytes + 2 * B * Sk * Hk * D * e + B * H * Sq * 4, "flops": 14 * pairs * H * D}
    return {"bytes": 2 * q_bytes + 2 * kv_bytes + (B * H * Sq * 4 if case["kind"] == "forward" else 0),
            "flops": 4 * pairs * H * D}


# ---- 64-bit results, one key/value head at a time, gradients by automatic differentiation ---------
def exact(case, seed):
    st = prepare(case, seed)
    B, Sq, Sk, H, Hk, D = (case[x] for x in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
    f64 = dict(dtype=torch.float64, device="cuda")
    starts = _starts(case)
    lens = _kv_lens(case) if case.get("ragged") else [Sk] * B
    prefixes = _prefixes(case) if case.get("prefix") else [0] * B
    columns = torch.arange(Sk, device="cuda")
    index = None
    if case.get("buckets"):
        of, top = torch.tensor(_bucket_of(case), device="cuda"), case["max_distance"]
        index = lambda rel: of[torch.clamp(rel, min=-top, max=top) + top]  # noqa: E731
    if case["kind"] == "bias":
        rel = columns[None, :] - torch.arange(Sq, device="cuda")[:, None]
        where = index(rel)
        out = torch.stack([st["scores"][:, h].double() + st["table"][h].double()[where] for h in range(H)], 1)
        dtable = torch.zeros(H, case["buckets"], **f64)
        for n in range(case["buckets"]):
            for h in range(H):
                dtable[h, n] = st["dscores"][:, h].double().sum(0)[where == n].sum()
        return out, dtable
    G, train = H // Hk, case["kind"] == "train"
    o, lse = torch.zeros(B, Sq, H, D, **f64), torch.zeros(B, H, Sq, **f64)
    dq, dk, dv = (torch.zeros(B, n, h, D, **f64) if train else None for n, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))
    dtable = torch.zeros(H, case["buckets"], **f64) if train and case.get("buckets") else None
    for b in range(B):
        position = torch.arange(Sq, device="cuda") + starts[b]
        rel = columns[None, :] - position[:, None]
        seen = (columns < lens[b])[None, :].expand(Sq, Sk)
        if case.get("causal"):
            seen = seen & ((rel <= 0) | (columns < prefixes[b])[None, :])
        if case.get("docs"):
            seen = seen & (st["docs"][b][:, None] == st["docs"][b][None, :])
        for hk in range(Hk):
            with torch.set_grad_enabled(train):
                heads = slice(hk * G, hk * G + G)
                q = st["q"][b, :, heads].double().permute(1, 0, 2).detach().requires_grad_(train)
                k = st["k"][b, :, hk].double().detach().requires_grad_(train)
                v = st["v"][b, :, hk].double().detach().requires_grad_(train)
                s = torch.einsum("gid,jd->gij", q, k) / math.sqrt(D)
                if case.get("cap"):
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if case.get("slopes"):
                    s = s - st["slopes"][heads].double()[:, None, None] * rel.abs()
                bias = None
                if index is not None:
                    bias = st["table"][heads].double()[:, index(rel)].detach().requires_grad_(train)
                    s = s + bias
                s = torch.where(seen, s, torch.full((), -math.inf, **f64))
                z = torch.logsumexp(s, -1)
                y = torch.einsum("gij,jd->gid", torch.exp(s - z[..., None]), v)
                if train:
                    wrt = [q, k, v] + ([bias] if bias is not None else [])
                    got = torch.autograd.grad(y, wrt, st["dout"][b, :, heads].double().permute(1, 0, 2))
                    dq[b, :, heads] = got[0].permute(1, 0, 2)
                    dk[b, :, hk] = got[1]
                    dv[b, :, hk] = got[2]
                    if bias is not None:
                        for n in range(case["buckets"]):
                            dtable[heads, n] += got[3].mul(index(rel) == n).sum((1, 2))
                o[b, :, heads] = y.detach().permute(1, 0, 2)
                lse[b, heads] = z.detach()
    if case["kind"] == "step":
        return o
    if not train:
        return o, lse
    out = {"o": o, "lse": lse}
    if dtable is not None:
        out["dtable"] = dtable
    out.update(dq=dq, dk=dk, dv=dv)
    return out
