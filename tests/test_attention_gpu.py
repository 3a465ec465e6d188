"""The attention operators against their formulas in 64 bits (tests/attention_reference.py holds the
formulas and the bounds, entry by entry)."""
import math

import pytest
import torch

from attention_reference import check, reference
from dl_cuda_b200 import capi, ops

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def make(seed, dtype, B, Sq, Sk, H, Hk, D, layout="fused", std=1.5):
    """q, k, v, dout on the GPU, as views of what programs hold."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[dtype]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)

    if layout == "fused" and Sq == Sk:  # one projection: heads side by side
        x = normal(B, Sq, H + 2 * Hk, D, scale=std)
        q, k, v = x[:, :, :H], x[:, :, H:H + Hk], x[:, :, H + Hk:]
    elif layout == "heads_first":  # [batch, head, token, column]
        q, k, v = (normal(B, h, s, D, scale=std).transpose(1, 2) for h, s in ((H, Sq), (Hk, Sk), (Hk, Sk)))
    else:
        q, k, v = (normal(B, s, h, D, scale=std) for h, s in ((H, Sq), (Hk, Sk), (Hk, Sk)))
    return q, k, v, normal(B, Sq, H, D)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def options(kind, B, Sq, Sk, H, seed=0):
    gen = torch.Generator().manual_seed(seed + 17)
    how = {}
    for part in kind.split("+"):
        if part == "causal":
            how["causal"] = True
        elif part == "cap":
            how["cap"] = 5.0  # far into the bend
        elif part == "slopes":
            how["slopes"] = torch.rand(H, generator=gen).cuda()
        elif part in ("table", "table1"):
            both = part == "table"
            how["bucket_of"] = ops.rel_bucket_map(16, 40, both).cuda()
            how["table"] = torch.randn(H, 16, generator=gen).cuda()
        elif part == "docs":
            n = max(Sq, Sk)
            d = torch.randint(0, 3, (B, n), generator=gen).sort(1)[0].int().cuda()
            how["q_docs"], how["kv_docs"] = d[:, n - Sq:].contiguous(), d[:, :Sk].contiguous()
        elif part == "mixed_docs":  # in no order, with queries whose document has no key
            how["q_docs"] = torch.randint(0, 5, (B, Sq), generator=gen).int().cuda()
            how["kv_docs"] = torch.randint(1, 4, (B, Sk), generator=gen).int().cuda()
        elif part == "lens":
            how["kv_lens"] = torch.randint(0, Sk + 1, (B,), generator=gen).int().cuda()
            how["kv_lens"][0] = 0  # a sequence without a key
        elif part == "prefix":
            how["prefix"] = torch.randint(0, Sk + 1, (B,), generator=gen).int().cuda()
        elif part == "start":
            how["q_start"] = torch.randint(-3, Sk, (B,), generator=gen).int().cuda()
    return how


def run_both(q, k, v, dout, how, grads=True):
    values, bounds = reference(q, k, v, dout if grads else None, **how)
    o, lse = ops.attn_fwd(q, k, v, **how)
    got = dict(o=o, lse=lse)
    if grads:
        dq, dk, dv, dtable = ops.attn_bwd(dout, q, k, v, o, lse, **how)
        got.update(dq=dq, dk=dk, dv=dv, dtable=dtable)
    check(got, values, bounds)
    assert capi.pipeline_timeouts() == 0
    return got


KINDS = ["plain", "causal", "cap+causal", "slopes+causal", "table", "table1+causal", "cap+table+docs", "docs+causal",
         "mixed_docs", "lens", "lens+causal+start", "prefix+causal", "prefix+causal+lens+slopes",
         "cap+slopes+table+causal+docs+lens+prefix"]
SHAPES = [  # B, Sq, Sk, H, Hk, D
    (2, 1, 1, 2, 2, 16), (1, 64, 64, 2, 1, 64), (3, 65, 65, 4, 2, 32), (2, 130, 130, 4, 4, 64), (1, 257, 257, 3, 1, 128),
    (2, 33, 190, 4, 2, 80), (2, 200, 70, 2, 2, 128), (1, 300, 300, 2, 2, 8),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, kind, dtype):
    B, Sq, Sk, H, Hk, D = shape
    q, k, v, dout = make(sum(shape), dtype, *shape)
    run_both(q, k, v, dout, options(kind, B, Sq, Sk, H))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 4, 17, 24, 40, 63, 72, 96, 100, 120, 127])
def test_head_widths(D, dtype):
    q, k, v, dout = make(D, dtype, 1, 70, 70, 4, 2, D)
    run_both(q, k, v, dout, dict(causal=True))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "plain"])
@pytest.mark.parametrize("D", [64, 20])
def test_layouts(layout, D, dtype):
    q, k, v, dout = make(5, dtype, 2, 96, 96, 4, 2, D, layout)
    run_both(q, k, v, dout.transpose(1, 2).contiguous().transpose(1, 2) if layout == "heads_first" else dout, dict(causal=True))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_repeated_inputs_and_strided_outputs(dtype):
    """Keys of one sequence broadcast over the batch (stride 0), a broadcast gradient, outputs inside larger buffers."""
    q, k, v, dout = make(9, dtype, 3, 70, 70, 4, 2, 64, "plain")
    k, v = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)
    dout = dout[:, :1].expand(-1, 70, -1, -1)
    how = dict(causal=True)
    values, bounds = reference(q, k, v, dout, **how)
    wide = torch.full((3, 70, 8, 64), 7.0, dtype=q.dtype, device="cuda")
    o, lse = ops.attn_fwd(q, k, v, out=wide[:, :, 2:6], **how)
    room = [torch.full((3, 72, h + 1, 64), 7.0, dtype=q.dtype, device="cuda") for h in (4, 2, 2)]
    views = [r[:, 1:71, :h] for r, h in zip(room, (4, 2, 2))]
    dq, dk, dv, _ = ops.attn_bwd(dout, q, k, v, o, lse, dq=views[0], dk=views[1], dv=views[2], **how)
    check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv), values, bounds)
    assert (wide[:, :, :2] == 7).all() and (wide[:, :, 6:] == 7).all()
    for r, h in zip(room, (4, 2, 2)):
        assert (r[:, 0] == 7).all() and (r[:, 71:] == 7).all() and (r[:, :, h] == 7).all()


@pytest.mark.parametrize("offset", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_addresses_off_the_vector_grid(dtype, offset):
    q, k, v, dout = make(11, dtype, 1, 66, 66, 2, 2, 64, "plain")

    def moved(t):
        flat = torch.zeros(t.numel() + 64, dtype=t.dtype, device="cuda")
        view = flat[offset:offset + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    run_both(moved(q), moved(k), moved(v), moved(dout), dict(causal=True))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("G", [1, 2, 4, 7, 8, 16, 24])
@pytest.mark.parametrize("q_len", [1, 2, 5])
def test_few_queries_against_a_cache(q_len, G, dtype):
    """Single and few new tokens against ragged caches whose unused part holds NaN."""
    B, Sk, Hk, D = 5, 700, 2, 128
    q, k, v, _ = make(q_len * 31 + G, dtype, B, q_len, Sk, G * Hk, Hk, D, "plain")
    lens = ints([q_len, 64, 129, 700, 333])
    for b, n in enumerate(lens.tolist()):
        k[b, n:] = math.nan
        v[b, n:] = math.nan
    for extra in ({}, dict(cap=5.0), options("slopes", B, q_len, Sk, G * Hk), options("table1", B, q_len, Sk, G * Hk)):
        how = dict(causal=True, kv_lens=lens, q_start=lens - q_len, **extra)
        run_both(q, k, v, None, how, grads=False)
    # without lengths the causal bound alone keeps the unused part out
    run_both(q, k, v, None, dict(causal=True, q_start=lens - q_len), grads=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [16, 20, 64, 80, 128])
@pytest.mark.parametrize("Sk", [1, 63, 64, 65, 1000, 5000])
def test_one_token_lengths_and_widths(Sk, D, dtype):
    q, k, v, _ = make(Sk + D, dtype, 2, 1, Sk, 8, 2, D, "plain")
    run_both(q, k, v, None, dict(kv_lens=ints([Sk, (Sk + 1) // 2])), grads=False)
    run_both(q, k, v, None, options("mixed_docs", 2, 1, Sk, 8), grads=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_unused_keys_may_hold_anything_in_training(dtype):
    B, S = 3, 200
    q, k, v, dout = make(21, dtype, B, S, S, 4, 2, 64, "plain")
    lens = ints([1, 131, 200])
    for b, n in enumerate(lens.tolist()):
        k[b, n:] = math.nan
        v[b, n:] = math.inf
    for extra in ({}, dict(cap=5.0), options("slopes", B, S, S, 4), options("table", B, S, S, 4),
                  dict(cap=5.0, **options("table+docs", B, S, S, 4))):
        got = run_both(q, k, v, dout, dict(kv_lens=lens, **extra))
        for b, n in enumerate(lens.tolist()):
            assert (got["dk"][b, n:] == 0).all() and (got["dv"][b, n:] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_table_entries_that_hide_their_keys(dtype):
    q, k, v, dout = make(23, dtype, 2, 150, 150, 2, 2, 64)
    how = options("table", 2, 150, 150, 2)
    how["table"][0, 3:9] = -math.inf
    how["table"][1, 9:] = torch.finfo(torch.float32).min
    run_both(q, k, v, dout, how)
    how["table"][1] = torch.finfo(torch.float32).min  # head 1 sees nothing at all
    got = run_both(q, k, v, dout, how)
    assert (got["o"][:, :, 1] == 0).all() and (got["dq"][:, :, 1] == 0).all() and (got["dv"][:, :, 1] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_large_scores(dtype):
    """Scores of some hundreds: the running maximum has to carry them."""
    q, k, v, dout = make(25, dtype, 1, 190, 190, 2, 2, 64, std=8.0)
    run_both(q, k, v, dout, dict(causal=True))
    run_both(q, k, v, dout, dict(causal=True, cap=30.0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_empty_sizes(dtype):
    dt = DTYPES[dtype]
    e = lambda *s: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    o, lse = ops.attn_fwd(e(0, 5, 2, 16), e(0, 7, 2, 16), e(0, 7, 2, 16))
    assert o.shape == (0, 5, 2, 16) and lse.shape == (0, 2, 5)
    o, lse = ops.attn_fwd(e(2, 0, 2, 16), e(2, 7, 2, 16), e(2, 7, 2, 16))
    assert o.numel() == 0
    q = e(2, 5, 2, 16) + 1
    o, lse = ops.attn_fwd(q, e(2, 0, 2, 16), e(2, 0, 2, 16))
    assert (o == 0).all() and (lse == -math.inf).all()
    dq, dk, dv, _ = ops.attn_bwd(q, q, e(2, 0, 2, 16), e(2, 0, 2, 16), o, lse)
    assert (dq == 0).all() and dk.numel() == 0
    k = e(2, 7, 2, 16) + 1
    how = options("table", 2, 0, 7, 2)
    none = e(2, 0, 2, 16)
    dq, dk, dv, dtable = ops.attn_bwd(none, none, k, k, none, torch.zeros(2, 2, 0, device="cuda"), **how)
    assert dq.numel() == 0 and (dk == 0).all() and (dv == 0).all() and (dtable == 0).all()


@pytest.mark.parametrize("kind", ["plain", "causal", "cap+causal", "slopes+causal", "table", "table64", "mixed_docs", "lens"])
@pytest.mark.parametrize("shape", [(2, 19, 19, 4, 2, 64), (1, 200, 200, 2, 1, 128), (2, 130, 400, 2, 2, 20), (1, 700, 700, 2, 1, 16),
                                   (1, 150, 150, 2, 2, 72)])
def test_values_with_a_common_part(shape, kind):
    """Values that share a large part: the output's rounding, times the output's gradient, is far more than the score
    gradients, and must not reach dq and dk through delta."""
    B, Sq, Sk, H, Hk, D = shape
    q, k, v, dout = make(sum(shape) + 1, "bf16", *shape, layout="plain", std=1.0)
    v = (v.float() * 0.25 + 6.0).bfloat16()
    if kind == "table64":  # more buckets than leave room for four threads a row
        how = dict(table=torch.randn(H, 64, generator=torch.Generator().manual_seed(4)).cuda(), bucket_of=ops.rel_bucket_map(64, 90).cuda())
    else:
        how = options(kind, B, Sq, Sk, H)
    values, bounds = reference(q, k, v, dout, exact_delta=True, **how)
    o, lse = ops.attn_fwd(q, k, v, **how)
    dq, dk, dv, dtable = ops.attn_bwd(dout, q, k, v, o, lse, **how)
    check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv, dtable=dtable), values, bounds)


@pytest.mark.parametrize("D,buckets", [(64, 2), (64, 64), (128, 2), (128, 32), (128, 64), (20, 2)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_bucket_map_that_alternates(D, buckets, dtype):
    """A map whose buckets change at every distance, over some 2000 keys: every addition to a bucket's sum counts.
    An output that puts delta off by D shows what the sums' roundings are worth: the gradient of the table must not
    move with it, since a row's score gradients add up to zero whatever delta is taken.  (dq and dk hold for the
    forward's own output, and so does every bound.)"""
    B, Sq, S, H = 1, 128, 1900, 2
    gen = torch.Generator(device="cuda").manual_seed(D + buckets)
    q = torch.zeros(B, Sq, H, D, device="cuda", dtype=DTYPES[dtype])
    k, v = (torch.randn(B, S, H, D, generator=gen, device="cuda").to(DTYPES[dtype]) for _ in range(2))
    dout = torch.ones_like(q)
    how = dict(q_start=ints([S // 2 - Sq // 2]), table=torch.zeros(H, buckets, device="cuda"),
               bucket_of=ints([0, 1, 1, 1] * 512 + [0]))
    values, bounds = reference(q, k, v, dout, exact_delta=dtype == "bf16", **how)
    o, lse = ops.attn_fwd(q, k, v, **how)
    dq, dk, dv, dtable = ops.attn_bwd(dout, q, k, v, o, lse, **how)
    check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv, dtable=dtable), values, bounds)
    moved = ops.attn_bwd(dout, q, k, v, torch.ones_like(o), lse, **how)[3]
    # Each of Sq rows: D times the error of a bucket's share w of the probabilities.  In fp32 a sum of n additions is off
    # by n / 2 steps of 2^-24 of it (its addends are alike), n <= S / 16 + 32 with four threads a row, twice that with
    # two; the two buckets' errors move the share w by at most w (1 - w) each, and w is 1/4.
    error = D * Sq * 2 * 0.1875 * (S / 8 + 64) * 2.0 ** -24 + D * Sq * 2.0 ** -21
    assert ((moved.double() - values["dtable"]).abs() <= error + bounds["dtable"]).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("kind", ["plain", "cap+causal", "slopes", "table", "table+causal+docs"])
def test_backward_of_shares_of_the_keys(kind, D, dtype):
    """The keys in three calls with o and lse of all of them: each its own dk and dv and a part of dq and dtable."""
    B, Sq, Sk, H, Hk = 2, 150, 400, 4, 2
    q, k, v, dout = make(D, dtype, B, Sq, Sk, H, Hk, D, "plain", std=1.0)
    how = options(kind, B, Sq, Sk, H)
    values, bounds = reference(q, k, v, dout, shares=True, q_start=ints([250, 100]), **how)
    o, lse = ops.attn_fwd(q, k, v, q_start=ints([250, 100]), **how)
    u = torch.finfo(q.dtype).eps / 2
    dq, dk, dv, dtable = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), [], [], 0.0
    for first, last in ((0, 130), (130, 257), (257, 400)):
        share = dict(how, q_start=ints([250 - first, 100 - first]))
        if "kv_docs" in how:
            share["kv_docs"] = how["kv_docs"][:, first:last].contiguous()
        got = ops.attn_bwd(dout, q, k[:, first:last], v[:, first:last], o, lse, **share)
        dq += got[0].double()
        bounds["dq"] += u / (1 - u) * got[0].double().abs()  # each share's dq is rounded by itself
        dk.append(got[1])
        dv.append(got[2])
        if got[3] is not None:
            dtable = dtable + got[3].double()
    got = dict(o=o, lse=lse, dq=dq, dk=torch.cat(dk, 1), dv=torch.cat(dv, 1))
    check(dict(got, dtable=dtable) if how.get("table") is not None else got, values, bounds)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_a_share_with_nearly_all_the_weight(D, dtype):
    """A first share of the keys that holds all but some 1e-4 of every row's weight is not taken for the whole."""
    B, Sq, Sk, H = 1, 100, 300, 2
    q, k, v, dout = make(D + 3, dtype, B, Sq, Sk, H, H, D, "plain", std=0.3)
    q[..., 0] = 4.5 * D ** 0.25
    k[:, :150, :, 0], k[:, 150:, :, 0] = D ** 0.25, -D ** 0.25  # 9 between the shares' scores
    v[:, 150:] += 30.0  # and one sign for what the little weight brings
    dout = 1.0 + 0.1 * dout
    u = torch.finfo(q.dtype).eps / 2
    how = options("table", B, Sq, Sk, H)
    values, bounds = reference(q, k, v, dout, shares=True, **how)
    o, lse = ops.attn_fwd(q, k, v, **how)
    dq, dtable, dk, dv = 0.0, 0.0, [], []
    for first, last in ((0, 150), (150, 300)):
        got = ops.attn_bwd(dout, q, k[:, first:last], v[:, first:last], o, lse, **dict(how, q_start=ints([-first])))
        dq = dq + got[0].double()
        bounds["dq"] += u / (1 - u) * got[0].double().abs()
        dk.append(got[1])
        dv.append(got[2])
        dtable = dtable + got[3].double()
    check(dict(dq=dq, dk=torch.cat(dk, 1), dv=torch.cat(dv, 1), dtable=dtable), values, bounds)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_empty_sizes_with_documents(dtype):
    dt = DTYPES[dtype]
    full = lambda *s: torch.ones(*s, dtype=dt, device="cuda")  # noqa: E731
    docs = lambda b, n: torch.zeros(b, n, dtype=torch.int32, device="cuda")  # noqa: E731
    for B, Sq, Sk in ((2, 5, 0), (2, 1, 0), (2, 0, 7), (0, 5, 7), (2, 0, 0)):
        q, k = full(B, Sq, 2, 16), full(B, Sk, 2, 16)
        how = dict(q_docs=docs(B, Sq), kv_docs=docs(B, Sk))
        o, lse = ops.attn_fwd(q, k, k, **how)
        assert (o == 0).all() and (lse == -math.inf).all()
        dq, dk, dv, _ = ops.attn_bwd(q, q, k, k, o, lse, **how)
        assert dq.shape == q.shape and dk.shape == k.shape
        assert (dq == 0).all() and (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 20])
def test_same_bits_every_time_and_in_a_graph(D, dtype):
    """The second call gives the first one's bits; a captured step follows lengths that change between replays."""
    B, S, H = 2, 300, 4
    q, k, v, dout = make(27, dtype, B, S, S, H, 2, D)
    how = options("cap+table1+causal+docs", B, S, S, H)
    lens = ints([300, 211])
    how["kv_lens"] = lens

    def step():
        o, lse = ops.attn_fwd(q, k, v, **how)
        return (o, lse) + ops.attn_bwd(dout, q, k, v, o, lse, **how)

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    for a, b in zip(first, held):
        assert torch.equal(a, b)
    lens.copy_(ints([17, 300]))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(step(), held):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_two_streams_at_once(dtype):
    """Two calls in flight, each with its own workspace, do not disturb each other."""
    sets = [make(40 + n, dtype, 2, 1, 3000, 8, 2, 64, "plain")[:3] for n in range(2)]
    want = [ops.attn_fwd(*s)[0].clone() for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(10):
        for n, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[n] = ops.attn_fwd(*s)[0]
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["causal", "cap+table1+causal"])
def test_gradients_against_differences(kind):
    """Central differences of the 64-bit forward along random directions, against the kernels' fp32 gradients."""
    B, S, H, Hk, D = 1, 70, 2, 1, 16
    q, k, v, dout = make(51, "fp32", B, S, S, H, Hk, D, "plain")
    how = options(kind, B, S, S, H)
    o, lse = ops.attn_fwd(q, k, v, **how)
    grads = dict(zip(("q", "k", "v", "table"), ops.attn_bwd(dout, q, k, v, o, lse, **how)))
    inputs = dict(q=q, k=k, v=v, table=how.get("table"))
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = 1e-4  # the difference quotient is off by about h^2 of the third derivative: 1e-8
    for name, x in inputs.items():
        if x is None:
            continue
        along = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)

        def loss(sign):
            moved = {n: (y.double() + sign * h * along if n == name else y) for n, y in inputs.items()}
            rest = {n: y for n, y in how.items() if n != "table"}
            if moved["table"] is not None:
                rest["table"] = moved["table"]
            return (reference(moved["q"].double(), moved["k"].double(), moved["v"].double(), **rest)[0]["o"] * dout.double()).sum()

        want = ((loss(1) - loss(-1)) / (2 * h)).item()
        got = (grads[name].double() * along).sum().item()
        size = (grads[name].double() * along).abs().sum().item()
        assert abs(got - want) <= 2e-6 * size + 1e-6, (name, got, want)


def test_wrong_device_and_wrong_arguments():
    q, k, v, dout = make(61, "fp32", 1, 8, 8, 2, 2, 16, "plain")
    o, lse = ops.attn_fwd(q, k, v)
    with pytest.raises(ValueError):
        ops.attn_fwd(q.cpu(), k, v)
    with pytest.raises(ValueError):
        ops.attn_fwd(q, k.cpu(), v)
    with pytest.raises(TypeError):
        ops.attn_fwd(q, k.bfloat16(), v)
    with pytest.raises(TypeError):
        ops.attn_fwd(q.half(), k.half(), v.half())
    with pytest.raises(ValueError):
        ops.attn_fwd(q.transpose(2, 3), k, v)
    with pytest.raises(ValueError):
        ops.attn_fwd(q, k, v, kv_lens=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.attn_fwd(q, k, v, table=torch.zeros(2, 4, device="cuda"))
    with pytest.raises(capi.DlbError):
        ops.attn_fwd(q, k, v, q_docs=torch.zeros(1, 8, dtype=torch.int32, device="cuda"))
    with pytest.raises(capi.DlbError):
        ops.attn_fwd(q, k[:, :, :1].expand(-1, -1, 3, -1), v[:, :, :1].expand(-1, -1, 3, -1))
    with pytest.raises(capi.DlbError):
        ops.attn_fwd(q, k, v, out=o[:, :1].expand(-1, 8, -1, -1))
    with pytest.raises(ValueError):
        ops.attn_bwd(dout[:, :4], q, k, v, o, lse)


# --- bucketed position bias on a score matrix ------------------------------------------------------
BIAS_SHAPES = [(1, 1, 1, 1), (2, 3, 64, 64), (1, 4, 33, 130), (3, 2, 127, 65), (2, 2, 5, 1000), (1, 12, 200, 200)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("q_start", [0, 7, -200])
@pytest.mark.parametrize("shape", BIAS_SHAPES)
def test_bias_matrix(shape, q_start, dtype):
    B, H, Sq, Sk = shape
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    dt, u = DTYPES[dtype], 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    scores = torch.randn(shape, generator=gen, device="cuda").to(dt)
    table = torch.randn(H, 32, generator=gen, device="cuda")
    for both in (True, False):
        bucket_of = ops.rel_bucket_map(32, 50, both).cuda()
        rel = torch.arange(Sk, device="cuda")[None] - (q_start + torch.arange(Sq, device="cuda"))[:, None]
        bucket = bucket_of.long()[rel.clamp(-50, 50) + 50]
        bias = table.double()[:, bucket]
        for s in (scores, None):
            out = ops.rel_bias_fwd(table, bucket_of, scores=s, shape=shape, q_start=q_start, dtype=dt)
            want = bias[None].expand(shape) if s is None else s.double() + bias
            # one fp32 addition, one rounding to the storage type
            assert ((out.double() - want).abs() <= (u + 2.0 ** -24) * want.abs() + 1e-30).all()
        inside = scores.clone()
        ops.rel_bias_fwd(table, bucket_of, scores=inside, q_start=q_start, out=inside)
        assert torch.equal(inside, ops.rel_bias_fwd(table, bucket_of, scores=scores, q_start=q_start))
        d = ops.rel_bias_bwd(scores, bucket_of, 32, q_start=q_start)
        assert torch.equal(d, ops.rel_bias_bwd(scores, bucket_of, 32, q_start=q_start))
        one = torch.nn.functional.one_hot(bucket, 32).double()
        want = torch.einsum("bhij,ijn->hn", scores.double(), one)
        size = torch.einsum("bhij,ijn->hn", scores.double().abs(), one)
        # at most B * Sq * (Sk / 256 + 2) fp32 additions stand one behind another, shared out over the row groups
        chain = B * Sq * (Sk / 256 + 2) / max(1, min(B * Sq, 888 // H)) + Sk / 256 + 300
        assert ((d.double() - want).abs() <= chain * 2.0 ** -24 * size + 1e-30).all()


def test_bias_matrix_in_the_unfused_chain():
    """Scores by dlb_gemm_f32, the bias, dlb_softmax_fwd and the product with the values: the fused call's result,
    and the same gradient of the table by both ways."""
    B, S, H, D = 2, 70, 3, 16
    q, k, v, dout = make(71, "fp32", B, S, S, H, H, D, "plain")
    how = options("table", B, S, S, H)
    values, bounds = reference(q, k, v, dout, **how)
    hf = lambda x: x.permute(0, 2, 1, 3).reshape(B * H, S, D).contiguous()  # noqa: E731
    scores = ops.gemm(hf(q), hf(k).transpose(1, 2), alpha=D ** -0.5).view(B, H, S, S)
    biased = ops.rel_bias_fwd(how["table"], how["bucket_of"], scores=scores)
    p = ops.softmax_fwd(biased)
    o = ops.gemm(p.view(B * H, S, S), hf(v)).view(B, H, S, D).permute(0, 2, 1, 3)
    check(dict(o=o), values, bounds)
    fused, lse = ops.attn_fwd(q, k, v, **how)
    check(dict(o=fused, lse=lse), values, bounds)
    dp = ops.gemm(hf(dout), hf(v).transpose(1, 2)).view(B, H, S, S)
    ds = ops.softmax_bwd(dp, p)
    by_matrix = ops.rel_bias_bwd(ds, how["bucket_of"], 16)
    by_fusion = ops.attn_bwd(dout, q, k, v, fused, lse, **how)[3]
    check(dict(dtable=by_matrix), values, bounds)
    check(dict(dtable=by_fusion), values, bounds)


# --- what only long or unusual calls reach -----------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shift", [-95.0, -88.0, -86.0, -70.0, -30.0, 25.0, 60.0, 85.0])
@pytest.mark.parametrize("q_len", [1, 150])
def test_scores_far_from_zero(q_len, shift, dtype):
    """A bias common to all keys changes lse alone, also where 2^score would leave fp32's range."""
    B, S, H, D = 2, 300, 2, 64
    q, k, v, dout = make(81, dtype, B, q_len, S, H, H, D, "plain")
    how = options("table", B, q_len, S, H)
    how["table"] = how["table"] + shift
    run_both(q, k, v, dout, how, grads=q_len > 1)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_steep_distance_bias(causal, dtype):
    """Slopes that take neighbouring tiles 2^100 apart, keys on both sides, the near ones partly hidden."""
    B, S, H, D = 2, 700, 2, 64
    q, k, v, dout = make(83, dtype, B, S, S, H, H, D, "plain")
    how = dict(causal=causal, slopes=torch.tensor([1.0, 0.7], device="cuda"), prefix=ints([650, 0]) if causal else None,
               kv_lens=ints([700, 300]))
    run_both(q, k, v, dout, how)


@pytest.mark.parametrize("q_len,Sk,H,Hk,D", [(17, 5000, 8, 2, 128), (64, 3000, 2, 1, 64), (200, 2048, 1, 1, 80), (300, 900, 2, 2, 128),
                                            (40, 1025, 4, 4, 32)])
@pytest.mark.parametrize("kind", ["plain", "cap+causal", "table", "mixed_docs", "lens"])
def test_a_chunk_against_a_long_cache(q_len, Sk, H, Hk, D, kind):
    """More queries than a single-token call has, too few to fill the GPU: the key tiles are shared out."""
    B = 2
    q, k, v, _ = make(q_len + Sk, "bf16", B, q_len, Sk, H, Hk, D, "plain")
    how = options(kind, B, q_len, Sk, H)
    if how.get("causal"):
        how["q_start"] = ints([Sk - q_len, Sk // 2])
        how["kv_lens"] = ints([Sk, Sk // 2 + q_len])
        k[1, Sk // 2 + q_len:] = math.nan
        v[1, Sk // 2 + q_len:] = math.inf
    run_both(q, k, v, None, how, grads=False)
    assert torch.equal(ops.attn_fwd(q, k, v, **how)[0], ops.attn_fwd(q, k, v, **how)[0])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_64_buckets_and_the_longest_map(D, dtype):
    B, S, H = 1, 400, 2
    q, k, v, dout = make(85, dtype, B, S, S, H, H, D, "plain")
    gen = torch.Generator().manual_seed(1)
    how = dict(table=torch.randn(H, 64, generator=gen).cuda(), bucket_of=ops.rel_bucket_map(64, 1024, True).cuda())
    run_both(q, k, v, dout, how)
    how["bucket_of"] = torch.randint(0, 64, (2 * 300 + 1,), generator=gen).int().cuda()  # a map of one's own
    run_both(q, k, v, dout, how)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["causal", "lens", "cap+table+causal", "prefix+causal+slopes", "returning_docs", "returning_docs+causal"])
@pytest.mark.parametrize("shape", [(1, 1700, 1700, 8, 2, 128), (1, 2300, 2300, 4, 1, 64), (2, 1100, 1500, 4, 2, 40)])
def test_long_sequences(shape, kind, dtype):
    """Many tiles in the rings of both passes, times the heads of a group; documents that come back leave gaps in
    the list of tiles."""
    B, Sq, Sk, H, Hk, D = shape
    q, k, v, dout = make(sum(shape), dtype, *shape, layout="plain", std=1.0)
    how = options(kind.replace("returning_docs", "plain"), B, Sq, Sk, H)
    if Sq != Sk:
        how["q_start"] = ints([Sk - Sq] * B)
    if "returning_docs" in kind:  # three numbers in runs of 170 tokens
        runs = torch.randint(0, 3, (B, Sk // 170 + 1), generator=torch.Generator().manual_seed(Sk))
        docs = runs.repeat_interleave(170, 1)[:, :Sk].int().cuda()
        how["q_docs"], how["kv_docs"] = docs[:, Sk - Sq:].contiguous(), docs.contiguous()
    values, bounds = reference(q, k, v, dout, exact_delta=dtype == "bf16", **how)
    o, lse = ops.attn_fwd(q, k, v, **how)
    dq, dk, dv, dtable = ops.attn_bwd(dout, q, k, v, o, lse, **how)
    check(dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv, dtable=dtable), values, bounds)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_bucket_map_edges(dtype):
    """A map of one entry; values outside 0..buckets-1 count as the nearest bucket."""
    q, k, v, dout = make(87, dtype, 1, 40, 40, 2, 2, 64, "plain")
    table = torch.randn(2, 4, generator=torch.Generator().manual_seed(2)).cuda()
    run_both(q, k, v, dout, dict(table=table, bucket_of=ints([2])))
    run_both(q, k, v, dout, dict(table=table, bucket_of=ints([-7, 1, 9, 3, 2])))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_positions_far_out(dtype):
    """Starts at the ends of the range that is served, and beyond it (clamped)."""
    q, k, v, dout = make(89, dtype, 4, 30, 50, 2, 2, 64, "plain")
    starts = torch.tensor([2 ** 30, -2 ** 30, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64).int().cuda()
    run_both(q, k, v, dout, dict(q_start=starts, causal=True))
    how = options("table", 4, 30, 50, 2)
    run_both(q, k, v, dout, dict(q_start=starts, **how))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_negative_and_zero_scales(dtype):
    q, k, v, dout = make(91, dtype, 1, 90, 90, 2, 1, 64, "plain")
    for scale in (0.0, -0.2, 1e-3, 3.0):
        run_both(q, k, v, dout, dict(scale=scale, causal=True))


@pytest.mark.parametrize("cap", [1e-3, 0.5, 200.0, 1e5])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_caps_from_tight_to_loose(cap, dtype):
    q, k, v, dout = make(93, dtype, 1, 150, 150, 2, 1, 64, "plain")
    run_both(q, k, v, dout, dict(cap=cap, causal=True))
    run_both(q[:, :1], k, v, None, dict(cap=cap), grads=False)


def test_rows_behind_the_outputs_stay_as_they_were():
    """Outputs that are the front part of larger buffers: nothing is written behind them."""
    for dtype in ("fp32", "bf16"):
        for q_len, Sk in ((1, 900), (5, 100), (100, 100), (130, 260)):
            q, k, v, dout = make(95, dtype, 2, q_len, Sk, 4, 2, 64, "plain")
            room = {n: torch.full((2, t + 3, h, 64), 7.0, dtype=q.dtype, device="cuda")
                    for n, t, h in (("o", q_len, 4), ("dq", q_len, 4), ("dk", Sk, 2), ("dv", Sk, 2))}
            o, lse = ops.attn_fwd(q, k, v, out=room["o"][:, :q_len])
            ops.attn_bwd(dout, q, k, v, o, lse, dq=room["dq"][:, :q_len], dk=room["dk"][:, :Sk], dv=room["dv"][:, :Sk])
            for n, t in (("o", q_len), ("dq", q_len), ("dk", Sk), ("dv", Sk)):
                assert (room[n][:, t:] == 7).all(), (dtype, q_len, n)
                assert not (room[n][:, :t] == 7).all()


def test_two_host_threads():
    """Calls of one kernel with different needs of shared memory from two host threads at once."""
    import threading
    sets = []
    for n, (D, docs) in enumerate(((64, 40), (64, 3000))):
        q, k, v, dout = make(97 + n, "bf16", 1, 130, docs, 2, 2, D, "plain")
        how = dict(bucket_of=ops.rel_bucket_map(16, 40 + 900 * n, True).cuda(), table=torch.randn(2, 16, device="cuda"))
        o, lse = ops.attn_fwd(q, k, v, **how)
        sets.append(((q, k, v), how, dout, o, lse, ops.attn_bwd(dout, q, k, v, o, lse, **how)))
    torch.cuda.synchronize()
    failures = []

    def work(n):
        try:
            (q, k, v), how, dout, o, lse, want = sets[n]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    got = ops.attn_bwd(dout, q, k, v, *ops.attn_fwd(q, k, v, **how), **how)
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(x, y) for x, y in zip(got, want)):
                failures.append("results differ")
        except Exception as e:  # noqa: BLE001
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
