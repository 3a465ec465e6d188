"""Host side of the attention operators: refusals before any device is touched, and the bucket map."""
import ctypes
import math

import pytest
import torch

from dl_cuda_b200 import capi, ops

FAKE = 0x1000  # never dereferenced: every call below is refused on the host


def block(**changes):
    h = capi.Heads(FAKE, 4096, 64, 16)
    a = capi.Attn(batch=2, heads=4, kv_heads=2, q_len=8, kv_len=8, head_dim=16, dtype=capi.F32, causal=0, scale=0.25,
                  cap=0.0, buckets=8, max_distance=16, q=h, k=h, v=h, o=h)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


BAD = [
    (dict(batch=-1), capi.ERR_INVALID_ARG), (dict(heads=0), capi.ERR_INVALID_ARG), (dict(heads=5), capi.ERR_INVALID_ARG),
    (dict(kv_heads=0), capi.ERR_INVALID_ARG), (dict(q_len=-1), capi.ERR_INVALID_ARG), (dict(head_dim=0), capi.ERR_INVALID_ARG),
    (dict(head_dim=129), capi.ERR_UNSUPPORTED), (dict(dtype=2), capi.ERR_INVALID_ARG), (dict(causal=2), capi.ERR_INVALID_ARG),
    (dict(scale=math.nan), capi.ERR_INVALID_ARG), (dict(scale=math.inf), capi.ERR_INVALID_ARG),
    (dict(cap=-1.0), capi.ERR_INVALID_ARG), (dict(cap=math.inf), capi.ERR_INVALID_ARG),
    (dict(q_docs=FAKE), capi.ERR_INVALID_ARG), (dict(kv_docs=FAKE), capi.ERR_INVALID_ARG),
    (dict(table=FAKE), capi.ERR_INVALID_ARG), (dict(table=FAKE, bucket_of=FAKE, buckets=0), capi.ERR_INVALID_ARG),
    (dict(table=FAKE, bucket_of=FAKE, buckets=65), capi.ERR_UNSUPPORTED),
    (dict(table=FAKE, bucket_of=FAKE, max_distance=1025), capi.ERR_UNSUPPORTED),
    (dict(q=capi.Heads(None, 0, 0, 0)), capi.ERR_INVALID_ARG), (dict(k=capi.Heads(FAKE, -1, 64, 16)), capi.ERR_INVALID_ARG),
    (dict(kv_len=(1 << 29) + 1), capi.ERR_UNSUPPORTED),
    (dict(batch=1 << 20, heads=1 << 10, kv_heads=1 << 10, q_len=1 << 12), capi.ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("changes,status", BAD)
def test_forward_and_backward_refuse(changes, status):
    lib = capi.lib()
    a = block(lse=FAKE, **changes)
    h = capi.Heads(FAKE, 4096, 64, 16)
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
    assert lib.dlb_attn_fwd(ctypes.byref(a), FAKE, 1 << 30, None) == status
    assert b"attn_fwd" in lib.dlb_last_error()
    assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), FAKE, 1 << 30, None) == status
    assert lib.dlb_attn_fwd_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.dlb_attn_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(g)) == 0


def test_null_blocks_and_overlapping_outputs():
    lib = capi.lib()
    assert lib.dlb_attn_fwd(None, None, 0, None) == capi.ERR_INVALID_ARG
    assert lib.dlb_attn_bwd(None, None, None, 0, None) == capi.ERR_INVALID_ARG
    a = block(lse=FAKE)
    assert lib.dlb_attn_bwd(ctypes.byref(a), None, FAKE, 1 << 30, None) == capi.ERR_INVALID_ARG
    assert lib.dlb_attn_fwd(ctypes.byref(block(o=capi.Heads(FAKE, 0, 64, 16))), FAKE, 1 << 30, None) == capi.ERR_INVALID_ARG
    h, flat = capi.Heads(FAKE, 4096, 64, 16), capi.Heads(FAKE, 4096, 64, 0)
    for name in ("dq", "dk", "dv"):
        g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
        setattr(g, name, flat)
        assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), FAKE, 1 << 30, None) == capi.ERR_INVALID_ARG
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h, dtable=FAKE)
    assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), FAKE, 1 << 30, None) == capi.ERR_INVALID_ARG  # no table
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
    assert lib.dlb_attn_bwd(ctypes.byref(block()), ctypes.byref(g), FAKE, 1 << 30, None) == capi.ERR_INVALID_ARG  # no lse


@pytest.mark.parametrize("dtype,off", [(capi.F32, 1), (capi.F32, 2), (capi.BF16, 1)])
def test_addresses_between_elements(dtype, off):
    """They would fault on the GPU; the host refuses them."""
    lib = capi.lib()
    size = 4 if dtype == capi.F32 else 2
    need = 1 << 30
    h, bad = capi.Heads(FAKE, 4096, 64, 16), capi.Heads(FAKE + off, 4096, 64, 16)
    for name in ("q", "k", "v", "o"):
        a = block(dtype=dtype, lse=FAKE, **{name: bad})
        assert lib.dlb_attn_fwd(ctypes.byref(a), FAKE, need, None) == capi.ERR_INVALID_ARG, name
        assert name.encode() in lib.dlb_last_error()
    for name in ("dout", "dq", "dk", "dv"):
        g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
        setattr(g, name, bad)
        assert lib.dlb_attn_bwd(ctypes.byref(block(dtype=dtype, lse=FAKE)), ctypes.byref(g), FAKE, need, None) == capi.ERR_INVALID_ARG, name
    pair = dict(table=FAKE, bucket_of=FAKE)
    for extra in (dict(kv_lens=FAKE + off), dict(q_start=FAKE + off), dict(prefix=FAKE + off), dict(q_docs=FAKE, kv_docs=FAKE + off),
                  dict(q_docs=FAKE + off, kv_docs=FAKE), dict(slopes=FAKE + off), dict(pair, table=FAKE + off),
                  dict(pair, bucket_of=FAKE + off), dict(lse=FAKE + off)):
        assert lib.dlb_attn_fwd(ctypes.byref(block(dtype=dtype, **extra)), FAKE, need, None) == capi.ERR_INVALID_ARG, extra
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h, dtable=FAKE + off)
    assert lib.dlb_attn_bwd(ctypes.byref(block(dtype=dtype, lse=FAKE, **pair)), ctypes.byref(g), FAKE, need, None) == capi.ERR_INVALID_ARG

    def bias(scores=FAKE, table=FAKE, of=FAKE, out=FAKE):
        return lib.dlb_rel_bias_fwd(scores, table, of, out, 1, 2, 3, 4, 0, 8, 16, dtype, None)

    def gradient(scores=FAKE, of=FAKE, out=FAKE):
        return lib.dlb_rel_bias_bwd(scores, of, out, FAKE, need, 1, 2, 3, 4, 0, 8, 16, dtype, None)

    for call in (bias, gradient):
        assert call(scores=FAKE + off) == call(of=FAKE + off) == call(out=FAKE + off) == capi.ERR_INVALID_ARG
    assert bias(table=FAKE + size // 2) == capi.ERR_INVALID_ARG


def test_documents_of_an_empty_side():
    """The address of an array without elements says nothing: an empty tensor's is NULL."""
    lib = capi.lib()
    h = capi.Heads(FAKE, 4096, 64, 16)
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
    for docs in (dict(q_docs=FAKE), dict(kv_docs=FAKE), dict(q_docs=FAKE, kv_docs=FAKE)):
        assert lib.dlb_attn_fwd(ctypes.byref(block(q_len=0, **docs)), None, 0, None) == capi.OK
        assert lib.dlb_attn_fwd(ctypes.byref(block(batch=0, **docs)), None, 0, None) == capi.OK
        # refused for the workspace alone, not for the documents
        a = block(kv_len=0, lse=FAKE, **docs)
        assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), None, 0, None) == capi.ERR_WORKSPACE
        assert lib.dlb_attn_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(g)) > 0


def test_workspace_is_asked_for():
    lib = capi.lib()
    a = block(lse=FAKE)
    h = capi.Heads(FAKE, 4096, 64, 16)
    g = capi.AttnGrad(dout=h, dq=h, dk=h, dv=h)
    need = lib.dlb_attn_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(g))
    assert need >= 2 * 4 * 8 * 8  # two floats per (batch, head, query)
    assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), FAKE, need - 1, None) == capi.ERR_WORKSPACE
    assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), None, need, None) == capi.ERR_WORKSPACE
    assert lib.dlb_attn_bwd(ctypes.byref(a), ctypes.byref(g), FAKE + 8, need, None) == capi.ERR_WORKSPACE
    long = block(q_len=1, kv_len=1 << 16)
    need = lib.dlb_attn_fwd_workspace_bytes(ctypes.byref(long))
    assert need > 0
    assert lib.dlb_attn_fwd(ctypes.byref(long), FAKE, need - 1, None) == capi.ERR_WORKSPACE
    assert lib.dlb_attn_fwd(ctypes.byref(block(batch=0)), None, 0, None) == capi.OK
    assert lib.dlb_attn_fwd(ctypes.byref(block(q_len=0)), None, 0, None) == capi.OK


def test_bias_matrix_refusals():
    lib = capi.lib()
    fwd = lambda *shape, dtype=0: lib.dlb_rel_bias_fwd(FAKE, FAKE, FAKE, FAKE, *shape, dtype, None)  # noqa: E731
    assert fwd(1, 2, -3, 4, 0, 8, 16) == capi.ERR_INVALID_ARG
    assert fwd(1, 2, 3, 4, 0, 0, 16) == capi.ERR_INVALID_ARG
    assert fwd(1, 2, 3, 4, 0, 65, 16) == capi.ERR_UNSUPPORTED
    assert fwd(1, 2, 3, 4, 0, 8, 1025) == capi.ERR_UNSUPPORTED
    assert fwd(1, 2, 3, 4, 0, 8, 16, dtype=7) == capi.ERR_INVALID_ARG
    assert fwd(1 << 12, 1 << 12, 1 << 8, 4, 0, 8, 16) == capi.ERR_UNSUPPORTED
    assert lib.dlb_rel_bias_fwd(None, None, None, None, 1, 2, 3, 4, 0, 8, 16, 0, None) == capi.ERR_INVALID_ARG
    assert lib.dlb_rel_bias_fwd(None, None, None, None, 0, 2, 3, 4, 0, 8, 16, 0, None) == capi.OK
    need = lib.dlb_rel_bias_bwd_workspace_bytes(1, 2, 3, 4, 8)
    assert need >= 2 * 8 * 4
    assert lib.dlb_rel_bias_bwd(FAKE, FAKE, FAKE, FAKE, need - 1, 1, 2, 3, 4, 0, 8, 16, 0, None) == capi.ERR_WORKSPACE
    assert lib.dlb_rel_bias_bwd(None, FAKE, FAKE, FAKE, need, 1, 2, 3, 4, 0, 8, 16, 0, None) == capi.ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 16)
    with pytest.raises(ValueError):
        ops.attn_fwd(x, x, x)
    with pytest.raises(ValueError):
        ops.attn_bwd(x, x, x, x, x, torch.zeros(1, 2, 4))
    with pytest.raises(ValueError):
        ops.rel_bias_fwd(torch.zeros(2, 8), torch.zeros(5, dtype=torch.int32), shape=(1, 2, 3, 4))
    with pytest.raises(ValueError):
        ops.rel_bias_bwd(torch.zeros(1, 2, 3, 4), torch.zeros(5, dtype=torch.int32), 8)


def exact_bucket(distance, each, top):
    """Bucket of a distance >= 0 by comparing whole numbers: no logarithm, so no rounding at a border."""
    own = each // 2
    if distance < own:
        return distance
    wide, k = each - own, 0
    while k + 1 < wide and distance ** wide * own ** (k + 1) >= top ** (k + 1) * own ** wide:
        k += 1
    return own + k


@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("buckets,top", [(32, 128), (16, 64), (8, 128), (32, 100), (4, 20), (64, 1024), (2, 8), (12, 31), (64, 37)])
def test_bucket_map(buckets, top, both):
    each = buckets // 2 if both else buckets
    if each // 2 < 1:
        with pytest.raises(capi.DlbError):
            ops.rel_bucket_map(buckets, top, both)
        return
    got = ops.rel_bucket_map(buckets, top, both).tolist()
    assert len(got) == 2 * top + 1
    for rel in range(-top, top + 1):
        if both:
            want = exact_bucket(-rel, each, top) if rel <= 0 else each + exact_bucket(rel, each, top)
        else:
            want = exact_bucket(max(-rel, 0), each, top)
        assert got[rel + top] == want, rel


def test_bucket_map_refusals():
    for buckets, top, both in ((0, 10, True), (7, 10, True), (32, 4, False), (66, 100, False), (32, 2000, True), (1, 5, False)):
        with pytest.raises(capi.DlbError):
            ops.rel_bucket_map(buckets, top, both)


@pytest.mark.parametrize("private", [True, False])
def test_stream_with_and_without_the_private_call(monkeypatch, private):
    """The address of the current stream also comes from torch's public interface alone."""
    class Stream:
        def __init__(self, device):
            self.cuda_stream = 100 + device

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    if private:
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 200 + device, raising=False)
    else:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    first = 200 if private else 100
    assert capi.current_stream() == first + 3 and capi.current_stream(1) == first + 1
