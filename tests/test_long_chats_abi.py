"""The entry points of long conversations (verification of drafted tokens, attention with sinks, the 8-bit block cache)
refuse bad arguments on the host, with a status and a message, before anything is launched (no GPU needed)."""
import ctypes

import torch

from w8a8 import _lib

F = ctypes.c_void_p(0x100000)     # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x100001)
EINVAL, EALIGN, ENOTSUP = _lib.W8A8_EINVAL, _lib.W8A8_EALIGN, _lib.W8A8_ENOTSUP
BIG = 1 << 50
NAN, INF = float("nan"), float("inf")


def refused(name, ok, changes):
    L = _lib.lib()
    for change, want, word in changes:
        assert set(change) <= set(ok), change
        rc = getattr(L, name)(*{**ok, **change}.values())
        msg = L.w8a8_last_error().decode()
        assert rc == want and word in msg, (change, rc, msg)


def test_verify_drafts():
    ok = dict(logits=F, draft=F, f32=1, gs=5000, rs=1000, dgs=4000, drs=1000, tok=F, ts=4, u=F, us=5, parents=None, ps=0, lengths=None,
              B=2, N=4, V=1000, temperature=1.0, accepted=F, path=F, next=F, ws=F, wsb=BIG, stream=None)
    refused("w8a8_verify_drafts", ok, [
        (dict(N=129), ENOTSUP, "129"), (dict(N=-1), EINVAL, "N=-1"), (dict(B=0), EINVAL, "B=0"), (dict(V=0), EINVAL, "V=0"),
        (dict(V=1 << 30), EINVAL, "V="), (dict(B=1 << 40), EINVAL, "B="), (dict(temperature=0.0), EINVAL, "temperature"),
        (dict(temperature=-1.0), EINVAL, "temperature"), (dict(temperature=NAN), EINVAL, "temperature"), (dict(temperature=INF), EINVAL, "temperature"),
        (dict(temperature=1e-320), EINVAL, "temperature"), (dict(parents=F), ENOTSUP, "tree"), (dict(logits=None), EINVAL, "null"),
        (dict(u=None), EINVAL, "null"), (dict(tok=None), EINVAL, "null"), (dict(path=None), EINVAL, "null"), (dict(next=None), EINVAL, "null"),
        (dict(rs=999), EINVAL, "strides"), (dict(drs=999), EINVAL, "strides"), (dict(gs=-1), EINVAL, "strides"), (dict(ts=-4), EINVAL, "strides"),
        (dict(ws=None), EINVAL, "workspace"), (dict(wsb=100), EINVAL, "workspace"), (dict(logits=ODD), EALIGN, "aligned"),
        (dict(tok=ODD), EALIGN, "aligned"), (dict(u=ODD), EALIGN, "aligned"), (dict(accepted=ODD), EALIGN, "aligned"), (dict(ws=ODD), EALIGN, "aligned"),
        (dict(lengths=ODD), EALIGN, "aligned"),
    ])
    size = _lib.lib().w8a8_verify_drafts_workspace_bytes
    assert 0 < size(1, 0, 1) < size(1, 4, 1000) < size(8, 8, 262144)
    for bad in ((0, 4, 100), (1, -1, 100), (1, 129, 100), (1, 4, 0), (1, 4, 1 << 30), (1 << 23, 4, 100)):
        assert size(*bad) == -1, bad


def test_sinks():
    ok = dict(q=F, qhs=5120, qrs=256, k=F, khs=25600, krs=256, v=F, vhs=25600, vrs=256, H=8, KV=2, Tq=20, Tk=100, D=256, start=80, dev=None,
              window=30, sinks=4, scale=1.0, o=F, ohs=5120, ors=256, lse=None, ws=F, wsb=BIG, stream=None)
    refused("w8a8_attention_sinks_bf16", ok, [
        (dict(D=64), ENOTSUP, "head_dim"), (dict(H=7), EINVAL, "H=7"), (dict(KV=0), EINVAL, "KV=0"), (dict(Tq=0), EINVAL, "Tq=0"),
        (dict(Tq=101), EINVAL, "Tq=101"), (dict(start=81), EINVAL, "q_start"), (dict(start=-1), EINVAL, "q_start"),
        (dict(start=3, dev=F), EINVAL, "q_start"), (dict(window=-1), EINVAL, "window"), (dict(sinks=-1), EINVAL, "sinks"),
        (dict(scale=0.0), EINVAL, "scale"), (dict(scale=NAN), EINVAL, "scale"), (dict(scale=INF), EINVAL, "scale"), (dict(q=None), EINVAL, "null"),
        (dict(v=None), EINVAL, "null"), (dict(o=None), EINVAL, "null"), (dict(krs=248), EINVAL, "strides"), (dict(vrs=-256), EINVAL, "strides"),
        (dict(qhs=-8), EINVAL, "strides"), (dict(ohs=8), EINVAL, "overlap"), (dict(krs=257), EALIGN, "strides"), (dict(ohs=1020), EALIGN, "strides"),
        (dict(k=ODD), EALIGN, "aligned"), (dict(dev=ODD, start=-1), EALIGN, "aligned"), (dict(krs=1 << 24), ENOTSUP, "apart"),
        (dict(Tk=1 << 40), EINVAL, "Tk="), (dict(H=1 << 20, Tq=100), EINVAL, "H="),
    ])
    L = _lib.lib()
    long = dict(Tk=100000, start=90000, Tq=1, window=0)
    need = L.w8a8_attention_sinks_workspace_bytes(8, 2, 1, 100000, 256, 90000, 0, 4)
    assert need > 0
    refused("w8a8_attention_sinks_bf16", {**ok, **long}, [(dict(ws=None), EINVAL, "workspace"), (dict(wsb=need - 1), EINVAL, "workspace")])
    size = L.w8a8_attention_sinks_workspace_bytes
    assert size(8, 1, 1, 10, 256, 9, 0, 0) == 0
    for bad in ((8, 3, 1, 10, 256, 0, 0, 0), (8, 1, 11, 10, 256, 0, 0, 0), (8, 1, 1, 10, 96, 0, 0, 0), (8, 1, 1, 10, 256, 10, 0, 0),
                (8, 1, 1, 10, 256, -2, 0, 0), (8, 1, 1, 10, 256, 0, -1, 0), (8, 1, 1, 10, 256, 0, 0, -1)):
        assert size(*bad) == -1, bad
        assert L.w8a8_attention_sinks_plan(*bad, None, None) == EINVAL


def test_block_cache():
    L = _lib.lib()
    size = L.w8a8_block_cache_bytes
    assert size(1, 64, 128) == size(1, 1, 128) < size(1, 65, 128)
    codes = 8 * 65536 * 128
    assert 2 * codes < size(8, 65536, 128) < 2 * codes * 1.01  # half of a bf16 cache and little more
    for bad in ((0, 64, 128), (1, 0, 128), (1, 64, 96), (1 << 17, 64, 128), (1, 1 << 40, 128)):
        assert size(*bad) == -1, bad
    ok = dict(cache=F, KV=2, capacity=100, D=256, e4m3=0, k=F, khs=25600, krs=256, v=F, vhs=25600, vrs=256, m=10, n=90, dev=None, stream=None)
    refused("w8a8_block_append", ok, [
        (dict(D=64), ENOTSUP, "head_dim"), (dict(KV=0), EINVAL, "KV=0"), (dict(capacity=0), EINVAL, "capacity"), (dict(cache=None), EINVAL, "null"),
        (dict(cache=ODD), EALIGN, "aligned"), (dict(n=91), EINVAL, "rows"), (dict(n=-1), EINVAL, "rows"), (dict(m=101), EINVAL, "rows"),
        (dict(m=-1), EINVAL, "rows"), (dict(n=5, dev=F), EINVAL, "rows"), (dict(k=None), EINVAL, "null"), (dict(v=None), EINVAL, "null"),
        (dict(krs=128), EINVAL, "strides"), (dict(vhs=-8), EINVAL, "strides"), (dict(krs=260), EALIGN, "strides"), (dict(k=ODD), EALIGN, "aligned"),
        (dict(dev=ODD, n=-1), EALIGN, "aligned"),
    ])
    assert L.w8a8_block_append(*{**ok, "m": 0, "k": None, "v": None}.values()) == _lib.W8A8_OK
    ok = dict(cache=F, KV=2, capacity=100, D=256, e4m3=0, start=5, n=50, k=F, v=F, stream=None)
    refused("w8a8_block_read", ok, [
        (dict(D=64), ENOTSUP, "head_dim"), (dict(start=-1), EINVAL, "rows"), (dict(start=51), EINVAL, "rows"), (dict(n=101), EINVAL, "rows"),
        (dict(k=None), EINVAL, "null"), (dict(v=ODD), EALIGN, "aligned"), (dict(cache=ODD), EALIGN, "aligned"),
    ])
    assert L.w8a8_block_read(*{**ok, "start": 50, "k": None}.values()) == _lib.W8A8_OK


def test_block_attention():
    ok = dict(q=F, qhs=5120, qrs=256, cache=F, H=8, KV=2, N=20, capacity=100, D=256, e4m3=0, n=90, dev=None, window=30, sinks=4, scale=1.0, o=F,
              ohs=5120, ors=256, lse=None, ws=F, wsb=BIG, stream=None)
    refused("w8a8_block_attention", ok, [
        (dict(D=64), ENOTSUP, "head_dim"), (dict(H=7), EINVAL, "H=7"), (dict(N=0), EINVAL, "N=0"), (dict(N=101), EINVAL, "N=101"),
        (dict(n=19), EINVAL, "n=19"), (dict(n=101), EINVAL, "n=101"), (dict(n=-1), EINVAL, "n=-1"), (dict(n=50, dev=F), EINVAL, "n=50"),
        (dict(window=-1), EINVAL, "window"), (dict(sinks=-1), EINVAL, "sinks"), (dict(scale=0.0), EINVAL, "scale"), (dict(scale=NAN), EINVAL, "scale"),
        (dict(q=None), EINVAL, "null"), (dict(cache=None), EINVAL, "null"), (dict(o=None), EINVAL, "null"), (dict(qrs=248), EINVAL, "strides"),
        (dict(ohs=8), EINVAL, "overlap"), (dict(qhs=5124), EALIGN, "strides"), (dict(cache=ODD), EALIGN, "aligned"), (dict(lse=ODD), EALIGN, "aligned"),
    ])
    L = _lib.lib()
    size = L.w8a8_block_attention_workspace_bytes
    need = size(8, 2, 1, 100000, 256, 90000, 0, 0)
    assert need > 0 and size(8, 2, 1, 100, 256, 50, 0, 0) == 0 and size(8, 2, 1, 100000, 256, -1, 0, 0) >= need
    refused("w8a8_block_attention", {**ok, "N": 1, "capacity": 100000, "n": 90000, "window": 0},
            [(dict(ws=None), EINVAL, "workspace"), (dict(wsb=need - 1), EINVAL, "workspace")])
    for bad in ((8, 3, 1, 10, 256, 9, 0, 0), (8, 1, 11, 10, 256, 10, 0, 0), (8, 1, 1, 10, 96, 9, 0, 0), (8, 1, 1, 10, 256, 11, 0, 0), (8, 1, 2, 10, 256, 1, 0, 0),
                (8, 1, 1, 10, 256, -2, 0, 0), (8, 1, 1, 10, 256, 9, -1, 0), (8, 1, 1, 10, 256, 9, 0, -1)):
        assert size(*bad) == -1, bad


def test_native_path_declines_host_tensors():
    n = _lib.launch_module()
    assert n is not None
    b, f = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(3, 8)
    i64 = torch.zeros(2, dtype=torch.int64)
    assert n.verify_drafts(f, i64, f[0, :3], None, None, None, 1.0) is None
    assert n.sink_attention(b, b, b, 0, 4, 1, 1.0) is None
    data = torch.zeros(1 << 20, dtype=torch.uint8)
    assert n.block_append(data, 4, 64, 128, 0, b, b, 0) is None
    assert n.block_read(data, 4, 64, 128, 0, 0, 2) is None
    assert n.block_attention(b, data, 4, 64, 128, 0, 2, 0, 0, 1.0) is None
    for name in ("verify_drafts", "sink_attention", "block_append", "block_read", "block_attention"):
        assert getattr(n, name)(None) is None
