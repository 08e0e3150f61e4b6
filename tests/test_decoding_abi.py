"""The entry points of decoding over a cache (tree attention, key weights, eviction, reordering, beams) refuse bad
arguments on the host, with a status and a message, before anything is launched (no GPU needed)."""
import ctypes

import pytest

from w8a8 import _lib

F = ctypes.c_void_p(0x100000)     # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x100002)


def status(name, args):
    L = _lib.lib()
    rc = getattr(L, name)(*args.values())
    return rc, L.w8a8_last_error().decode()


def refused(name, ok, changes):
    for change, want, word in changes:
        assert set(change) <= set(ok), change
        rc, msg = status(name, {**ok, **change})
        assert rc == want and word in msg, (change, rc, msg)


EINVAL, EALIGN, ENOTSUP = _lib.W8A8_EINVAL, _lib.W8A8_EALIGN, _lib.W8A8_ENOTSUP
BIG = 1 << 40


def test_tree():
    ok = dict(q=F, qhs=1024, qrs=256, k=F, khs=25600, krs=256, v=F, vhs=25600, vrs=256, H=8, KV=2, N=4, M=6, Tk=100, D=256,
              parents=F, n_past=94, past_dev=None, window=0, scale=1.0, o=F, ohs=1024, ors=256, lse=None, ws=F, wsb=BIG,
              stream=None)
    refused("w8a8_attention_tree_bf16", ok, [
        (dict(D=64), ENOTSUP, "head_dim"), (dict(M=129, Tk=1000), ENOTSUP, "nodes"), (dict(N=7), EINVAL, "N=7"),
        (dict(N=0), EINVAL, "N=0"), (dict(H=7), EINVAL, "H=7"), (dict(KV=0), EINVAL, "KV=0"), (dict(n_past=95), EINVAL, "n_past"),
        (dict(n_past=-1), EINVAL, "n_past"), (dict(n_past=3, past_dev=F), EINVAL, "n_past"), (dict(window=-1), EINVAL, "window"),
        (dict(scale=0.0), EINVAL, "scale"), (dict(scale=float("nan")), EINVAL, "scale"), (dict(q=None), EINVAL, "null"),
        (dict(parents=None), EINVAL, "null"), (dict(ws=None), EINVAL, "workspace"), (dict(wsb=15), EINVAL, "workspace"),
        (dict(krs=248), EINVAL, "strides"), (dict(vrs=-256), EINVAL, "strides"), (dict(qhs=-8), EINVAL, "strides"),
        (dict(krs=257), EALIGN, "strides"), (dict(ohs=1020), EALIGN, "strides"), (dict(k=ODD), EALIGN, "aligned"),
        (dict(parents=ODD), EALIGN, "aligned"), (dict(krs=1 << 30), ENOTSUP, "32-bit"),
    ])
    L = _lib.lib()
    size = L.w8a8_attention_tree_workspace_bytes
    assert size(8, 1, 8, 8, 8, 512, 0, 0) == 0 and size(8, 1, 8, 8, 5000, 512, 4000, 0) > 0
    assert size(8, 1, 8, 8, 5000, 512, -1, 0) >= size(8, 1, 8, 8, 5000, 512, 4000, 0)
    for bad in ((8, 3, 8, 8, 100, 512, 0, 0), (8, 1, 9, 8, 100, 512, 0, 0), (8, 1, 8, 8, 100, 96, 0, 0), (8, 1, 8, 8, 100, 512, 93, 0),
                (8, 1, 8, 8, 100, 512, -2, 0), (8, 1, 8, 8, 100, 512, 0, -1), (8, 1, 8, 8, 1 << 40, 512, 0, 0)):
        assert size(*bad) == -1, bad


def test_key_weights():
    ok = dict(q=F, qhs=1024, qrs=256, k=F, khs=25600, krs=256, lse=F, lhs=20, H=8, KV=2, Tq=20, Tk=100, D=256, q_start=80,
              start_dev=None, window=0, scale=1.0, w=F, whs=100, ws=F, wsb=BIG, stream=None)
    refused("w8a8_attention_key_weights", ok, [
        (dict(D=96), ENOTSUP, "head_dim"), (dict(H=9), EINVAL, "H=9"), (dict(Tq=0), EINVAL, "Tq=0"), (dict(Tk=19), EINVAL, "Tk=19"),
        (dict(q_start=81), EINVAL, "q_start"), (dict(q_start=-1), EINVAL, "q_start"), (dict(q_start=-1, start_dev=F), ENOTSUP, "rows"),
        (dict(window=-3), EINVAL, "window"), (dict(scale=float("inf")), EINVAL, "scale"), (dict(lse=None), EINVAL, "null"),
        (dict(krs=128), EINVAL, "strides"), (dict(qrs=260), EALIGN, "strides"), (dict(lhs=19), EINVAL, "lse"),
        (dict(whs=99), EINVAL, "weights"), (dict(q=ODD), EALIGN, "aligned"), (dict(w=ODD), EALIGN, "aligned"),
        (dict(krs=1 << 31), ENOTSUP, "stride"),
        (dict(H=1 << 16, KV=1 << 16), EINVAL, "KV=65536"),                                    # past a launch's second dimension
    ])
    size = _lib.lib().w8a8_attention_key_weights_workspace_bytes
    assert size(8, 1, 1, 5000, 512, 4999, 0) == 0 and size(8, 1, 1, 5000, 512, -1, 0) == 0
    assert size(8, 1, 3658, 3658, 512, 0, 0) > 0
    for bad in ((8, 3, 1, 10, 512, 0, 0), (8, 1, 11, 10, 512, 0, 0), (8, 1, 5, 10, 512, 6, 0), (8, 1, 5, 10, 512, -1, 0),
                (8, 1, 1, 10, 64, 0, 0), (8, 1, 1, 10, 512, 0, -1)):
        assert size(*bad) == -1, bad


def test_evict():
    ok = dict(k=F, kh=25600, kr=256, v=F, vh=25600, vr=256, row=256, KV=2, n=100, w=F, whs=100, pos=F, phs=100, budget=40, recent=8,
              kept=F, khs=40, wo=F, wos=40, po=F, pos_os=40, ws=F, wsb=BIG, stream=None)
    refused("w8a8_evict", ok, [
        (dict(budget=0), EINVAL, "budget"), (dict(budget=101), EINVAL, "budget"), (dict(recent=41), EINVAL, "recent"),
        (dict(recent=-1), EINVAL, "recent"), (dict(n=0), EINVAL, "n=0"), (dict(KV=0), EINVAL, "KV=0"), (dict(w=None), EINVAL, "null"),
        (dict(wsb=7), EINVAL, "workspace"), (dict(row=8), EINVAL, "rows of"), (dict(kr=240), EINVAL, "strides"), (dict(vh=-16), EINVAL, "strides"),
        (dict(kr=264), EALIGN, "16 bytes"), (dict(row=248), EALIGN, "16 bytes"), (dict(v=ODD), EALIGN, "16 bytes"),
        (dict(whs=99), EINVAL, "weights"), (dict(khs=39), EINVAL, "outputs"), (dict(pos=ODD), EALIGN, "4-byte"),
    ])
    size = _lib.lib().w8a8_evict_workspace_bytes
    assert 0 < size(2, 100, 100) < size(2, 100, 40) < size(4, 100, 40)
    assert size(1, 0, 1) == size(1, 10, 11) == size(0, 10, 5) == size(1, 1 << 40, 5) == -1


def test_reorder():
    def rows(**change):
        r = dict(data=0x100000, outer_stride=1 << 20, axis_stride=4096, run_stride=0, runs=1, run_bytes=4096)
        return (_lib.Rows * 1)(_lib.Rows(*{**r, **change}.values()))
    ok = dict(tensors=rows(), count=1, index=F, stride=0, n=4, size=8, outer=1, stream=None)
    refused("w8a8_reorder_rows", ok, [
        (dict(count=-1), EINVAL, "count"), (dict(n=9), ENOTSUP, "rows"), (dict(n=65, size=100), ENOTSUP, "at most 64"), (dict(size=0), EINVAL, "size"),
        (dict(outer=0), EINVAL, "outer"), (dict(tensors=None), EINVAL, "null"), (dict(index=None), EINVAL, "null"), (dict(index=ODD), EALIGN, "index"),
        (dict(outer=2, stride=3), EINVAL, "stride"), (dict(tensors=rows(axis_stride=4095)), EINVAL, "overlap"),
        (dict(tensors=rows(axis_stride=-4096)), EINVAL, "overlap"), (dict(tensors=rows(outer_stride=0), outer=2), EINVAL, "overlap"),
        (dict(tensors=rows(runs=2, run_stride=100)), EINVAL, "overlap"), (dict(tensors=rows(data=None)), EINVAL, "tensor 0"),
        (dict(tensors=rows(runs=-1)), EINVAL, "tensor 0"),
    ])
    twice = (_lib.Rows * 3)(rows()[0], rows(data=0x900000)[0], rows()[0])
    refused("w8a8_reorder_rows", ok, [(dict(tensors=twice, count=3), EINVAL, "0 and 2 are the same memory")])
    assert status("w8a8_reorder_rows", {**ok, "count": 0})[0] == 0
    assert status("w8a8_reorder_rows", {**ok, "n": 0})[0] == 0
    assert status("w8a8_reorder_rows", {**ok, "tensors": rows(runs=0)})[0] == 0


def test_beams():
    ok = dict(x=F, f32=1, gs=400, rs=100, scores=F, ss=4, B=2, nb=4, V=100, k=8, os=F, ob=F, ot=F, ws=F, wsb=BIG, stream=None)
    refused("w8a8_beam_select", ok, [
        (dict(k=0), EINVAL, "k=0"), (dict(k=65), EINVAL, "k=65"), (dict(nb=257, ss=257), EINVAL, "nb=257"), (dict(V=1), EINVAL, "V=1"),
        (dict(V=0), EINVAL, "V=0"), (dict(B=0), EINVAL, "B=0"), (dict(x=None), EINVAL, "null"), (dict(ot=None), EINVAL, "null"),
        (dict(rs=99), EINVAL, "strides"), (dict(ss=3), EINVAL, "strides"), (dict(wsb=8), EINVAL, "workspace"), (dict(x=ODD), EALIGN, "aligned"),
        (dict(ob=ODD), EALIGN, "aligned"), (dict(B=1 << 30), EINVAL, "B="),
        (dict(B=1 << 22), EINVAL, "B="), (dict(B=70000, nb=256, ss=256), EINVAL, "B=70000"),   # launches past 2^32 threads
    ])
    size = _lib.lib().w8a8_beam_select_workspace_bytes
    assert size(1, 4, 262144, 8) > 0 and size(1, 4, 262144, 65) == -1 and size(1, 2, 3, 7) == -1


def test_python_layer_refuses_cpu_tensors():
    import torch

    from w8a8 import attention, cache, ops
    b = torch.zeros(8, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        attention.decode_tree(b, b, b, torch.zeros(4, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="GPU tensor"):
        attention.add_key_weights(b, b, torch.zeros(8, 4), torch.zeros(8, 4))
    with pytest.raises(ValueError, match="GPU tensor"):
        cache.evict(b, b, torch.zeros(8, 4), torch.zeros(8, 4, dtype=torch.int32), 4, 2)
    with pytest.raises(ValueError, match="on the GPU"):
        cache.reorder(b, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="one GPU"):
        ops.beam_select(torch.zeros(2, 9), torch.zeros(2), 2)
