"""The native launch path of decoding over a cache (tree attention, key weights, beams, reordering, eviction) takes
the plain calls and gives bit for bit what the wrappers' own code gives."""
import pytest
import torch

from w8a8 import _lib, attention, cache, ops

DEV = "cuda"


def test_declines_host_tensors():
    n = _lib.launch_module()
    assert n is not None
    b, f = torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 2)
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    assert n.decode_tree(b, b, b, i32, 0, 0, 1.0) is None
    assert n.add_key_weights(b, b, f, f, 0, 0, 1.0) is None
    assert n.beam_select(f, f[0], 1) is None
    assert n.reorder([b], i64, 0) is None
    assert n.evict(b, b, f, f.int(), 2, 1, 0) is None
    for name in ("decode_tree", "add_key_weights", "beam_select", "reorder", "evict"):
        assert getattr(n, name)(None) is None


@pytest.fixture
def both(monkeypatch):
    """Runs f through the native path, which must take it, and through the wrappers' own code."""
    native = _lib.launch_module()

    def run(name, f):
        taken = []

        class Spy:
            def __getattr__(self, x):
                def call(*a):
                    r = getattr(native, x)(*a)
                    taken.append((x, r is not None))
                    return r
                return call
        out = []
        for way in (Spy(), None):
            for m in (attention, cache, ops):
                monkeypatch.setattr(m, "_native", way)
            out.append(f())
        assert (name, True) in taken, taken
        flat = lambda r: [r] if isinstance(r, torch.Tensor) else list(r)
        for x, y in zip(flat(out[0]), flat(out[1])):
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)
    return run


@pytest.mark.gpu
def test_the_same_results(both):
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(8, 6, 256, generator=g, device=DEV).bfloat16()
    kv = torch.randn(2, 3, 400, 256, generator=g, device=DEV).bfloat16()
    k, v = kv[0, 1:], kv[1, :2]
    parents = torch.tensor([-1, 0, 0, 1, 3, 3, 9], dtype=torch.int32, device=DEV)
    pos = torch.tensor([300], dtype=torch.int32, device=DEV)
    for past in (0, 300, pos):
        for window in (0, 128):
            both("decode_tree", lambda: attention.decode_tree(q, k, v, parents, past, window, 0.5))
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    both("decode_tree", lambda: attention.decode_tree(qt, k.transpose(0, 1).contiguous().transpose(0, 1), v, parents, 100))
    lse = torch.full((8, 6), 7.0, device=DEV)
    for args in ((q, k, lse, 300), (q[:, 0], k, lse[:, 0].contiguous(), 399), (q[:, 0], k, lse[:, :1], 5), (q[:, :1], k, lse[:, :1], pos)):
        both("add_key_weights", lambda: attention.add_key_weights(args[0], args[1], args[2], torch.ones(2, 400, device=DEV), args[3], 64))
    for x in (torch.randn(3, 5, 1000, generator=g, device=DEV), torch.randn(5, 999, generator=g, device=DEV).bfloat16()):
        s = torch.randn(x.shape[:-1], generator=g, device=DEV)
        both("beam_select", lambda: ops.beam_select(x, s, 7))
    both("beam_select", lambda: ops.beam_select(x[1:4, 3:], s[1:4], 7))
    t = torch.randn(4, 2, 50, 64, generator=g, device=DEV)

    def reorder(make, index, dim=0):
        c = t.clone()
        cache.reorder(make(c), index, dim)
        return c
    index = torch.tensor([3, 0, 0, 1], device=DEV)
    both("reorder", lambda: reorder(lambda c: c, index))
    both("reorder", lambda: reorder(lambda c: [c[:, :, :20], c[:, :, 20:31]], index))
    both("reorder", lambda: reorder(lambda c: (c[0], c[1]), index, 1))
    both("reorder", lambda: reorder(lambda c: c[0], torch.tensor([[4, 2, 9], [8, 8, 1]], device=DEV), -2))

    def evict(view):
        a, b = view(kv[0].clone()), view(kv[1].clone())
        return (*cache.evict(a, b, w, p, 350, 100, 20), a, b)
    w, p = torch.rand(3, 400, generator=g, device=DEV), torch.arange(400, device=DEV, dtype=torch.int32).repeat(3, 1)
    both("evict", lambda: evict(lambda x: x))
    w, p = w[:1], p[:1]
    both("evict", lambda: evict(lambda x: x[1:2]))


@pytest.mark.gpu
def test_what_the_wrapper_refuses_stays_refused():
    q = torch.zeros(8, 2, 128, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 50, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        attention.decode_tree(q, k, k, torch.zeros(1, dtype=torch.int32, device=DEV), 0)
    with pytest.raises(_lib.W8A8Error):
        attention.decode_tree(q, k, k, torch.zeros(2, dtype=torch.int32, device=DEV), 0, 0, float("nan"))
    with pytest.raises(_lib.W8A8Error):
        attention.add_key_weights(q, k, torch.zeros(8, 2, device=DEV), torch.zeros(1, 50, device=DEV), 0, 0, 0.0)
    with pytest.raises(ValueError):
        cache.reorder([k, k[0]], torch.zeros(1, dtype=torch.int64, device=DEV))
