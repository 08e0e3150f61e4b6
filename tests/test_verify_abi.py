"""ops.verify_drafts' C entry: calls that are too large for a launch are refused on the host (no GPU needed)."""
import ctypes

from w8a8 import _lib

F = ctypes.c_void_p(0x100000)     # never dereferenced: validation fails first
ok = dict(logits=F, draft=F, f32=1, gs=64, rs=8, dgs=64, drs=8, tok=F, ts=4, u=F, us=5, parents=None, ps=0, lengths=None, B=2, N=4, V=8,
          temperature=1.0, accepted=F, path=F, next=F, ws=F, wsb=1 << 50, stream=None)


def test_a_launch_holds_fewer_than_2_32_threads():
    L = _lib.lib()
    size = L.w8a8_verify_drafts_workspace_bytes
    for B, N, V in ((1 << 22, 4, 1), (1 << 22, 3, 8), (1 << 17, 127, 1), (1 << 22, 0, 9000), (1 << 13, 0, (1 << 22) + 1)):
        assert size(B, N, V) == -1, (B, N, V)
        rc = L.w8a8_verify_drafts(*{**ok, "B": B, "N": N, "V": V, "rs": V, "drs": V, "draft": None}.values())
        assert rc == _lib.W8A8_EINVAL and f"B={B}" in L.w8a8_last_error().decode()
    # with draft logits the rows are more: 2^22 requests of 2 tokens are 12.6 million rows, and 8.4 of the draft
    assert size(1 << 22, 2, 1) > 0 and size((1 << 22) - 1, 3, 1) > 0
    rc = L.w8a8_verify_drafts(*{**ok, "B": 1 << 22, "N": 2, "V": 1, "rs": 1, "drs": 1}.values())
    assert rc == _lib.W8A8_EINVAL and "draft logits" in L.w8a8_last_error().decode()
