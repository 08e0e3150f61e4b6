"""The addresses of attention over the 8-bit block cache, walked on the host: the kernel's index arithmetic written out again,
for every row tile, over short, odd and long lengths, with windows and sinks (no GPU needed).  Every block that a row sees is
taken by exactly one part, every query once, and every access lies in its own array."""
import random

import numpy as np
import pytest

from w8a8 import _lib

BLK = 64
lib = _lib.lib


def layout(KV, capacity, D):
    """Element ranges of the cache's parts: (offset, bytes) of codes, ring and scales; and the whole."""
    up = lambda n: (n + 255) // 256 * 256
    blocks = (capacity + BLK - 1) // BLK
    codes, ring, scales = up(KV * blocks * BLK * D), KV * 2 * BLK * D * 2, up(KV * blocks * 4)
    return blocks, {"k": (0, codes), "v": (codes, codes), "kt": (2 * codes, ring), "vt": (2 * codes + ring, ring),
                    "ks": (2 * codes + 2 * ring, scales), "vs": (2 * codes + 2 * ring + scales, scales)}, 2 * (codes + ring + scales)


def row_tile(rows, D):
    return 1 if rows <= 16 else 2 if rows <= 32 else 4 if D >= 256 or rows <= 64 else 8


def parts_at_most(H, N, D, need):
    per = H * N * (D + 2) * 4
    assert need % per == 0
    return max(1, need // per)


def walk(H, KV, N, capacity, D, n, window, sinks, on_device):
    need = lib().w8a8_block_attention_workspace_bytes(H, KV, N, capacity, D, -1 if on_device else n, window, sinks)
    assert need >= 0
    G, rows = H // KV, N * (H // KV)
    nparts, rt = parts_at_most(H, N, D, need), row_tile(rows, D)
    R, groups = 16 * rt, 1 if rt == 1 else 2
    waves, ntiles = 4 * groups, (rows + R - 1) // R
    blocks, where, size = layout(KV, capacity, D)
    assert size == lib().w8a8_block_cache_bytes(KV, capacity, D)
    sinks = sinks if window else 0
    inside = lambda what, lo, hi: 0 <= lo and hi <= where[what][1]
    lane = np.arange(64)
    seen_rows = np.zeros((N, G), dtype=int)
    for tile in range(ntiles):
        r0, r1 = tile * R, min(tile * R + R, rows) - 1
        pmin, pmax = n - N + r0 // G, n - N + r1 // G
        wb = max(0, pmin - window + 1) // BLK if window else 0
        sb = (min(sinks, n) + BLK - 1) // BLK
        skip = max(0, wb - sb)
        nb = pmax // BLK + 1 - skip
        parts = min(nparts, nb)
        assert nb >= 1 and parts <= 512
        whole = n // BLK
        # the quotient by G in fp32
        first, odd = tile * R // G, tile * R - tile * R // G * G
        r = np.arange(R)
        x = ((odd + r).astype(np.float32) + np.float32(0.5)) * (np.float32(1.0) / np.float32(G))
        x = x.astype(np.int64)
        assert np.array_equal(x, (odd + r) // G)
        h, live = odd + r - x * G, tile * R + r < rows
        assert (h >= 0).all() and (h < G).all() and (first + x[live] >= 0).all() and (first + x[live] < N).all()
        np.add.at(seen_rows, (first + x[live], h[live]), 1)
        taken = []
        for part in range(parts):
            lo, hi = part * nb // parts, (part + 1) * nb // parts
            assert hi > lo
            ids = [i if i < sb else i + skip for i in range(lo, hi)]
            ring = ids[-1] >= whole
            assert all(b < whole for b in ids[:-1]) and (not ring or ids[-1] == whole)
            for b in ids[: len(ids) - ring]:
                taken.append(b)
                for g in (0, KV - 1):
                    base = (g * blocks + b) * BLK * D
                    k_last = base + 3 * 16 * D + 63 * 16 + (D // 64 - 1) * 1024 + 16
                    nv = D // 16 // waves
                    v_last = base + (waves - 1) * nv * 1024 + 63 * 16 + (nv - 1) * 1024 + 16
                    assert k_last == v_last == base + BLK * D
                    assert inside("k", base, k_last) and inside("v", base, v_last) and inside("ks", 4 * (g * blocks + b), 4 * (g * blocks + b) + 4)
            if ring:
                taken.append(whole)
                live_rows = n - whole * BLK
                assert 0 < live_rows < BLK and pmax >= whole * BLK
                for g in (0, KV - 1):
                    at = (g * 2 + (whole & 1)) * BLK * D
                    nkk, nv = D // 32, D // 16 // waves
                    k_end = at + (3 * nkk * 64 + 63) * 8 + (nkk - 1) * 512 + 8
                    v_end = at + ((waves - 1) * nv * 2 * 64 + 63) * 8 + (2 * (nv - 1) + 1) * 512 + 8
                    assert inside("kt", 2 * at, 2 * k_end) and inside("vt", 2 * at, 2 * v_end) and k_end == v_end == at + BLK * D
            if parts > 1:  # sums and references of rows in the workspace
                for g in (0, KV - 1):
                    at = (g * nparts + part) * rows + r[live] + tile * R
                    assert (at * D + D <= need // 4).all() and (4 * H * N * nparts * D + 8 * (at + 1) <= need).all()
                    assert (at < (g * nparts + part + 1) * rows).all()
        # the blocks that some row of the tile sees are among those taken, none twice
        assert len(set(taken)) == len(taken)
        for p in {pmin, pmax, (pmin + pmax) // 2}:
            near = range(max(0, p - window + 1) // BLK if window else 0, p // BLK + 1)
            far = range(0, (min(sinks, p + 1) + BLK - 1) // BLK)
            assert set(near) | set(far) <= set(taken)
        # queries in LDS: chunk c of row r at c ^ (r & 15), and the fragments that are read from there
        for d8 in (0, D // 8 - 1):
            assert ((r * D + 8 * (d8 ^ (r & 15)) + 8) <= R * D).all()
        lpr, rpi = D // 8, 64 // (D // 8)
        staged = np.concatenate([w * (R // waves) + i * rpi + lane // lpr for w in range(waves) for i in range(R // waves // rpi)])
        assert np.array_equal(np.bincount(staged, minlength=R), np.full(R, lpr))
        for k in range(D // 32):
            c = 8 * (k >> 1) + 2 * (lane >> 4) + (k & 1)
            assert (c < lpr).all()
    assert (seen_rows == 1).all()


SHAPES = [  # H, KV, D, N: every tile of rows for each head_dim
    (8, 1, 512, 1), (16, 1, 256, 1), (4, 4, 128, 1), (12, 4, 128, 5), (8, 1, 512, 3), (8, 1, 256, 4), (32, 8, 128, 7), (8, 1, 512, 5),
    (5, 5, 256, 17), (8, 2, 512, 33), (24, 2, 128, 5), (3, 1, 128, 200), (20, 1, 256, 9), (24, 2, 128, 100), (8, 1, 256, 509), (200, 1, 128, 3), (7, 1, 128, 61),
]


@pytest.mark.parametrize("H,KV,D,N", SHAPES)
def test_in_range(H, KV, D, N):
    rng = random.Random(H * 1000 + D + N)
    lengths = {N, N + 1, max(N, 63), max(N, 64), max(N, 65), max(N, 127), N + 700, N + 4095, 8191, 32749}
    for n in sorted(lengths):
        for window, sinks in ((0, 0), (1, 0), (1, 1), (100, 3), (512, 64), (4096, 65), (rng.randint(1, 5000), rng.randint(0, 6000))):
            if n > 5000 and N > 100 and window not in (0, 4096):
                continue
            walk(H, KV, N, n, D, n, window, sinks, False)
            walk(H, KV, N, n + 100, D, n, window, sinks, True)
            if n < 1000:
                walk(H, KV, N, 40000, D, n, window, sinks, True)


def test_ring_order():
    """Every value of a block's ring slot has a place of its own, for keys and for values."""
    for D in (128, 256, 512):
        r, d = np.meshgrid(np.arange(BLK), np.arange(D), indexing="ij")
        key = (((r >> 4) * (D >> 5) + 2 * (d >> 6) + ((d >> 3) & 1)) * 64 + 16 * ((d >> 4) & 3) + (r & 15)) * 8 + (d & 7)
        value = (((d >> 4) * 2 + (r >> 5)) * 64 + 16 * ((r >> 2) & 3) + (d & 15)) * 8 + 4 * ((r >> 4) & 1) + (r & 3)
        for at in (key, value):
            assert np.array_equal(np.sort(at.ravel()), np.arange(BLK * D))
