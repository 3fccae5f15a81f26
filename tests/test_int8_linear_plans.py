"""Every way that int8.int8_linear can take: which one it is (h24_int8_linear_plan, no GPU), and its outputs against the
product in 64 bits, with the bounds of test_gpu_int8_linear.py.  The sizes are the smallest that reach a way with
odd edges: outputs that end inside a warp's 32, tokens that end inside a tile, rows on and off 16 bytes."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_gpu_int8_linear import _check, _inputs

ROWS, TILE, PAIR = 0, 1, 2
# (tokens, out, in): pairs of CTAs, by the tokens of a tile (32, 64, ... 256).
PAIRS = [(5, 38434, 32), (6, 37951, 25), (2330, 389, 3536), (2330, 389, 3528), (3399, 270, 3200), (3399, 270, 3197),
         (4080, 315, 3280), (3733, 280, 5465), (3132, 515, 2560), (3132, 515, 2546), (3965, 564, 1616),
         (3965, 564, 1615), (3491, 807, 960), (3491, 807, 946), (4078, 790, 1136), (4078, 790, 1129),
         (978, 12357, 4996), (324, 42497, 913)]
# Tiles whose sum is one CTA's, or that of 2, 4 or 8.
TILES = [(5, 25, 32), (5, 26, 24), (149, 5476, 2960), (149, 5476, 2957), (2884, 268, 2064), (2884, 268, 2055),
         (5, 25, 1424), (21, 25, 1427), (10, 25, 1968), (10, 25, 1961), (1000, 333, 48), (2000, 3000, 33), (300, 7001, 64)]
# Three and four tokens of a large layer: fewer than the box of a tile.
FEW = [(3, 50688, 1920), (4, 50688, 1920), (3, 13003, 2021), (4, 50687, 1921)]
# Weight rows by dp4a: one to four tokens, the three numbers of rows a warp, one pass over the tokens or more.
VECTORS = [(t, out, k) for t in (1, 2, 3, 4) for out in (101, 5003, 9475) for k in (1920, 1911)] + \
          [(t, 201, k) for t in (1, 2, 3, 4) for k in (9008, 9001, 20001)]


def _plan(lib, tokens, out, in_, dtype=0):
    p = (ctypes.c_int32 * 3)()
    assert lib.h24_int8_linear_plan(tokens, out, in_, dtype, p) == 0
    return tuple(p)


def test_the_sizes_reach_every_way(lib):
    for aligned in (True, False):
        pairs = [s for s in PAIRS if (s[2] % 16 == 0) == aligned]
        plans = [_plan(lib, *s, d) for s in pairs for d in (0, 1)]
        assert {p[0] for p in plans} == {PAIR} and {p[1] for p in plans} == set(range(32, 257, 32))
        assert all(s[1] % 32 and s[0] % _plan(lib, *s)[1] for s in pairs)
        tiles = [s for s in TILES if (s[2] % 16 == 0) == aligned]
        plans = [_plan(lib, *s) for s in tiles]
        assert {p[0] for p in plans} == {TILE} and {p[2] for p in plans} == {1, 2, 4, 8}
    assert all(_plan(lib, *s)[0] != ROWS and s[0] < _plan(lib, *s)[1] for s in FEW)
    assert all(_plan(lib, *s)[0] == ROWS for s in VECTORS)


def test_plan_refusals(lib):
    from pollux_b200 import _native as N
    p = (ctypes.c_int32 * 3)()
    for args in ((0, 8, 8, 0), (1, 0, 8, 0), (1, 8, -1, 0), (1, 8, 131001, 0), (1, 8, 8, 3), (1 << 31, 8, 8, 0)):
        assert lib.h24_int8_linear_plan(*args, p) == N.H24_ERR_INVALID
    assert lib.h24_int8_linear_plan(1, 8, 8, 0, None) == N.H24_ERR_INVALID
    assert _plan(lib, 5, 8, 0)[0] == TILE  # an empty sum never takes the pairs


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,out_f,in_f", PAIRS + TILES + FEW + VECTORS)
def test_matches_exact(lib, tokens, out_f, in_f):
    from pollux_b200 import int8
    q, scale, w, mu, b = _inputs(tokens, out_f, in_f, tokens + out_f + in_f)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        s = scale / max(1, in_f) ** 0.5 / 50 if dtype == torch.float16 else scale  # within fp16's range
        for bias in (None, b):
            _check(int8.int8_linear(q, s, w, mu, bias, dtype), q, s, w, mu, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,out_f,in_f", [PAIRS[1], PAIRS[5], PAIRS[16], TILES[2], TILES[5], FEW[2], VECTORS[3]])
def test_writes_its_outputs_alone(lib, tokens, out_f, in_f):
    """The memory around y keeps its values, and rows off 16 bytes give what aligned ones do."""
    from pollux_b200 import _native as N, int8
    q, scale, w, mu, b = _inputs(tokens, out_f, in_f, 17)
    want = int8.int8_linear(q, scale, w, mu, b)
    room = torch.full((tokens * out_f + 2048,), 12345.0, device="cuda")
    for at in (1024, 1025):
        room.fill_(12345.0)
        N.call("h24_int8_linear", q.data_ptr(), scale.data_ptr(), tokens, in_f, w.data_ptr(), mu.data_ptr(), out_f, in_f,
               b.data_ptr(), N.DTYPE_F32, room.data_ptr() + 4 * at, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(room[at:at + want.numel()].view_as(want), want)
        assert (room[:at] == 12345.0).all() and (room[at + want.numel():] == 12345.0).all()
