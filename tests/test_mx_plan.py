"""Which kernels an expert call on 4-bit weights takes, on the CPU: the height of its token
tiles, read off the workspace it asks for (the tile map has two numbers per tile)."""

from __future__ import annotations

import pytest
import torch

from reframework_amd import _capi
from reframework_amd.mx import padded

F32, BF16, F16 = 0, 1, 2


def _tile_rows(T, H, I, E, K, dtype):
    """The heights whose tile map, with some number of column parts, explains the bytes."""
    def up(n):
        return -(-n // 256) * 256
    R, Hp, Ip = T * K, padded(H), padded(I)
    active = min(R, E)
    blocks = 1 if R <= 1024 else -(-R // 256)
    fixed = sum(up(n) for n in (blocks * E * 4, (E + 1) * 4, R * 4, R * 4, T * Hp, T * Hp // 32,
                                R * Ip, R * Ip // 32))
    n = _capi.mx_workspace_bytes(T, H, I, E, K, dtype, torch.device("cpu"))
    found = set()
    for rows in (16, 64, 128, 256):
        tiles = up((2 + 2 * ((R + active * (rows - 1)) // rows)) * 4)
        ys = [up(s * R * H * 4) for s in (1, 2, 4, 8)] + [up(R * H * 2) + up(R * (Hp // 64))]
        if n - fixed - tiles in ys:
            found.add(rows)
    assert len(found) == 1, (found, T, H, I, E, K, dtype)
    return found.pop()


# Rows per expert and columns at which both sides were measured, and the faster height there
# (capi_mx.hip has the times). The choice goes by these alone; 256 experts make the tile
# maps of the heights differ by more than the workspace's alignment.
@pytest.mark.parametrize("H,I,rows,dtype,tile", [
    (4096, 14336, 8, BF16, 16), (4096, 14336, 14, BF16, 64), (2048, 1408, 12, BF16, 16),
    (2048, 1408, 14, BF16, 64), (2048, 8192, 10, BF16, 16), (1280, 3328, 12, F16, 16),
    (7168, 2048, 60, BF16, 256), (4096, 14336, 60, BF16, 64), (4096, 14336, 75, BF16, 256),
    (2048, 1408, 105, BF16, 64), (2048, 1408, 135, BF16, 256),
    (1280, 3328, 180, BF16, 64), (1280, 3328, 200, BF16, 256),
    (768, 1536, 180, BF16, 64), (768, 1536, 220, BF16, 64),
    (2048, 1408, 160, F16, 64), (2048, 1408, 230, F16, 128), (2048, 1408, 420, F32, 128),
])
def test_the_faster_height_is_taken(H, I, rows, dtype, tile):
    assert _tile_rows(64 * rows, H, I, 256, 4, dtype) == tile
