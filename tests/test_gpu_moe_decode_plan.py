"""A thread block whose plan of matrix rows does not fit: the launch says so instead of leaving rows out."""
import pytest
import torch

from test_gpu_moe_block import BF16, E4M3, on_device
from test_gpu_moe_decode import bank, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_plan_without_room_gives_up(kind):
    from kanjoos_b200 import _lib
    from kanjoos_b200.moe import MoeBlock
    L = _lib.lib()
    T, H, k = 16, 256, 8   # some hundred experts in use: most borders between thread blocks lie inside one
    blk = MoeBlock(on_device(bank(kind, 200, H, 48, 45)), top_k=k)
    x, w = rows(T, H, 46).cuda(), torch.ones(H, dtype=BF16, device="cuda")
    want = blk.decode(x, next_norm=w)
    blk.status()
    L.knj_decode_wait_limit(1 << 22)   # two milliseconds
    L.knj_moe_block_decode_test_stall(3)
    try:
        out, h = blk.decode(x, next_norm=w)
        with pytest.raises(_lib.KnjError) as e:
            blk.status()
        assert e.value.code == -5
        assert torch.isnan(out).all() and torch.isnan(h).all()
    finally:
        L.knj_moe_block_decode_test_stall(0)
        L.knj_decode_wait_limit(0)
    again = blk.decode(x, next_norm=w)
    blk.status()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
