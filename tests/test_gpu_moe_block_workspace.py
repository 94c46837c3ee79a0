"""A block over a workspace that run alone needs: run has its results, decode refuses."""
import pytest
import torch

from test_gpu_moe_block import BF16, bank_of, on_device

pytestmark = pytest.mark.gpu


def test_run_without_room_for_decode():
    from kanjoos_b200 import _lib
    from kanjoos_b200.moe import MoeBlock
    T, H, F, E, k = 3, 256, 4096, 8, 4
    d = on_device(bank_of(BF16, E, H, F, 5))
    L = _lib.lib()
    least = L.knj_moe_block_launch_workspace_bytes(T, H, F, E, k, _lib.DT_BF16)
    assert least < L.knj_moe_block_workspace_bytes(T, H, F, E, k, _lib.DT_BF16)
    behind = 4096
    room = torch.full((least + behind,), 0xA5, dtype=torch.uint8, device="cuda")
    blk, full = MoeBlock(d, top_k=k, max_tokens=T, workspace=room[:least]), MoeBlock(d, top_k=k, max_tokens=T)
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(6)).cuda()
    want = full.run(x)
    assert torch.equal(blk.run(x), want)
    blk.status()
    with pytest.raises(_lib.KnjError) as e:
        blk.decode(x)
    assert e.value.code == -4
    assert torch.equal(blk.run(x), want) and (room[least:] == 0xA5).all()
    assert full.decode(x).shape == (T, H)
