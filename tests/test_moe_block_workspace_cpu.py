"""Each form of the MoE block asks for the workspace that it needs itself, decided on the host before any device work."""
import ctypes as C

import pytest
import torch

from test_block_ops_cpu import L, refused  # noqa: F401
from test_moe_block_cpu import block_args

# tokens, hidden, ffn, experts, top_k, and what the chain of launches needs of them in bf16
SIZES = [((1, 2048, 8192, 8, 2), 62976), ((16, 256, 4096, 8, 8), 1206784)]


@pytest.mark.parametrize("sizes,chain", SIZES)
def test_each_launch_checks_its_own_need(L, sizes, chain):
    T, H, F, E, k = sizes
    both = L.knj_moe_block_workspace_bytes(*sizes, 1)
    assert L.knj_moe_block_launch_workspace_bytes(*sizes, 1) == chain < both

    def call(entry, nbytes):   # a short output row is refused behind the workspace's check
        return getattr(L, entry)(C.byref(block_args(L, n_tokens=T, hidden=H, ffn=F, n_experts=E, top_k=k, ldx=H, ldo=H - 1, workspace_bytes=nbytes)), None)
    refused(L, call("knj_moe_block_launch", chain), "stride", -1)
    refused(L, call("knj_moe_block_launch", chain - 1), "workspace", -4)
    refused(L, call("knj_moe_block_decode_launch", both), "stride", -1)
    refused(L, call("knj_moe_block_decode_launch", both - 1), "workspace", -4)


def test_no_tokens_and_many(L):
    assert L.knj_moe_block_launch_workspace_bytes(0, 256, 64, 8, 2, 1) == 256
    # of many tokens the chain's need is the larger
    for kind in (1, 2, 3, 5):
        assert L.knj_moe_block_launch_workspace_bytes(4096, 2048, 768, 128, 8, kind) == L.knj_moe_block_workspace_bytes(4096, 2048, 768, 128, 8, kind)


@pytest.mark.parametrize("sizes,chain", SIZES)
def test_a_block_takes_the_workspace_that_run_needs(monkeypatch, L, sizes, chain):
    from kanjoos_b200 import moe
    T, H, F, E, k = sizes
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    bank = moe.FloatExpertBank(gate=torch.empty(E, F, H, dtype=torch.bfloat16), up=torch.empty(E, F, H, dtype=torch.bfloat16),
                               down=torch.empty(E, H, F, dtype=torch.bfloat16), router=torch.empty(E, H, dtype=torch.bfloat16))
    room = torch.zeros(chain + 256, dtype=torch.uint8)
    room = room[-room.data_ptr() % 256:]
    assert moe.MoeBlock(bank, top_k=k, max_tokens=T, workspace=room[:chain]).workspace.numel() == chain
    with pytest.raises(ValueError, match="workspace"):
        moe.MoeBlock(bank, top_k=k, max_tokens=T, workspace=room[:chain - 1])
