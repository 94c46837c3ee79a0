"""MoeBlock.status() of a block that has not run yet, without a device."""
import torch


def test_status_before_the_first_run(monkeypatch):
    from kanjoos_b200 import moe
    calls = []

    class Library:
        def knj_moe_block_workspace_bytes(self, *sizes):
            return 256

        def knj_moe_block_status(self, *args):
            calls.append(args)
            return 0
    monkeypatch.setattr(moe, "lib", Library)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    E, H, F = 2, 256, 16
    bank = moe.FloatExpertBank(gate=torch.zeros(E, F, H).bfloat16(), up=torch.zeros(E, F, H).bfloat16(), down=torch.zeros(E, H, F).bfloat16(),
                               router=torch.zeros(E, H).bfloat16())
    workspace = torch.zeros(1024, dtype=torch.uint8)
    at = -workspace.data_ptr() % 256
    moe.MoeBlock(bank, top_k=1, max_tokens=1, workspace=workspace[at:at + 256]).status()
    assert not calls


def test_a_type_that_no_row_has_is_refused_for_the_next_block(monkeypatch):
    import pytest
    from kanjoos_b200 import moe

    class Library:
        def knj_moe_block_workspace_bytes(self, *sizes):
            return 256
    monkeypatch.setattr(moe, "lib", Library)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    E, H, F = 2, 256, 16
    bank = moe.FloatExpertBank(gate=torch.zeros(E, F, H).bfloat16(), up=torch.zeros(E, F, H).bfloat16(), down=torch.zeros(E, H, F).bfloat16(),
                               router=torch.zeros(E, H).bfloat16())
    workspace = torch.zeros(1024, dtype=torch.uint8)
    at = -workspace.data_ptr() % 256
    block = moe.MoeBlock(bank, top_k=1, max_tokens=1, workspace=workspace[at:at + 256])
    for bad in (torch.int32, torch.float64, torch.float8_e5m2):
        with pytest.raises(ValueError, match="next_dtype"):
            block.run(torch.zeros(1, H), next_norm=torch.zeros(H), next_dtype=bad)
