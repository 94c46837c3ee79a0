"""What a bank of unquantised experts keeps of its file: norm weights as they stand there, and word of a router that does not."""
import numpy as np
import pytest
import torch

from test_moe_block_cpu import write_float_file


def stored(g, name):
    """A tensor's values as the file holds them, f32."""
    return np.asarray(g.payload(g.require(name))).view(np.float32)


@pytest.mark.parametrize("e4m3", [False, True])
def test_norm_weights_keep_the_files_values(tmp_path, e4m3):
    gguf = pytest.importorskip("gguf")
    from kanjoos_b200 import gguf_bank
    write_float_file(tmp_path / "f.gguf", gguf, 4, 256, 64, 2, "bf16")
    g = gguf_bank.GgufFile(str(tmp_path / "f.gguf"))
    bank, _ = gguf_bank.load_float_expert_bank(g, 0, device="cpu", e4m3=e4m3)
    for t, name in ((bank.pre_norm, "ffn_norm"), (bank.post_norm, "post_ffw_norm")):
        assert t.dtype == torch.float32 and np.array_equal(t.numpy(), stored(g, f"blk.0.{name}.weight"))
    router = stored(g, "blk.0.ffn_gate_inp.weight").reshape(4, 256)
    assert bank.router.dtype == torch.bfloat16 and not np.array_equal(bank.router.float().numpy(), router)
    assert bank.router_exact is False


def test_a_bf16_router_is_the_files(tmp_path):
    gguf = pytest.importorskip("gguf")
    from kanjoos_b200 import gguf_bank
    E, H, F = 2, 256, 16
    rng = np.random.Generator(np.random.Philox(3))
    kind = gguf.GGMLQuantizationType

    def bits(*shape):
        return (rng.standard_normal(shape).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    w = gguf.GGUFWriter(str(tmp_path / "b.gguf"), "qwen3moe")
    w.add_block_count(1)
    w.add_expert_count(E)
    w.add_expert_used_count(1)
    arrays = {"ffn_gate_inp": bits(E, H), "ffn_norm": bits(H), "ffn_gate_exps": bits(E, F, H), "ffn_up_exps": bits(E, F, H), "ffn_down_exps": bits(E, H, F)}
    post = rng.standard_normal(H).astype(np.float16)
    for name, a in arrays.items():
        w.add_tensor(f"blk.0.{name}.weight", a.view(np.uint8).reshape(a.shape[:-1] + (a.shape[-1] * 2,)), raw_dtype=kind.BF16)
    w.add_tensor("blk.0.post_ffw_norm.weight", post)
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    bank, k = gguf_bank.load_float_expert_bank(gguf_bank.GgufFile(str(tmp_path / "b.gguf")), 0, device="cpu")
    assert k == 1 and bank.router_exact is True
    assert np.array_equal(bank.router.view(torch.int16).numpy().view(np.uint16), arrays["ffn_gate_inp"])
    # norms of different types in the file meet in f32, which holds both
    assert bank.pre_norm.dtype == bank.post_norm.dtype == torch.float32
    assert np.array_equal(bank.pre_norm.numpy().view(np.uint32), arrays["ffn_norm"].astype(np.uint32) << 16)
    assert np.array_equal(bank.post_norm.numpy(), post.astype(np.float32))


@pytest.mark.gpu
def test_the_next_blocks_norm_may_be_narrower_than_the_banks():
    """Banks from files carry f32 norms; a caller's 16-bit weights for the next block are taken as the values they are."""
    from dataclasses import replace
    from kanjoos_b200.moe import MoeBlock
    from test_gpu_moe_block import bank_of, on_device
    b = on_device(bank_of(torch.bfloat16, 8, 256, 128, 4))
    b = replace(b, pre_norm=b.pre_norm.float() * 1.001, post_norm=b.post_norm.float() * 0.999)
    x = torch.randn((5, 256), device="cuda")
    nxt = torch.randn(256, device="cuda")
    for t in (torch.bfloat16, torch.float16):
        blk = MoeBlock(b, top_k=2, max_tokens=8)
        got, want = blk.run(x, next_norm=nxt.to(t)), blk.run(x, next_norm=nxt.to(t).float())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="next_norm"):
        MoeBlock(replace(b, pre_norm=b.pre_norm.bfloat16(), post_norm=None), top_k=2, max_tokens=8).run(x, next_norm=nxt)
