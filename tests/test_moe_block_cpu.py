"""The MoE block's refusals, its weights' conversion to e4m3 blocks and the reader of unquantised GGUF experts, without a device."""
import ctypes as C

import numpy as np
import pytest
import torch

from kanjoos_b200 import _lib

A = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from kanjoos_b200 import build
    build.build()
    return _lib.lib()


def block_args(L, **kw):
    a = _lib.MoeBlockArgs(n_tokens=4, hidden=256, ffn=64, n_experts=8, top_k=2, x_dtype=0, out_dtype=0, w_dtype=1, alpha=1.0, beta=1.0, eps=1e-6, x=A,
                          ldx=256, out=A, ldo=256, pre_w=A, w_router=A, w_gate=A, w_up=A, w_down=A, workspace=A, workspace_bytes=1 << 30)
    a.w_norm_dtype = 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word,code", [
    (dict(hidden=0), "sizes", -1), (dict(n_tokens=-1), "sizes", -1), (dict(hidden=320), "multiple of 256", -1), (dict(ffn=72), "of 16", -1),
    (dict(hidden=33024), "32768", -1), (dict(n_experts=257), "out of range", -1), (dict(top_k=9), "out of range", -1),
    (dict(top_k=3, n_experts=2), "out of range", -1), (dict(w_dtype=0), "experts are", -1), (dict(x=None), "null", -1), (dict(out=None), "null", -1),
    (dict(w_down=None), "null", -1), (dict(w_router=None), "null", -1), (dict(w_dtype=3), "scales", -1), (dict(next_w=A), "go together", -1),
    (dict(workspace=None), "workspace", -4), (dict(workspace_bytes=64), "workspace", -4), (dict(workspace=A + 16), "256-byte", -1),
    (dict(gate_kind=1), "gate", -1), (dict(ldo=255), "stride", -1), (dict(ldx=255), "stride", -1), (dict(x_dtype=3), "f32, bf16 or f16", -1),
    (dict(out_dtype=3), "f32, bf16 or f16", -1), (dict(next_w=A, h_next=A, ld_h_next=256, h_next_dtype=3), "h_scale", -1),
])
def test_block_refusals(L, change, word, code):
    assert L.knj_moe_block_launch(C.byref(block_args(L, **change)), None) == code
    assert word in L.knj_last_error_string().decode()


def test_empty_block_and_workspace_sizes(L):
    assert L.knj_moe_block_launch(None, None) == -1
    assert L.knj_moe_block_launch(C.byref(_lib.MoeBlockArgs(n_tokens=0, hidden=256, ffn=64, n_experts=8, top_k=2)), None) == 0
    assert L.knj_moe_block_workspace_bytes(0, 256, 64, 8, 2, 1) == 256
    small, more, q = (L.knj_moe_block_workspace_bytes(*v) for v in ((8, 256, 64, 8, 2, 1), (16, 256, 64, 8, 2, 1), (8, 256, 64, 8, 2, 3)))
    assert small < more and small < q


@pytest.mark.parametrize("shape", [(128, 128), (3, 130, 200), (1, 1), (2, 64, 300)])
def test_e4m3_blocks(shape):
    import block_ops_ref as ref
    from kanjoos_b200.moe import e4m3_blocks
    g = torch.Generator()
    g.manual_seed(shape[-1])
    w = torch.randn(shape, generator=g)
    if shape[-1] == 300:
        w[0, :, :128] = 0          # a block of zeros
    q, s = e4m3_blocks(w)
    assert q.dtype == torch.float8_e4m3fn and q.shape == w.shape and s.shape == w.shape[:-2] + (-(-shape[-2] // 128), -(-shape[-1] // 128))
    v = ref.matrix_value(q, s)
    step = ref.matrix_value(torch.ones_like(w), s)
    # half a step of e4m3: 2^-4 relative, 2^-10 of the scale below the normal range; the division before it 2^-23
    assert ((v - w.double()).abs() <= (2.0 ** -4 + 2.0 ** -22) * w.double().abs() + 2.0 ** -10 * step).all()


def write_float_file(path, gguf, E, H, F, K, ftype):
    rng = np.random.Generator(np.random.Philox(77))
    kind = gguf.GGMLQuantizationType.F16 if ftype == "f16" else gguf.GGMLQuantizationType.BF16

    def bits(*shape):
        v = (rng.standard_normal(shape) * 0.05).astype(np.float32)
        return v.astype(np.float16).view(np.uint16) if ftype == "f16" else (v.view(np.uint32) >> 16).astype(np.uint16)
    arrays = {"gate": bits(E, F, H), "up": bits(E, F, H), "down": bits(E, H, F)}
    w = gguf.GGUFWriter(str(path), "qwen3moe")
    w.add_block_count(1)
    w.add_expert_count(E)
    w.add_expert_used_count(K)
    w.add_layer_norm_rms_eps(1e-6)
    w.add_tensor("blk.0.ffn_norm.weight", (1 + 0.1 * rng.standard_normal(H)).astype(np.float32))
    w.add_tensor("blk.0.post_ffw_norm.weight", (1 + 0.1 * rng.standard_normal(H)).astype(np.float32))
    w.add_tensor("blk.0.ffn_gate_inp.weight", (rng.standard_normal((E, H)) * 0.05).astype(np.float32))
    for key, name in (("gate", "ffn_gate_exps"), ("up", "ffn_up_exps"), ("down", "ffn_down_exps")):
        a = arrays[key]
        w.add_tensor(f"blk.0.{name}.weight", a.view(np.uint8).reshape(a.shape[:-1] + (a.shape[-1] * 2,)), raw_dtype=kind)
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    return arrays


@pytest.mark.parametrize("ftype", ["f16", "bf16"])
def test_reader_of_unquantised_experts(tmp_path, ftype):
    gguf = pytest.importorskip("gguf")
    from kanjoos_b200 import gguf_bank
    E, H, F, K = 4, 256, 64, 2
    arrays = write_float_file(tmp_path / "f.gguf", gguf, E, H, F, K, ftype)
    g = gguf_bank.GgufFile(str(tmp_path / "f.gguf"))
    a = gguf_bank.float_layer_arrays(g, 0)
    assert a["top_k"] == K and a["expert_type"] == ftype and a["router"].shape == (E, H) and not a["router_exact"] and "post_norm" in a
    for key in ("gate", "up", "down"):
        assert np.array_equal(a[key], arrays[key])
    assert gguf_bank.verify_against_gguf_py(str(tmp_path / "f.gguf")) == 6
    with pytest.raises(ValueError, match="Q4_K"):
        gguf_bank.layer_arrays(g, 0)      # the quantised path still refuses them
