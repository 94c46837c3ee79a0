"""Refusals of the int8 operators, decided on the host before any device work, and the conversion of matrices, without a device."""
import ctypes as C

import numpy as np
import pytest
import torch

from kanjoos_b200 import _lib
from test_block_ops_cpu import A, L, gemm_args, refused  # noqa: F401
from test_moe_block_cpu import block_args, write_float_file


def test_empty_calls_and_workspaces(L):
    assert L.knj_int8_rows_launch(None, 0, 0, 0, 64, None, None, None) == 0
    assert L.knj_int8_matmul_launch(C.byref(_lib.Int8MatmulArgs(n_in=64, n_out=64, m=0)), None) == 0
    refused(L, L.knj_int8_matmul_launch(None, None), "null")
    assert L.knj_int8_matmul_workspace_bytes(0, 64) == 0 and L.knj_int8_matmul_workspace_bytes(9, 130) == 1280 + 256


def test_few_rows_need_no_workspace(L):
    for m, k, few in ((1, 40960, True), (1, 40976, False), (2, 20480, True), (3, 10240, True), (3, 10256, False), (4, 10240, True),
                      (5, 16, False)):
        assert (L.knj_int8_matmul_workspace_bytes(m, k) == 0) == few, (m, k)


@pytest.mark.parametrize("args,word", [
    ((A, 0, 64, -1, 64, A, A), "sizes"), ((A, 0, 64, 1, 0, A, A), "sizes"), ((None, 0, 64, 1, 64, A, A), "null"), ((A, 0, 64, 1, 64, None, A), "null"),
    ((A, 0, 64, 1, 64, A, None), "null"), ((A, 3, 64, 1, 64, A, A), "f32, bf16 or f16"), ((A, 5, 64, 1, 64, A, A), "f32, bf16 or f16"),
    ((A, 0, 63, 1, 64, A, A), "stride"),
])
def test_rows_refusals(L, args, word):
    refused(L, L.knj_int8_rows_launch(*args, None), word)


@pytest.mark.parametrize("change,word,code", [
    (dict(n_in=0), "sizes", -1), (dict(n_out=0), "sizes", -1), (dict(m=-1), "sizes", -1), (dict(W=None), "null", -1), (dict(S=None), "null", -1),
    (dict(x=None), "null", -1), (dict(y=None), "null", -1), (dict(n_in=72, ldx=72), "multiple of 16", -1), (dict(W=A + 8), "aligned", -1),
    (dict(n_in=131072, ldx=131072), "131072", -1), (dict(dt=3), "f32, bf16, f16 or int8", -1), (dict(dt=4), "f32, bf16, f16 or int8", -1),
    (dict(yt=5), "f32, bf16 or f16", -1), (dict(ldx=63), "stride", -1), (dict(ldy=7), "stride", -1), (dict(ws=None), "workspace", -4),
    (dict(nb=1023), "workspace", -4), (dict(ws=A + 16), "256-byte", -1), (dict(dt=5), "null", -1), (dict(dt=5, XS=A, ldx=72), "16-byte", -1),
    (dict(dt=5, XS=A, x=A + 4), "16-byte", -1), (dict(m=(1 << 30) + 1), "2^30", -1),
])
def test_matmul_refusals(L, change, word, code):
    v = dict(W=A, S=A, n_in=64, n_out=8, x=A, dt=0, XS=None, ldx=64, m=9, y=A, yt=0, ldy=8, ws=A, nb=1024)
    v.update(change)
    a = _lib.Int8MatmulArgs(w=v["W"], w_scale=v["S"], n_in=v["n_in"], n_out=v["n_out"], x=v["x"], x_dtype=v["dt"], x_scale=v["XS"], ldx=v["ldx"], m=v["m"],
                            y=v["y"], y_dtype=v["yt"], ldy=v["ldy"], workspace=v["ws"], workspace_bytes=v["nb"])
    rc = L.knj_int8_matmul_launch(C.byref(a), None)
    refused(L, rc, word, code)


I8 = dict(x_dtype=5, w_dtype=5, x_scale=A, w0_scale=A, w1_scale=A)


@pytest.mark.parametrize("change,word", [
    ({**I8, "x_scale": None}, "scales"), ({**I8, "w0_scale": None}, "scales"), ({**I8, "K": 40}, "16-byte"), ({**I8, "ldx": 72}, "16-byte"),
    ({**I8, "x_dtype": 1}, "one type"), ({**I8, "K": 131072, "ldx": 131072}, "32 bits"), ({**I8, "out_dtype": 5}, "outputs"),
])
@pytest.mark.parametrize("name", ["knj_expert_gateup_launch", "knj_expert_proj_launch"])
def test_expert_product_refusals(L, name, change, word):
    refused(L, getattr(L, name)(C.byref(gemm_args(**change)), None), word)


def test_gateup_needs_both_scales(L):
    refused(L, L.knj_expert_gateup_launch(C.byref(gemm_args(**{**I8, "w1_scale": None})), None), "scales")


def test_block_of_int8_experts_needs_scales_and_room(L):
    assert L.knj_moe_block_launch(C.byref(block_args(L, w_dtype=5)), None) == -1 and b"scales" in L.knj_last_error_string()
    need = L.knj_moe_block_workspace_bytes(4, 256, 64, 8, 2, 5)
    assert need > L.knj_moe_block_workspace_bytes(4, 256, 64, 8, 2, 1)
    a = block_args(L, w_dtype=5, gate_scale=A, up_scale=A, down_scale=A, workspace_bytes=need - 1)
    assert L.knj_moe_block_launch(C.byref(a), None) == -4


@pytest.mark.parametrize("shape", [(1, 1), (5, 300), (3, 130, 200)])
def test_int8_channels(shape):
    from kanjoos_b200.moe import int8_channels
    w = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    w[..., 0, :] = 0
    q, s = int8_channels(w.to(torch.bfloat16))
    assert q.dtype == torch.int8 and q.shape == w.shape and s.shape == w.shape[:-1] and s.dtype == torch.float32
    v = w.to(torch.bfloat16).double()
    assert (q[..., 0, :] == 0).all() and (s[..., 0] == 0).all()
    # half a step of the scale, and the roundings of the division in front of it and of the scale
    assert ((q.double() * s.double()[..., None] - v).abs() <= s.double()[..., None] * (0.5 + 127 * 2.0 ** -22)).all()
    if shape[-2] > 1:
        assert (q[..., 1:, :].abs().amax(-1) == 127).all()


def test_gguf_experts_as_int8(tmp_path):
    gguf = pytest.importorskip("gguf")
    from kanjoos_b200 import gguf_bank
    write_float_file(tmp_path / "f.gguf", gguf, 4, 256, 64, 2, "bf16")
    g = gguf_bank.GgufFile(str(tmp_path / "f.gguf"))
    plain, k = gguf_bank.load_float_expert_bank(g, 0, device="cpu")
    bank, k8 = gguf_bank.load_float_expert_bank(g, 0, device="cpu", int8=True)
    assert k == k8 and bank.gate.dtype == torch.int8 and bank.down_scale.shape == (4, 256) and bank.nbytes() * 2 == plain.nbytes()
    for n in ("gate", "up", "down"):
        w, q, s = getattr(plain, n).double(), getattr(bank, n).double(), getattr(bank, n + "_scale").double()
        assert ((q * s[..., None] - w).abs() <= 0.5001 * s[..., None]).all()
    with pytest.raises(ValueError, match="exclude"):
        gguf_bank.load_float_expert_bank(g, 0, device="cpu", e4m3=True, int8=True)


def test_codes_are_not_turned_into_codes_again():
    from kanjoos_b200.moe import FloatExpertBank
    g = torch.Generator().manual_seed(3)
    bank = FloatExpertBank(gate=torch.randn((2, 16, 256), generator=g).bfloat16(), up=torch.randn((2, 16, 256), generator=g).bfloat16(),
                           down=torch.randn((2, 256, 16), generator=g).bfloat16(), router=torch.randn((2, 256), generator=g).bfloat16())
    for codes in (bank.to_int8(), bank.to_e4m3()):
        with pytest.raises(ValueError, match="already"):
            codes.to_int8()
    with pytest.raises(ValueError, match="already"):
        bank.to_int8().to_e4m3()
