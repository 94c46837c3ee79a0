"""Refusals of the operators around an MoE block: every one is decided on the host before any device work, so they are
tested without a device, with addresses that are never followed."""
import ctypes as C

import pytest

from kanjoos_b200 import _lib

A = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from kanjoos_b200 import build
    build.build()
    return _lib.lib()


def refused(L, rc, word, code=-1):
    assert rc == code, rc
    text = L.knj_last_error_string().decode()
    assert word in text, text


def norm_args(**kw):
    a = _lib.BlockNormArgs(n_tokens=2, hidden=64, x=A, ldx=64, y=A, ldy=64, post_w=A, pre_w=A, stream_out=A, ld_stream=64, h=A, ldh=64,
                           alpha=1.0, beta=1.0, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(hidden=0), "sizes"), (dict(n_tokens=-1), "sizes"), (dict(hidden=32769, ldx=40000, ldy=40000, ld_stream=40000, ldh=40000), "32768"),
    (dict(x=None), "null"), (dict(stream_out=None, h=None, pre_w=None), "null"), (dict(h=None), "go together"), (dict(pre_w=None), "go together"),
    (dict(y=None), "need a block output"), (dict(gate_kind=1), "gate"), (dict(gate=A), "gate"), (dict(gate=A, gate_kind=4), "gate"),
    (dict(y=None, post_w=None, gate=A, gate_kind=1), "need a block output"),
    (dict(x_dtype=3), "f32, bf16 or f16"), (dict(y_dtype=3), "f32, bf16 or f16"), (dict(stream_dtype=3), "f32, bf16 or f16"),
    (dict(gate=A, gate_kind=1, gate_dtype=3), "f32, bf16 or f16"), (dict(w_dtype=3), "weights"), (dict(h_dtype=4), "h_dtype"),
    (dict(h_dtype=3), "h_scale"), (dict(ldx=63), "stride"), (dict(ldy=63), "stride"), (dict(ld_stream=63), "stride"), (dict(ldh=63), "stride"),
    (dict(gate=A, gate_kind=3, ldg=63), "stride"), (dict(gate=A, gate_kind=2, ldg=0), "stride"),
])
def test_block_norm_refusals(L, change, word):
    refused(L, L.knj_block_norm_launch(C.byref(norm_args(**change)), None), word)


def test_empty_calls_are_fine(L):
    assert L.knj_block_norm_launch(C.byref(_lib.BlockNormArgs(n_tokens=0, hidden=64)), None) == 0
    assert L.knj_block_norm_launch(None, None) == -1
    assert L.knj_fp8_rows_launch(None, 0, 0, 0, 64, None, None, None) == 0
    assert L.knj_fp8_matmul_launch(None, None, 64, 64, None, 0, 64, 0, None, 0, 64, None, 0, None, None) == 0
    for fn in (L.knj_expert_gateup_launch, L.knj_expert_proj_launch):
        assert fn(C.byref(_lib.ExpertGemmArgs(n_pairs=0, N=8, K=8, n_experts=1)), None) == 0
        assert fn(None, None) == -1
    assert L.knj_fp8_matmul_workspace_bytes(0, 64) == 0 and L.knj_fp8_matmul_workspace_bytes(3, 130) == 512 + 256


@pytest.mark.parametrize("args,word", [
    ((A, 0, 64, -1, 64, A, A), "sizes"), ((A, 0, 64, 1, 0, A, A), "sizes"), ((None, 0, 64, 1, 64, A, A), "null"), ((A, 0, 64, 1, 64, None, A), "null"),
    ((A, 0, 64, 1, 64, A, None), "null"), ((A, 3, 64, 1, 64, A, A), "f32, bf16 or f16"), ((A, 0, 63, 1, 64, A, A), "stride"),
])
def test_fp8_rows_refusals(L, args, word):
    refused(L, L.knj_fp8_rows_launch(*args, None), word)


def gemm_args(**kw):
    a = _lib.ExpertGemmArgs(x=A, ldx=64, w0=A, w1=A, pair_idx=A, pair_cnt=A, idx_stride=4, out=A, ldo=32, n_rows=4, n_pairs=4, N=32, K=64,
                            n_experts=2, row_div=1, x_dtype=1, w_dtype=1, out_dtype=0, out_scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


E8 = dict(x_dtype=3, w_dtype=3, x_scale=A, w0_scale=A, w1_scale=A)


@pytest.mark.parametrize("change,word", [
    (dict(N=0), "sizes"), (dict(K=0), "sizes"), (dict(n_experts=0), "sizes"), (dict(n_experts=257), "sizes"), (dict(n_pairs=-1), "sizes"),
    (dict(n_rows=-1), "sizes"), (dict(n_rows=0), "without a row"), (dict(w_dtype=0, x_dtype=0), "bf16, f16 or e4m3"), (dict(w_dtype=4, x_dtype=4), "bf16, f16 or e4m3"),
    (dict(x_dtype=2), "one type"), (dict(x=None), "null"), (dict(w0=None), "null"), (dict(pair_idx=None), "null"), (dict(pair_cnt=None), "null"),
    (dict(out=None), "null"), (dict(w_dtype=3, x_dtype=3), "scales"), ({**E8, "x_scale": None}, "scales"), ({**E8, "w0_scale": None}, "scales"),
    (dict(K=60, ldx=64), "16-byte"), (dict(ldx=68), "16-byte"), ({**E8, "K": 40}, "16-byte"), ({**E8, "ldx": 72}, "16-byte"),
    (dict(x=A + 8), "aligned"), (dict(w0=A + 8), "aligned"), (dict(ldx=56), "stride"), (dict(ldo=31), "stride"), (dict(idx_stride=0), "stride"),
    (dict(row_div=0), "row_div"), (dict(out_dtype=3), "outputs"),
])
@pytest.mark.parametrize("name", ["knj_expert_gateup_launch", "knj_expert_proj_launch"])
def test_expert_product_refusals(L, name, change, word):
    refused(L, getattr(L, name)(C.byref(gemm_args(**change)), None), word)


def test_gateup_needs_both_matrices(L):
    refused(L, L.knj_expert_gateup_launch(C.byref(gemm_args(w1=None)), None), "null")
    refused(L, L.knj_expert_gateup_launch(C.byref(gemm_args(w1=A + 8)), None), "aligned")
    refused(L, L.knj_expert_gateup_launch(C.byref(gemm_args(**{**E8, "w1_scale": None})), None), "scales")


@pytest.mark.parametrize("change,word,code", [
    (dict(n_in=0), "sizes", -1), (dict(n_out=0), "sizes", -1), (dict(m=-1), "sizes", -1), (dict(W=None), "null", -1), (dict(S=None), "null", -1),
    (dict(x=None), "null", -1), (dict(y=None), "null", -1), (dict(n_in=72, ldx=72), "multiple of 16", -1), (dict(W=A + 8), "aligned", -1),
    (dict(dt=3), "f32, bf16 or f16", -1), (dict(yt=3), "f32, bf16 or f16", -1), (dict(ldx=63), "stride", -1), (dict(ldy=7), "stride", -1),
    (dict(ws=None), "workspace", -4), (dict(nb=511), "workspace", -4), (dict(ws=A + 16), "256-byte", -1),
])
def test_fp8_matmul_refusals(L, change, word, code):
    v = dict(W=A, S=A, n_in=64, n_out=8, x=A, dt=0, ldx=64, m=2, y=A, yt=0, ldy=8, ws=A, nb=512)
    v.update(change)
    rc = L.knj_fp8_matmul_launch(v["W"], v["S"], v["n_in"], v["n_out"], v["x"], v["dt"], v["ldx"], v["m"], v["y"], v["yt"], v["ldy"], v["ws"],
                                 v["nb"], None, None)
    refused(L, rc, word, code)


def test_python_entry_points_refuse_tensors_off_the_device():
    import torch
    from kanjoos_b200 import ops
    if torch.cuda.is_available():
        pytest.skip("the current device would be a CUDA device")
    x = torch.zeros((2, 64))
    for call in (lambda: ops.fp8_rows(x), lambda: ops.block_norm(x, x), lambda: ops.fp8_matmul(x.to(torch.float8_e4m3fn), x, x)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_tables_and_rows_beyond_32_bit_counts_are_refused(L):
    for name in ("knj_expert_gateup_launch", "knj_expert_proj_launch"):
        refused(L, getattr(L, name)(C.byref(gemm_args(idx_stride=(1 << 30) + 1)), None), "2^30")
        refused(L, getattr(L, name)(C.byref(gemm_args(idx_stride=1 << 62)), None), "2^30")
        refused(L, getattr(L, name)(C.byref(gemm_args(n_pairs=(1 << 30) + 1)), None), "2^30")


def test_packed_bytes_are_the_structures():
    for cls in (_lib.BlockNormArgs, _lib.ExpertGemmArgs):
        values = list(range(1, len(cls._fields_) + 1))
        data = _lib.packed(cls)(*values)
        assert len(data) == C.sizeof(cls)
        back = cls.from_buffer_copy(data)
        assert [getattr(back, name) for name, _ in cls._fields_] == values
