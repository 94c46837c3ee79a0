"""Refusals of the MoE block of a decode step, decided on the host before any device work."""
import ctypes as C

import pytest

from test_block_ops_cpu import A, L, refused  # noqa: F401
from test_moe_block_cpu import block_args

CODES = dict(w_dtype=5, gate_scale=A, up_scale=A, down_scale=A)


@pytest.mark.parametrize("change,word,code", [
    (dict(hidden=0), "sizes", -1), (dict(n_tokens=-1), "sizes", -1), (dict(hidden=320), "multiple of 256", -1), (dict(ffn=72), "of 16", -1),
    (dict(n_experts=257), "out of range", -1), (dict(top_k=9), "out of range", -1), (dict(w_dtype=4), "experts are", -1), (dict(x=None), "null", -1),
    (dict(w_dtype=5), "scales", -1), (dict(w_dtype=3), "scales", -1), ({**CODES, "up_scale": None}, "scales", -1), (dict(next_w=A), "go together", -1),
    (dict(workspace=None), "workspace", -4), (dict(workspace_bytes=64), "workspace", -4), (dict(workspace=A + 16), "256-byte", -1),
    (dict(gate_kind=1), "gate", -1), (dict(ldo=255), "stride", -1), (dict(ldx=255), "stride", -1), (dict(x_dtype=3), "f32, bf16 or f16", -1),
    (dict(out_dtype=5), "f32, bf16 or f16", -1), (dict(w_norm_dtype=3), "weights", -1), (dict(next_w=A, h_next=A, ld_h_next=256, h_next_dtype=5), "h_dtype", -1),
    (dict(w_gate=A + 8), "aligned", -1), (dict(w_up=A + 4), "aligned", -1), (dict(w_down=A + 8), "aligned", -1), (dict(pre_w=A + 2), "aligned", -1),
    ({**CODES, "up_scale": A + 8}, "aligned", -1), (dict(w_router=A + 8), "aligned", -1), (dict(n_tokens=17), "at most 16", -1), (dict(ffn=40976, workspace_bytes=1 << 40), "40960", -1),
])
def test_refusals(L, change, word, code):
    refused(L, L.knj_moe_block_decode_launch(C.byref(block_args(L, **change)), None), word, code)


def test_no_tokens_and_no_arguments(L):
    assert L.knj_moe_block_decode_launch(C.byref(block_args(L, n_tokens=0)), None) == 0
    assert L.knj_moe_block_decode_launch(None, None) == -1


@pytest.mark.parametrize("tokens", [1, 16, 17, 64])
def test_one_workspace_serves_both_forms(L, tokens):
    """Room for the rows of pairs in f32 that the decode step keeps, whatever the sizes."""
    for hidden, ffn, experts, k, kind in ((2048, 768, 128, 8, 1), (256, 40960, 4, 2, 5), (1024, 8192, 8, 8, 3)):
        need = L.knj_moe_block_workspace_bytes(tokens, hidden, ffn, experts, k, kind)
        pairs = min(tokens, 16) * k
        assert need >= pairs * (ffn + hidden) * 4 + min(tokens, 16) * experts * 4 + 256
