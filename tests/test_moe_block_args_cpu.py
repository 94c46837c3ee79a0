"""What a whole MoE block refuses before its first launch: nothing of it may have run, not its norm, its router or its taps. Here without a
device, where a launch would be an error of another kind."""
import ctypes as C

import pytest

from test_moe_block_cpu import A, L, block_args  # noqa: F401

SCALES = dict(w_dtype=3, gate_scale=A, up_scale=A, down_scale=A)


@pytest.mark.parametrize("change,word", [
    (dict(w_gate=A + 8), "aligned"), (dict(w_up=A + 8), "aligned"), (dict(w_down=A + 8), "aligned"), (dict(w_router=A + 8), "aligned"),
    ({**SCALES, "w_down": A + 8}, "aligned"), (dict(n_tokens=(1 << 29) + 1, workspace_bytes=1 << 62), "2^30"),
])
def test_products_and_router_are_checked_before_anything_is_launched(L, change, word):  # noqa: F811
    assert L.knj_moe_block_launch(C.byref(block_args(L, **change)), None) == -1
    assert word in L.knj_last_error_string().decode()
