"""Banks whose experts are codes are not turned into codes again, whichever they hold and whichever are asked for."""
from dataclasses import replace

import pytest
import torch


def bank():
    from kanjoos_b200.moe import FloatExpertBank
    g = torch.Generator().manual_seed(4)
    w = lambda *shape: torch.randn(shape, generator=g).bfloat16()  # noqa: E731
    return FloatExpertBank(gate=w(2, 16, 256), up=w(2, 16, 256), down=w(2, 256, 16), router=w(2, 256))


@pytest.mark.parametrize("held", ["to_e4m3", "to_int8"])
@pytest.mark.parametrize("asked", ["to_e4m3", "to_int8"])
def test_every_pair(held, asked):
    codes = getattr(bank(), held)()
    with pytest.raises(ValueError, match="already"):
        getattr(codes, asked)()
    # codes whose scales have not been set yet, and scales beside values
    with pytest.raises(ValueError, match="already"):
        getattr(replace(codes, gate_scale=None, up_scale=None, down_scale=None), asked)()
    with pytest.raises(ValueError, match="already"):
        getattr(replace(bank(), down_scale=codes.down_scale), asked)()
