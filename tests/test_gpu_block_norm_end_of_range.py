"""The norm between two blocks over rows whose values all lie at the end of the f32 range: their squares sum up to more than the range holds
even from values * 2^-64."""
import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_norm_range import BF16, F32, ROWS, gen, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H", ROWS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_the_largest_values(T, H, dtype):
    """The inverse norm lies below the normal range, where it has 21 bits: 2^-20 of either result for it."""
    g = gen("end", T, H)
    big = (torch.where(torch.rand((T, H), generator=g) < 0.5, -3.35e38, 3.35e38) * (1 - 0.1 * torch.rand((T, H), generator=g))).to(dtype)
    small, w = torch.randn((T, H), generator=g), 1 + 0.3 * torch.randn(H, generator=g)
    assert torch.isfinite(big).all()
    _, got = run(big, None, pre_w=w)
    _, _, h, eh = ref.block_norm(big, None, None, None, False, 1.0, 1.0, w, 1e-6)
    ref.check(got, h, eh + 2.0 ** -20 * h.abs() + ref.held(h, F32), "normalised stream")
    got, _ = run(small, big, post_w=w)
    s, es, _, _ = ref.block_norm(small, big, w, None, False, 1.0, 1.0, None, 1e-6)
    ref.check(got, s, es + 2.0 ** -20 * (s - small.double()).abs() + ref.held(s, F32), "normalised output of a block")
