"""The MoE block of a decode step over rows at the end of the f32 range: what the norm makes of them is finite, and so is the block's part."""
from dataclasses import replace

import pytest
import torch

import block_ops_ref as ref
import moe_decode_ref as dr
from test_gpu_moe_block import BF16, F32
from test_gpu_moe_decode import KINDS, bank, rows, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1, 3, 9])
def test_rows_at_the_end_of_the_range(kind, dtype, T):
    """Logits as sums of x * w * router leave the range from some 1e37 on, x * w itself at its end. The inverse norm of such a row lies below
    the normal range, where it has 21 bits: the planes' place in the bound has 2^-20 for it."""
    H, k = 512, 3
    b = bank(kind, 8, H, 112, 41, post=False, gate=False)
    b = replace(b, beta=0.0, pre_norm=torch.linspace(0.5, 2.5, H).to(BF16), router=(4 * b.router.float()).to(BF16))
    for largest in (1e36, 1e37, 1e38, 3.35e38):
        x = rows(T, H, 20 + T).double()
        x[0] *= largest / x[0].abs().max()
        if T > 1:
            x[T - 1] *= -largest / x[T - 1].abs().max()
        x = x.to(dtype)
        assert torch.isfinite(x).all()
        out, pe, pw = run(b, x.cuda(), k)
        assert torch.isfinite(out).all(), largest
        pe, pw = pe.cpu(), pw.cpu()
        dr.check_routing(b, x, pe, pw, k)
        s, es, _, _ = dr.block(b, x, pe, pw, k, planes=max(2.0 ** -20, dr.PLANES[kind]))
        ref.check(out, s, es + ref.held(s.abs() + es, out.dtype), "large rows")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [512, 4096])
def test_all_values_of_a_row_at_the_end_of_the_range(kind, H):
    """Sums over H squares leave the range even from values * 2^-64."""
    T, k = 2, 3
    b = replace(bank(kind, 8, H, 112, 43, post=False, gate=False), beta=0.0)
    x = torch.where(rows(T, H, 7) < 0, -3.35e38, 3.35e38) * torch.linspace(1.0, 0.9, H)
    w = torch.linspace(0.5, 1.5, H).to(BF16)
    out, pe, pw = run(b, x.cuda(), k)
    pe, pw = pe.cpu(), pw.cpu()
    dr.check_routing(b, x, pe, pw, k)
    s, es, _, _ = dr.block(b, x, pe, pw, k, planes=max(2.0 ** -20, dr.PLANES[kind]))
    ref.check(out, s, es + ref.held(s, F32), "block")
    # the stream itself in front of the next block
    c = replace(b, beta=1.0)
    _, h, pe, pw = run(c, x.cuda(), k, next_norm=w.cuda())
    _, _, hs, eh = dr.block(c, x, pe.cpu(), pw.cpu(), k, w, planes=max(2.0 ** -20, dr.PLANES[kind]))
    ref.check(h, hs, eh + 2.0 ** -20 * hs.abs() + ref.held(hs, F32), "next block's rows")
