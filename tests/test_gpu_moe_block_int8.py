"""The whole MoE block with int8 experts, against the block in 64 bits and against its single calls."""
import pytest
import torch

import block_ops_ref as ref
import int8_ref as i8
from test_gpu_moe_block import BF16, F16, F32, bank_of, on_device

pytestmark = pytest.mark.gpu


def values(codes, scale):
    return codes.double() * scale.double()[..., None]


def block_64(b, x, pair_exp, pair_w, top_k):
    """The block in 64 bits over the device's routing; the roundings between its stages are those that the block documents."""
    _, _, h, _ = ref.block_norm(x, None, None, None, False, 1.0, 1.0, b.pre_norm, b.rms_eps)
    hv = values(*i8.rows(h.to(BF16)))
    mats = [values(getattr(b, n), getattr(b, n + "_scale")) for n in ("gate", "up", "down")]
    y = torch.zeros((x.shape[0], b.hidden), dtype=torch.float64)
    for t in range(x.shape[0]):
        for s in range(top_k):
            e = int(pair_exp[t * top_k + s])
            a = torch.nn.functional.silu(hv[t] @ mats[0][e].t()) * (hv[t] @ mats[1][e].t())
            y[t] += float(pair_w[t * top_k + s]) * (values(*i8.rows(a.to(BF16)[None]))[0] @ mats[2][e].t())
    return ref.block_norm(x, y, b.post_norm, b.out_gate, b.gate_sigmoid, b.alpha, b.beta, torch.ones(b.hidden), b.rms_eps)


@pytest.mark.parametrize("T,E,H,F,k,stream", [(1, 16, 512, 256, 4, F32), (9, 16, 512, 272, 4, BF16), (70, 8, 768, 384, 2, F16), (300, 4, 512, 144, 3, F32)])
def test_block_against_64_bits(T, E, H, F, k, stream):
    from kanjoos_b200.moe import MoeBlock
    b = bank_of(BF16, E, H, F, T + H).to_int8()
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(T)).to(stream)
    blk = MoeBlock(on_device(b), top_k=k, max_tokens=T)
    out, h, pe, pw = blk.run(x.cuda(), next_norm=torch.ones(H, dtype=BF16, device="cuda"), next_dtype=F32, return_routing=True)
    blk.status()
    s, _, hs, _ = block_64(b, x, pe.cpu(), pw.cpu(), k)
    # Between the stages a value may be rounded the other way than in 64 bits: bf16 2^-8 of single places, and then a code by one step,
    # 2^-6 of a usual value (127 steps for three to four times its size); a sum over F or H of places takes that over the root of their number.
    size = s.abs() + (s - b.beta * x.double()).square().mean(1, keepdim=True).sqrt()
    ref.check(out, s, 2.0 ** -8 * size + ref.held(s, stream), "stream")
    ref.check(h, hs, 2.0 ** -7 * (hs.abs() + 1) + ref.held(hs, F32), "next block's rows")


def test_block_is_its_single_calls():
    from kanjoos_b200 import ops
    from kanjoos_b200.moe import MoeBlock
    T, E, H, F, k = 37, 16, 512, 256, 4
    d = on_device(bank_of(BF16, E, H, F, 5).to_int8())
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    out, pe, pw = MoeBlock(d, top_k=k, max_tokens=64).run(x, return_routing=True)
    _, h = ops.block_norm(x, pre_w=d.pre_norm, eps=d.rms_eps)
    _, pe2, pw2 = ops.router_topk(h, d.router, k, d.router_bias)
    assert torch.equal(pe, pe2) and torch.equal(pw, pw2)
    idx, cnt, _, _ = ops.moe_permute(pe2, E, T)
    a = ops.expert_gateup(h, d.gate, d.up, idx, cnt, T * k, k, gate_scale=d.gate_scale, up_scale=d.up_scale)
    y = ops.expert_proj(a, d.down, idx, cnt, T * k, scale=d.down_scale)
    c = ops.moe_combine(y, pe2, pw2, T, k)
    out2, _ = ops.block_norm(x, c, post_w=d.post_norm, gate=d.out_gate, gate_sigmoid=True, alpha=d.alpha, beta=d.beta, eps=d.rms_eps)
    assert torch.equal(out, out2)


def test_block_refuses_a_bank_without_scales():
    from kanjoos_b200.moe import MoeBlock
    d = on_device(bank_of(BF16, 8, 256, 64, 1).to_int8())
    d.up_scale = d.up_scale[:, :32].contiguous()
    with pytest.raises(ValueError, match="up_scale"):
        MoeBlock(d, top_k=2)
