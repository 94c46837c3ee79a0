"""The whole MoE block with bf16, f16 and e4m3 experts (norm, routing, expert products, combine, norm behind the block, gate, scaled
residual, norm of the next block), as one call and as the single calls that it is made of, against the block in 64 bits."""
import numpy as np
import pytest
import torch

import block_ops_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def bank_of(kind, E, H, F, seed, post=True, gate=True):
    from kanjoos_b200.moe import FloatExpertBank
    g = torch.Generator()
    g.manual_seed(seed)
    mk = lambda *s: (torch.randn(s, generator=g) * 0.03)  # noqa: E731
    w16 = F16 if kind == F16 else BF16
    b = FloatExpertBank(gate=mk(E, F, H).to(w16), up=mk(E, F, H).to(w16), down=mk(E, H, F).to(w16), router=mk(E, H).to(BF16),
                        router_bias=torch.randn(E, generator=g), pre_norm=(1 + 0.1 * torch.randn(H, generator=g)).to(BF16),
                        post_norm=(1 + 0.1 * torch.randn(H, generator=g)).to(BF16) if post else None,
                        out_gate=torch.randn(H, generator=g).to(BF16) if gate else None, gate_sigmoid=True, alpha=0.6, beta=1.1)
    return b.to_e4m3() if kind == E4M3 else b


def on_device(b):
    from dataclasses import fields, replace
    return replace(b, **{f.name: getattr(b, f.name).cuda() for f in fields(b) if torch.is_tensor(getattr(b, f.name))})


def block_64(b, x, pair_exp, pair_w, top_k, kind, row_gate=None):
    """The block in 64 bits over the device's routing; the roundings between its stages are those that the block documents."""
    H = b.hidden
    act = F16 if kind == F16 else BF16
    _, _, h, _ = ref.block_norm(x, None, None, None, False, 1.0, 1.0, b.pre_norm, b.rms_eps)
    h = h.to(act)
    hv = ref.rows_value(*ref.fp8_rows(h)) if kind == E4M3 else h.double()
    mats = [ref.matrix_value(getattr(b, n), getattr(b, n + "_scale")) for n in ("gate", "up", "down")]
    y = torch.zeros((x.shape[0], H), dtype=torch.float64)
    for t in range(x.shape[0]):
        for s in range(top_k):
            e = int(pair_exp[t * top_k + s])
            a = torch.nn.functional.silu(hv[t] @ mats[0][e].t()) * (hv[t] @ mats[1][e].t())
            a = (a * 2.0 ** -6).to(F16).double() * 64 if kind == F16 else a.to(BF16)
            if kind == E4M3:
                a = ref.rows_value(*ref.fp8_rows(a[None]))[0]
            y[t] += float(pair_w[t * top_k + s]) * (a.double() @ mats[2][e].t())
    gate = b.out_gate if row_gate is None else row_gate
    return ref.block_norm(x, y, b.post_norm, gate, b.gate_sigmoid, b.alpha, b.beta, torch.ones(H), b.rms_eps)


CASES = [
    (BF16, 1, 16, 512, 256, 4, F32), (BF16, 9, 16, 512, 256, 4, BF16), (F16, 33, 8, 256, 272, 8, F32), (E4M3, 1, 16, 512, 256, 4, F32),
    (E4M3, 70, 8, 768, 384, 2, BF16), (BF16, 300, 4, 256, 128, 1, F32), (E4M3, 300, 4, 512, 144, 3, F16), (F16, 5, 200, 256, 48, 8, F16),
]


@pytest.mark.parametrize("kind,T,E,H,F,k,stream", CASES)
def test_block_against_64_bits(kind, T, E, H, F, k, stream):
    from kanjoos_b200.moe import MoeBlock
    b = bank_of(kind, E, H, F, T + H)
    d = on_device(b)
    g = torch.Generator()
    g.manual_seed(T)
    x = torch.randn((T, H), generator=g).to(stream)
    nxt = torch.ones(H, dtype=BF16)
    blk = MoeBlock(d, top_k=k, max_tokens=T)
    out, h, pe, pw = blk.run(x.cuda(), next_norm=nxt.cuda(), next_dtype=F32, return_routing=True)
    blk.status()
    assert out.dtype == stream
    pe, pw = pe.cpu(), pw.cpu()
    # the routing is a softmax over the router's logits of the normalised rows, renormalised over its top k
    act = F16 if kind == F16 else BF16
    _, _, hn, _ = ref.block_norm(x, None, None, None, False, 1.0, 1.0, b.pre_norm, b.rms_eps)
    logits = hn.to(act).double() @ b.router.double().t() + b.router_bias.double()
    top = logits.gather(1, pe.view(T, k).long())
    assert (top.min(1).values + 1e-4 >= logits.topk(k, 1).values.min(1).values).all()
    assert torch.allclose(pw.view(T, k).double(), top.softmax(1), atol=2e-5)
    s, _, hs, _ = block_64(b, x, pe, pw, k, kind)
    # Between the stages a value may be rounded the other way than in 64 bits: half a step of its type (bf16 2^-8, fp16 2^-11, e4m3
    # 2^-4) in single places. One place of F or H moves a sum of them by that share over sqrt(F); 16 bits: 2^-8 of the block's
    # size covers all places at once, e4m3: 2^-4 / sqrt(128) for the single places of one group.
    tol = {BF16: 2.0 ** -8, F16: 2.0 ** -10, E4M3: 2.0 ** -6}[kind]
    size = s.abs() + (s - b.beta * x.double()).square().mean(1, keepdim=True).sqrt()
    ref.check(out, s, tol * size + ref.held(s, stream), "stream")
    ref.check(h, hs, 2 * tol * (hs.abs() + 1) + ref.held(hs, F32), "next block's rows")


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_block_is_its_single_calls(kind):
    """One call gives the bits of the single operators in turn, with a row gate and e4m3 rows for the next block."""
    from kanjoos_b200 import ops
    from kanjoos_b200.moe import MoeBlock
    T, E, H, F, k = 37, 16, 512, 256, 4
    d = on_device(bank_of(kind, E, H, F, 5, gate=False))
    g = torch.Generator()
    g.manual_seed(1)
    x, gate = torch.randn((T, H), generator=g).to(BF16).cuda(), torch.randn((T, 1), generator=g).cuda()
    nxt = (1 + 0.1 * torch.randn(H, generator=g)).to(BF16).cuda()
    out, (q, s), pe, pw = MoeBlock(d, top_k=k, max_tokens=64).run(x, gate=gate, next_norm=nxt, next_dtype=E4M3, return_routing=True)
    _, h = ops.block_norm(x, pre_w=d.pre_norm, eps=d.rms_eps)
    _, pe2, pw2 = ops.router_topk(h, d.router, k, d.router_bias)
    assert torch.equal(pe, pe2) and torch.equal(pw, pw2)
    idx, cnt, _, _ = ops.moe_permute(pe2, E, T)
    a = ops.expert_gateup(h, d.gate, d.up, idx, cnt, T * k, k, gate_scale=d.gate_scale, up_scale=d.up_scale, out_dtype=BF16)
    y = ops.expert_proj(a, d.down, idx, cnt, T * k, scale=d.down_scale)
    c = ops.moe_combine(y, pe2, pw2, T, k)
    out2, (q2, s2) = ops.block_norm(x, c, post_w=d.post_norm, gate=gate, gate_sigmoid=True, alpha=d.alpha, beta=d.beta, pre_w=nxt, eps=d.rms_eps, norm_dtype=E4M3)
    assert torch.equal(out, out2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_block_in_place_captured_and_on_another_stream(kind):
    from kanjoos_b200.moe import MoeBlock
    T, E, H, F, k = 12, 8, 256, 128, 2
    d = on_device(bank_of(kind, E, H, F, 6))
    g = torch.Generator()
    g.manual_seed(2)
    x = torch.randn((T, H), generator=g).cuda()
    blk = MoeBlock(d, top_k=k, max_tokens=16)
    want = blk.run(x).clone()
    y = x.clone()
    assert blk.run(y, out=y).data_ptr() == y.data_ptr() and torch.equal(y, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = MoeBlock(d, top_k=k, max_tokens=16).run(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    # captured, replayed with other rows in the same buffer
    buf, out = x.clone(), torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        blk.run(buf, out=out)
    x2 = torch.randn((T, H), generator=g).cuda()
    buf.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, blk.run(x2))


def test_two_blocks_of_a_stack_share_a_workspace():
    """A small stack: each block's stream feeds the next, one workspace for both; strided rows and an empty batch."""
    from kanjoos_b200.moe import MoeBlock
    H = 256
    banks = [on_device(bank_of(kd, 8, H, 128, 10 + i)) for i, kd in enumerate((BF16, E4M3))]
    ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    blocks = [MoeBlock(b, top_k=2, max_tokens=20, workspace=ws) for b in banks]
    g = torch.Generator()
    g.manual_seed(3)
    x = torch.randn((20, H), generator=g).to(BF16).cuda()
    wide = torch.zeros((20, H + 8), dtype=BF16, device="cuda")
    wide[:, :H] = x
    a = blocks[1].run(blocks[0].run(x))
    b = blocks[1].run(blocks[0].run(wide[:, :H]))
    assert torch.equal(a, b) and torch.isfinite(a.float()).all()
    assert blocks[0].run(x[:0]).shape == (0, H)
    one = torch.cat([blocks[1].run(blocks[0].run(x[i:i + 1])) for i in range(20)])
    # a row alone meets other tile shapes than in a batch: f32 sums in another order, then the same bf16 roundings
    assert float((one.float() - a.float()).norm() / a.float().norm()) < 2.0 ** -7


@pytest.mark.parametrize("ftype,e4m3", [("f16", False), ("bf16", False), ("bf16", True)])
def test_block_fed_from_a_gguf_file(tmp_path, ftype, e4m3):
    gguf = pytest.importorskip("gguf")
    from kanjoos_b200 import gguf_bank
    from kanjoos_b200.moe import MoeBlock
    from test_moe_block_cpu import write_float_file
    E, H, F, K = 8, 256, 128, 2
    arrays = write_float_file(tmp_path / "f.gguf", gguf, E, H, F, K, ftype)
    bank, k = gguf_bank.load_float_expert_bank(gguf_bank.GgufFile(str(tmp_path / "f.gguf")), 0, e4m3=e4m3)
    assert k == K and bank.post_norm is not None
    if not e4m3:
        assert np.array_equal(bank.gate.cpu().view(torch.int16).numpy().view(np.uint16), arrays["gate"])
    g = torch.Generator()
    g.manual_seed(4)
    x = torch.randn((6, H), generator=g)
    out, pe, pw = MoeBlock(bank, top_k=k, max_tokens=8).run(x.cuda(), return_routing=True)
    from dataclasses import fields, replace
    host = replace(bank, **{f.name: getattr(bank, f.name).cpu() for f in fields(bank) if torch.is_tensor(getattr(bank, f.name))})
    kind = E4M3 if e4m3 else F16 if ftype == "f16" else BF16
    s, _, _, _ = block_64(host, x, pe.cpu(), pw.cpu(), k, kind)
    tol = {BF16: 2.0 ** -8, F16: 2.0 ** -10, E4M3: 2.0 ** -6}[kind]
    size = s.abs() + (s - x.double()).square().mean(1, keepdim=True).sqrt()
    ref.check(out, s, tol * size + ref.held(s, F32), "stream")
