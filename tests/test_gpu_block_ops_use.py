"""The operators around an MoE block as programs call them: tables that name pairs again and again, offsets beyond 32 bits, calls
captured into graphs and replayed, calls on two streams at once, and operands that are refused before anything is launched."""
from dataclasses import replace

import pytest
import torch

import block_ops_ref as ref
from test_gpu_block_ops import BF16, E4M3, F16, F32, form, gen  # noqa: F401
from test_gpu_moe_block import bank_of, on_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("kind", ["gateup", "proj"])
def test_tables_that_name_pairs_many_times(kind, dtype, form):
    """More tiles than the number of pairs says: every form walks over them with the CTAs it has."""
    from kanjoos_b200 import ops
    g = gen("again", kind, dtype)
    E, N, K, P, stride = 2, 272, 1024, 40, 3000
    mats = [ref.matrix((E, N, K), g, dtype) for _ in range(2)]
    x = torch.randn((P, K), generator=g).to(BF16)
    xv = ref.rows_value(*ref.fp8_rows(x)) if dtype == E4M3 else x.double()
    idx = torch.zeros((E, stride), dtype=torch.int32)
    idx[1] = torch.arange(stride) % P
    cnt = torch.tensor([0, stride], dtype=torch.int32)
    md = [m[0].cuda() for m in mats]
    sc = [None if m[1] is None else m[1].cuda() for m in mats]
    mv = [ref.matrix_value(*m)[1] for m in mats]
    if kind == "gateup":
        one = torch.arange(P, dtype=torch.int32)[None]
        want, err, _ = ref.gateup(xv, mv[0][None], mv[1][None], one, torch.tensor([P]), lambda p: p, P)
        got = ops.expert_gateup(x.cuda(), md[0], md[1], idx.cuda(), cnt.cuda(), P, 1, gate_scale=sc[0], up_scale=sc[1], out_dtype=F32)
    else:
        want, err = ref.product(xv, mv[0])
        got = ops.expert_proj(x.cuda(), md[0], idx.cuda(), cnt.cuda(), P, scale=sc[0])
    ref.check(got, want, err + ref.held(want.abs() + err, F32), kind)


def far(rows, cols, ld, dtype):
    """rows x cols, ld elements from row to row; what lies between is not initialised."""
    esz = torch.empty(0, dtype=dtype).element_size()
    return torch.empty((rows - 1) * ld * esz + cols * esz, dtype=torch.uint8, device="cuda").view(dtype).as_strided((rows, cols), (ld, 1))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_experts_rows_and_outputs_beyond_32_bits(dtype, form):
    from kanjoos_b200 import ops
    g = gen("far", dtype)
    E, N, K, P, ld = 130, 4096, 4096, 40, 1 << 26
    assert (E - 1) * N * K > 1 << 31 and (P - 1) * ld > 1 << 31
    w1, s1 = ref.matrix((1, N, K), g, dtype)
    w = torch.empty((E, N, K), dtype=dtype, device="cuda")
    w[E - 1] = w1[0].cuda()
    sc = None
    if dtype == E4M3:
        sc = torch.zeros((E, *s1.shape[1:]), device="cuda")
        sc[E - 1] = s1[0].cuda()
    x16 = torch.randn((P, K), generator=g).to(BF16)
    xv = ref.rows_value(*ref.fp8_rows(x16)) if dtype == E4M3 else x16.double()
    x, xs = x16.cuda(), None
    if dtype == E4M3:
        x, xs = ops.fp8_rows(x)
    wide = far(P, K, ld, dtype)
    wide.view(torch.uint8 if dtype == E4M3 else torch.int16).copy_(x.view(torch.uint8 if dtype == E4M3 else torch.int16))
    idx = torch.zeros((E, P), dtype=torch.int32, device="cuda")
    idx[E - 1] = torch.arange(P)
    cnt = torch.zeros(E, dtype=torch.int32, device="cuda")
    cnt[E - 1] = P
    out = far(P, N, ld, BF16)
    ops.expert_proj(wide, w, idx, cnt, P, scale=sc, a_scale=xs, out=out)
    want, err = ref.product(xv, ref.matrix_value(w1, s1)[0])
    ref.check(out, want, err + ref.held(want.abs() + err, BF16), "far")


def test_norm_and_rows_beyond_32_bits():
    """Few rows, many rows (through the ring) and rows of an odd width, in place; the same bits as over dense rows."""
    from kanjoos_b200 import ops
    for T, H, ld in ((40, 512, 1 << 26), (700, 2048, 1 << 22), (700, 2047, 1 << 22)):
        g = gen("far norm", T, H)
        x, y = (torch.randn((T, H), generator=g).to(BF16).cuda() for _ in range(2))
        w = torch.randn(H, generator=g).to(BF16).cuda()
        want = ops.block_norm(x, y, post_w=w, gate=y, pre_w=w, norm_dtype=E4M3)
        q = ops.fp8_rows(x)
        xw, yw = far(T, H, ld, BF16), far(T, H, ld, BF16)
        xw.copy_(x)
        yw.copy_(y)
        q2 = ops.fp8_rows(xw)
        assert torch.equal(q[0].view(torch.uint8), q2[0].view(torch.uint8)) and torch.equal(q[1], q2[1])
        s, h = ops.block_norm(xw, yw, post_w=w, gate=yw, pre_w=w, norm_dtype=E4M3, stream_out=xw)
        assert s is xw and torch.equal(xw, want[0])
        assert torch.equal(h[0].view(torch.uint8), want[1][0].view(torch.uint8)) and torch.equal(h[1], want[1][1])


def run_all(ops, x, w, sc, wb, idx, cnt, norm_w):
    """Every operator once, fed from one another: (stream, rows of the next block, dense product)."""
    P = idx.shape[1]
    _, (q, qs) = ops.block_norm(x, pre_w=norm_w, norm_dtype=E4M3)
    act = ops.expert_gateup(q, w, w, idx, cnt, P, 1, gate_scale=sc, up_scale=sc, x_scale=qs)
    y = ops.expert_proj(act, wb, idx, cnt, P, out_dtype=BF16)
    s, h = ops.block_norm(x, y, post_w=norm_w, gate=norm_w, gate_sigmoid=True, pre_w=norm_w)
    return s, h, ops.fp8_matmul(w[1], sc[1], h)


def operands(T):
    g = gen("use", T)
    E, H = 3, 512
    w, sc = ref.matrix((E, H, H), g, E4M3)
    wb, _ = ref.matrix((E, H, H), g, BF16)
    idx, cnt = ref.tables([T // 2, 0, T - T // 2], g, stride=T)
    return [t.cuda() for t in (w, sc, wb, idx, cnt, torch.randn(H, generator=g).to(BF16))], g


@pytest.mark.parametrize("T", [1, 37, 900])
def test_captured_and_replayed(T, form):
    """One graph of all operators, replayed over changed inputs and on another stream, interleaved with a second graph."""
    from kanjoos_b200 import ops
    o, g = operands(T)
    xs = [torch.randn((T, 512), generator=g).to(BF16).cuda() for _ in range(4)]
    want = [run_all(ops, x, *o) for x in xs]
    torch.cuda.synchronize()
    graphs, ins, outs = [], [], []
    for _ in range(2):
        x = xs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run_all(ops, x, *o)
        graphs.append(gr), ins.append(x), outs.append(out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(4):
            for k in range(2):
                ins[k].copy_(xs[(i + k) % 4])
                graphs[k].replay()
            for k in range(2):
                for a, b in zip(outs[k], want[(i + k) % 4]):
                    assert torch.equal(a, b), (i, k)
    side.synchronize()


@pytest.mark.parametrize("T", [1, 300])
def test_two_streams_at_once(T, form):
    from kanjoos_b200 import ops
    o, g = operands(T)
    xs = [torch.randn((T, 512), generator=g).to(BF16).cuda() for _ in range(2)]
    want = [run_all(ops, x, *o) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(25):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(run_all(ops, xs[k], *o))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            for a, b in zip(out, want[k]):
                assert torch.equal(a, b)


def test_operands_that_are_refused():
    from kanjoos_b200 import ops
    from kanjoos_b200.moe import MoeBlock
    (w, sc, wb, idx, cnt, norm_w), _ = operands(8)
    x = torch.randn((8, 512), device="cuda").to(BF16)
    for bad in (x.t().contiguous().t(), x[:1].expand(8, 512), x.cpu(), x.long(), x[0], x[:, ::2]):
        with pytest.raises(ValueError):
            ops.fp8_rows(bad)
        with pytest.raises(ValueError):
            ops.expert_proj(bad, wb, idx, cnt, 8)
        with pytest.raises((ValueError, IndexError)):
            ops.block_norm(bad, x, pre_w=norm_w)
        with pytest.raises((ValueError, IndexError)):
            ops.block_norm(x, bad, pre_w=norm_w)
    for args, kw in (((x, wb.cpu(), idx, cnt, 8), {}), ((x, wb.transpose(1, 2), idx, cnt, 8), {}), ((x, wb, idx.long(), cnt, 8), {}),
                     ((x, wb, idx[:2], cnt, 8), {}), ((x, wb, idx, cnt[:2], 8), {}), ((x, wb, idx, cnt, 8), dict(scale=sc)),
                     ((x, w, idx, cnt, 8), {}), ((x, w, idx, cnt, 8), dict(scale=sc.half())), ((x, w, idx, cnt, 8), dict(scale=sc[:, :2])),
                     ((x, wb, idx, cnt, 8), dict(out=torch.empty((8, 511), device="cuda"))), ((x, wb, idx, cnt, 8), dict(out_dtype=torch.int32)),
                     ((x, wb, idx, cnt, 8), dict(pair_row=torch.zeros(7, dtype=torch.int32, device="cuda")))):
        with pytest.raises(ValueError):
            ops.expert_proj(*args, **kw)
    for bad in ((w[0], sc[0].half(), x), (w[0], sc[0][:2], x), (wb[0], sc[0], x), (w[0], sc[0].cpu(), x), (w[0], sc[0], x[:, :256])):
        with pytest.raises(ValueError):
            ops.fp8_matmul(*bad)
    bank = on_device(bank_of(E4M3, 4, 256, 64, 3))
    for name, value in (("pre_norm", bank.pre_norm.cpu()), ("post_norm", bank.post_norm.cpu()), ("out_gate", bank.out_gate.cpu()),
                        ("router_bias", bank.router_bias.cpu()), ("down_scale", bank.down_scale.double()), ("gate_scale", None),
                        ("router", bank.router.cpu()), ("pre_norm", bank.pre_norm.float()), ("up", bank.up[:, :32])):
        with pytest.raises(ValueError):
            MoeBlock(replace(bank, **{name: value}), top_k=2, max_tokens=4)
    for ws in (torch.empty(1 << 22, dtype=torch.uint8), torch.empty(64, dtype=torch.uint8, device="cuda"),
               torch.empty(1 << 22, dtype=torch.uint8, device="cuda")[1:]):
        with pytest.raises(ValueError):
            MoeBlock(bank, top_k=2, max_tokens=4, workspace=ws)


@pytest.mark.parametrize("T,H,st,yt,wt,gate,sig,post,pre,ht", [
    (3, 129, BF16, F32, BF16, "channel", True, True, True, E4M3), (700, 513, BF16, BF16, F32, "row", True, True, True, E4M3),
    (2, 4095, F32, BF16, BF16, "full", True, True, True, F16), (2, 4097, BF16, F16, BF16, None, False, True, True, E4M3),
    (1, 16383, BF16, BF16, BF16, "channel", True, True, True, E4M3), (2, 16385, F16, BF16, BF16, "full", False, True, True, E4M3),
    (3, 30001, F32, None, F32, None, False, False, True, BF16), (5, 9999, BF16, BF16, BF16, "row", False, False, False, None),
])
@pytest.mark.parametrize("pad", [0, 3])
def test_norms_of_any_width(T, H, st, yt, wt, gate, sig, post, pre, ht, pad):
    from test_gpu_block_ops import test_block_norm
    test_block_norm(T, H, st, yt, wt, gate, sig, post, pre, ht, pad)


def test_special_rows_of_any_width():
    """Squares beyond the f32 range, zeros and a NaN, in rows without 16-byte units: each stays in its row."""
    from kanjoos_b200 import ops
    for H in (1001, 5003):
        x = torch.ones((4, H), device="cuda")
        x[0] *= 1e30
        x[1] = 0.0
        x[2, 7] = float("nan")
        w = torch.ones(H, device="cuda")
        s, h = ops.block_norm(x, x, post_w=w, pre_w=w, norm_dtype=F32, alpha=2.0)
        # the mean square is 1e60: n = 1 up to roundings of 2^-24 in the scaled sum, its root and two products
        assert torch.equal(s[0], x[0]) and (h[0] - 1).abs().max() < 8 * H * 2.0 ** -24
        assert (s[1] == 0).all() and (h[1] == 0).all() and torch.isnan(h[2]).all()
        assert (s[3] - 3).abs().max() < 1e-3 and (h[3] - 1).abs().max() < 1e-3
