"""The MoE block of a decode step in one launch against the block in 64 bits: every type of experts, one to sixteen tokens, sizes at
which tiles, steps, panels and thread blocks end inside a run, and everything that a block may have around its experts."""
from dataclasses import replace

import pytest
import torch

import block_ops_ref as ref
import moe_decode_ref as dr
from test_gpu_block_ops import strided
from test_gpu_moe_block import BF16, E4M3, F16, F32, bank_of, on_device

pytestmark = pytest.mark.gpu
I8 = torch.int8
KINDS = [BF16, F16, E4M3, I8]


def bank(kind, E, H, F, seed, post=True, gate=True):
    b = bank_of(F16 if kind == F16 else BF16, E, H, F, seed, post, gate)
    return b.to_e4m3() if kind == E4M3 else b.to_int8() if kind == I8 else b


def rows(T, H, seed, dtype=F32):
    return torch.randn((T, H), generator=torch.Generator().manual_seed(seed)).to(dtype)


def run(b, x, k, blk=None, **kw):
    from kanjoos_b200.moe import MoeBlock
    blk = blk or MoeBlock(on_device(b), top_k=k, max_tokens=16)
    got = blk.decode(x, return_routing=True, **kw)
    blk.status()
    return got


def compare(b, x, k, got, next_w=None, gate=None):
    out, h, pe, pw = got if next_w is not None else (got[0], None, got[1], got[2])
    pe, pw, xc = pe.cpu(), pw.cpu(), x.cpu()
    dr.check_routing(b, xc, pe, pw, k)
    s, es, hs, eh = dr.block(b, xc, pe, pw, k, next_w, gate)
    ref.check(out, s, es + ref.held(s.abs() + es, out.dtype), "stream")
    if out.dtype == F32:   # and on the whole: the planes' errors are independent, 2^-16 at most and a third of that in the mean, in each of two products
        off = (out.double().cpu() - s).square().mean().sqrt()
        assert off <= 2.0 ** -15 * (s - b.beta * xc.double()).square().mean().sqrt() + 2.0 ** -23 * s.square().mean().sqrt()
    if h is not None and not isinstance(h, tuple):
        ref.check(h, hs, eh + ref.held(hs.abs() + eh, h.dtype), "next block's rows")
    return s, es, hs, eh


SHAPES = [(16, 512, 256, 4), (8, 256, 272, 8), (200, 256, 48, 8), (256, 256, 16, 8), (4, 256, 16, 1), (3, 768, 1040, 2)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("E,H,F,k", SHAPES)
@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 16])
def test_block_against_64_bits(kind, E, H, F, k, T):
    b = bank(kind, E, H, F, T + H)
    x = rows(T, H, T, [F32, BF16, F16][T % 3])
    w = torch.linspace(0.5, 1.5, H).to(BF16)
    compare(b, x, k, run(b, x.cuda(), k, next_norm=w.cuda(), next_dtype=F32), w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 5, 16])
def test_full_size_layer(kind, T):
    b = bank(kind, 128, 2048, 768, 3)
    x = rows(T, 2048, T)
    compare(b, x, 8, run(b, x.cuda(), 8))


@pytest.mark.parametrize("kind", [BF16, I8])
@pytest.mark.parametrize("T,E,H,F,k", [(16, 2, 8192, 64, 1), (3, 2, 32768, 32, 2), (16, 2, 256, 8208, 2), (2, 1, 256, 40960, 1), (7, 2, 16384, 48, 1)])
def test_rows_that_the_panel_takes_in_passes(kind, T, E, H, F, k):
    """Long rows: an expert's tokens go through in passes, down to one at a time."""
    b = bank(kind, E, H, F, 7)
    x = rows(T, H, 1)
    compare(b, x, k, run(b, x.cuda(), k))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [9, 16])
def test_all_tokens_at_the_same_experts(kind, T):
    b = bank(kind, 32, 512, 240, 11)
    b = replace(b, router_bias=torch.full((32,), -100.0).index_fill_(0, torch.tensor([0, 17, 31]), 100.0))
    x = rows(T, 512, 2)
    got = run(b, x.cuda(), 3)
    assert sorted(set(got[1].tolist())) == [0, 17, 31]
    compare(b, x, 3, got)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_masked_experts(kind):
    """A bias of -inf: fewer experts than top_k are left (the others weigh nothing), then none at all (the block adds nothing)."""
    b = bank(kind, 16, 256, 64, 5)
    x = rows(4, 256, 3)
    bias = torch.full((16,), float("-inf"))
    bias[[3, 9]] = 0.0
    out, pe, pw = run(replace(b, router_bias=bias), x.cuda(), 4)
    pe, pw = pe.cpu().view(4, 4), pw.cpu().view(4, 4)
    assert (pe[:, :2].sort(1).values == torch.tensor([3, 9])).all() and (pw[:, 2:] == 0).all()
    s, es, _, _ = dr.block(b, x, pe.reshape(-1), pw.reshape(-1), 4)
    ref.check(out, s, es + ref.held(s, F32), "two experts")
    out, pe, pw = run(replace(b, router_bias=torch.full((16,), float("-inf"))), x.cuda(), 4)
    assert (pw == 0).all()
    ref.check(out, b.beta * x.double(), 2.0 ** -23 * (b.beta * x.double()).abs(), "none")


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_any_alignment_and_outputs_between_others(kind):
    b = bank(kind, 8, 256, 80, 9)
    x = rows(6, 256, 4)
    for dtype, pad in ((F32, 1), (BF16, 3), (F16, 8)):
        xd = x.to(dtype)
        wide = torch.full((6, 260), -7.0, dtype=dtype, device="cuda")
        part = wide[:, 1:257]
        out, pe, pw = run(b, strided(xd.cuda(), pad), 2, out=part)
        assert out is part and (wide[:, 0] == -7).all() and (wide[:, 257:] == -7).all()
        compare(b, xd, 2, (out, pe, pw))


@pytest.mark.parametrize("gates", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("norms", [(False, False), (True, False), (False, True), (True, True)])
def test_what_a_block_has_around_its_experts(gates, norms):
    T, H, k = 5, 512, 2
    b = bank(BF16, 8, H, 96, 13, post=norms[1], gate=gates == "channel")
    b = replace(b, pre_norm=b.pre_norm.float() if norms[0] else None, post_norm=b.post_norm.float() if norms[1] else None, gate_sigmoid=gates != "row")
    x = rows(T, H, 5)
    g = {"row": rows(T, 1, 6), "full": rows(T, H, 7, F16)}.get(gates)
    w = rows(1, H, 8)[0]
    compare(b, x, k, run(b, x.cuda(), k, gate=None if g is None else g.cuda(), next_norm=w.cuda(), next_dtype=BF16), w, g)


def test_e4m3_rows_for_the_next_block():
    T, H, k = 9, 768, 4
    b = bank(I8, 16, H, 128, 17)
    x = rows(T, H, 9, BF16)
    w = torch.linspace(0.5, 1.5, H).to(BF16)
    out, (q, sc), pe, pw = run(b, x.cuda(), k, next_norm=w.cuda(), next_dtype=E4M3)
    s, es, h, eh = dr.block(b, x, pe.cpu(), pw.cpu(), k, w)
    most, slack = (v.abs().unflatten(-1, (-1, 128)).amax(-1) for v in (h, eh))
    ref.check(sc, most / 448, slack / 448 + 3 * 2.0 ** -24 * most / 448, "scales")
    held = sc.double().cpu().repeat_interleave(128, 1)
    # half a step of e4m3: 2^-4 relative, 2^-10 of the scale below the normal range
    ref.check(ref.rows_value(q.cpu(), sc.cpu()), h, eh + 2.0 ** -4 * (h.abs() + eh) * (1 + 2.0 ** -20) + 2.0 ** -10 * held, "codes")


@pytest.mark.parametrize("kind", KINDS)
def test_rows_stand_for_themselves(kind):
    """A NaN, an infinity, zeros and rows near the ends of the f32 range: the other tokens' bits do not change."""
    H, k = 512, 3
    b = bank(kind, 8, H, 112, 19)
    x = rows(8, H, 10)
    blk_x = x.clone()
    blk_x[1, 5], blk_x[3, 7] = float("nan"), float("inf")
    blk_x[4] = 0
    blk_x[5] *= 1e25
    blk_x[6] *= 1e-25
    base, got = run(b, x.cuda(), k)[0].cpu(), run(b, blk_x.cuda(), k)
    out = got[0].cpu()
    assert torch.isnan(out[1]).any() and not torch.isfinite(out[3]).all()
    for t in (0, 2, 7):
        assert torch.equal(out[t], base[t]), t
    keep = [4, 5, 6]
    pe, pw = (v.cpu().view(8, k)[keep].reshape(-1) for v in got[1:])
    c = replace(b, beta=0.0)   # the stream of the huge row hides the block's part; its norm does not
    out0 = run(c, blk_x.cuda(), k)[0].cpu()
    s, es, _, _ = dr.block(c, blk_x[keep], pe, pw, k)
    # a row whose squares leave the f32 range does without eps, which does not count there; of tiny rows eps is all there is
    ref.check(out0[keep], s, es + 2.0 ** -22 * s.abs() + 2.0 ** -100, "extreme rows")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,F", [(512, 208), (1024, 1040), (2304, 48), (256, 4160)])
def test_a_token_has_the_same_bits_at_any_place(kind, H, F):
    """Up to sixteen tokens of an expert, in tiles of sixteen rows and of eight: alone, in front of or behind others."""
    from kanjoos_b200.moe import MoeBlock
    T, k = 16, 2
    blk = MoeBlock(on_device(bank(kind, 3, H, F, 34)), top_k=k, max_tokens=T)
    x = rows(T, H, 92).cuda()
    want, pe, pw = blk.decode(x, return_routing=True)
    assert pe.bincount().max() > 8
    for a, b in [(i, i + 1) for i in range(T)] + [(0, 5), (3, 12), (9, 16), (5, 14)]:
        out, e, w = blk.decode(x[a:b], return_routing=True)
        assert torch.equal(e, pe[a * k:b * k]) and torch.equal(w, pw[a * k:b * k])
        assert torch.equal(out, want[a:b]), (a, b)
    turned = blk.decode(x.flip(0))
    assert torch.equal(turned.flip(0), want)


@pytest.mark.parametrize("kind", KINDS)
def test_same_bits_again_in_place_captured_and_on_another_stream(kind):
    from kanjoos_b200.moe import MoeBlock
    T, H, k = 12, 512, 4
    blk = MoeBlock(on_device(bank(kind, 24, H, 208, 21)), top_k=k, max_tokens=64)
    ins = [rows(T, H, 30 + i).cuda() for i in range(3)]
    want = [blk.decode(v) for v in ins]
    for v, w in zip(ins, want):
        for _ in range(5):
            assert torch.equal(blk.decode(v), w)
    y = ins[0].clone()
    assert blk.decode(y, out=y) is y and torch.equal(y, want[0])
    x = ins[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = blk.decode(x)
        for v, w in list(zip(ins, want)) * 2:
            x.copy_(v)
            graph.replay()
            blk.status()
            assert torch.equal(out, w)
    torch.cuda.current_stream().wait_stream(side)
    # a block of many tokens and the decode step take turns over one workspace
    many = rows(50, H, 40).cuda()
    first = blk.run(many)
    assert torch.equal(blk.decode(ins[1]), want[1]) and torch.equal(blk.run(many), first) and torch.equal(blk.decode(ins[2]), want[2])


def test_two_launches_at_once():
    """Blocks with workspaces of their own on two streams: each launch takes every SM, so they run one behind the other."""
    from kanjoos_b200.moe import MoeBlock
    H, k = 512, 2
    d = on_device(bank(BF16, 16, H, 256, 23))
    blks = [MoeBlock(d, top_k=k) for _ in range(2)]
    ins = [rows(4, H, 50 + i).cuda() for i in range(2)]
    want = [blk.decode(v) for blk, v in zip(blks, ins)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i & 1]):
            got.append((i & 1, blks[i & 1].decode(ins[i & 1])))
    torch.cuda.synchronize()
    for j, v in got:
        assert torch.equal(v, want[j])
    for blk in blks:
        blk.status()


@pytest.mark.parametrize("barrier", [1, 2])
def test_a_barrier_that_gives_up(barrier):
    from kanjoos_b200 import _lib
    from kanjoos_b200.moe import MoeBlock
    L = _lib.lib()
    T, H, k = 3, 256, 2
    blk = MoeBlock(on_device(bank(BF16, 8, H, 64, 25)), top_k=k)
    x, w = rows(T, H, 60).cuda(), torch.ones(H, dtype=BF16, device="cuda")
    want = blk.decode(x, next_norm=w)
    L.knj_decode_wait_limit(1 << 22)   # two milliseconds
    L.knj_moe_block_decode_test_stall(barrier)
    try:
        out, (q, s) = blk.decode(x, next_norm=w, next_dtype=E4M3)
        with pytest.raises(_lib.KnjError) as e:
            blk.status()
        assert e.value.code == -5
        assert torch.isnan(out).all() and torch.isnan(q.float()).all() and torch.isnan(s).all()
    finally:
        L.knj_moe_block_decode_test_stall(0)
        L.knj_decode_wait_limit(0)
    again = blk.decode(x, next_norm=w)
    blk.status()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_run_and_decode_agree():
    """run rounds the rows and the activations to bf16, half a step of which is 2^-8 of each value: it stays within the bound of the
    block in 64 bits whose values come with that error in place of the planes', and decode does so all the more."""
    from kanjoos_b200.moe import MoeBlock
    T, H, k = 7, 512, 4
    b = bank(BF16, 16, H, 256, 27)
    b = replace(b, router_bias=torch.arange(16.0) * 3)   # the same experts for all tokens: no routing on the edge
    blk = MoeBlock(on_device(b), top_k=k)
    x = rows(T, H, 70)
    d, pe, pw = blk.decode(x.cuda(), return_routing=True)
    r, pe2, pw2 = blk.run(x.cuda(), return_routing=True)
    assert torch.equal(pe, pe2)
    # the weights, too, come from rounded rows: that much the sums of the experts move
    s, es, _, _ = dr.block(b, x, pe.cpu(), pw.cpu(), k, planes=2.0 ** -8)
    s2, es2, _, _ = dr.block(b, x, pe.cpu(), pw2.cpu(), k, planes=2.0 ** -8)
    ref.check(d, s, es + ref.held(s, F32), "decode")
    ref.check(r, s2, es2 + ref.held(s2, F32), "run")


@pytest.mark.parametrize("kind", [BF16, I8])
def test_experts_rows_and_outputs_beyond_32_bits(kind):
    """The last experts' matrices and the last rows lie more than 2^31 elements behind the first."""
    from kanjoos_b200.moe import FloatExpertBank, MoeBlock
    from test_gpu_block_ops_use import far
    E, H, F, T, ld = 132, 4096, 4096, 3, 1 << 30
    assert (E - 3) * H * F > 1 << 31 and (T - 1) * ld >= 1 << 31
    few = bank(kind, 3, H, F, 31)
    full = {}
    for n in ("gate", "up", "down"):
        m = getattr(few, n)
        full[n] = torch.empty((E, *m.shape[1:]), dtype=m.dtype, device="cuda")
        full[n][E - 3:] = m.cuda()
        sc = getattr(few, n + "_scale")
        if sc is not None:
            full[n + "_scale"] = torch.zeros((E, *sc.shape[1:]), device="cuda")
            full[n + "_scale"][E - 3:] = sc.cuda()
    router = torch.zeros((E, H), dtype=BF16)
    router[E - 3:] = few.router
    bias = torch.full((E,), float("-inf"))
    bias[E - 3:] = 0.0
    big = FloatExpertBank(**full, router=router.cuda(), router_bias=bias.cuda(), pre_norm=few.pre_norm.cuda())
    x = rows(T, H, 90, BF16)
    wide, out = far(T, H, ld, BF16), far(T, H, ld, F32)
    wide.copy_(x)
    blk = MoeBlock(big, top_k=2)
    got, pe, pw = blk.decode(wide, out=out, return_routing=True)
    blk.status()
    assert got is out and (pe >= E - 3).all()
    small = replace(few, router_bias=torch.zeros(3), post_norm=None, out_gate=None, alpha=1.0, beta=1.0)
    compare(small, x, 2, (got, pe - (E - 3), pw))


def test_status_word_and_workspace_of_ones_own():
    """Nothing in the workspace or the status word has to be cleared before the first launch, nor after a launch of another block."""
    from kanjoos_b200.moe import MoeBlock
    H, k = 256, 2
    a, b = (MoeBlock(on_device(bank(kind, 8, H, 64, 33)), top_k=k) for kind in (BF16, E4M3))
    need = max(a.workspace.numel(), b.workspace.numel())
    a, b = (MoeBlock(m.bank, top_k=k, max_tokens=64, workspace=torch.full((8 * need,), 0xA5, dtype=torch.uint8, device="cuda")) for m in (a, b))
    shared = [MoeBlock(m.bank, top_k=k, workspace=a.workspace) for m in (a, b)]
    x = rows(3, H, 91).cuda()
    want = [a.decode(x), b.decode(x)]
    for _ in range(3):
        for m, w in zip(shared, want):
            m._status.fill_(77)
            assert torch.equal(m.decode(x), w)
            m.status()
            m.run(x)


def test_refusals():
    from kanjoos_b200.moe import MoeBlock
    blk = MoeBlock(on_device(bank(BF16, 8, 256, 64, 29)), top_k=2, max_tokens=32)
    x = rows(17, 256, 80).cuda()
    with pytest.raises(ValueError, match="at most 16"):
        blk.decode(x)
    assert blk.run(x).shape == (17, 256)
    assert blk.decode(x[:0]).shape == (0, 256)
    with pytest.raises(ValueError, match="rows of 256"):
        blk.decode(x[:4, :128])
    small = MoeBlock(blk.bank, top_k=2, max_tokens=4)
    with pytest.raises(ValueError, match="at most 4"):
        small.decode(x[:5])
