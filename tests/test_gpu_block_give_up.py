"""Waits that run out in the operators around an MoE block: a hook withholds one arrival (the copy or the product itself completes), the
limit is a millisecond. What the kernel did not form is NaN, the status word is raised, everything else is right, and the next launch is
an ordinary one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def short_limit():
    from kanjoos_b200 import _lib
    L = _lib.lib()
    L.knj_decode_wait_limit(2_000_000)
    yield L
    L.knj_decode_wait_limit(0)


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("T,H,xt,with_y,h", [(3000, 512, BF16, True, BF16), (3000, 2048, BF16, True, E4M3), (9000, 1024, F32, False, F32),
                                             (700, 8200, BF16, True, E4M3), (400, 16384, F32, True, BF16)])
def test_norm_whose_row_never_lands(T, H, xt, with_y, h, short_limit):
    """The first CTA gives up in its first row: that row and all that it would have formed behind it are NaN, over several laps of the
    ring; no row of another CTA is touched."""
    from kanjoos_b200 import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    x = torch.randn((T, H), device="cuda", generator=g).to(xt)
    y = torch.randn((T, H), device="cuda", generator=g).to(BF16) if with_y else None
    w = torch.ones(H, dtype=BF16, device="cuda")

    def run(status):
        s, n = ops.block_norm(x, y, post_w=w if with_y else None, pre_w=w, norm_dtype=h, stream_dtype=xt, status=status)
        return (s.float(), n[0].float(), n[1]) if h == E4M3 else (s.float(), n.float())
    status = word()
    want = run(status)
    torch.cuda.synchronize()
    assert int(status) == 0
    short_limit.knj_block_norm_test_stall(1)
    try:
        got = run(status)
        torch.cuda.synchronize()
    finally:
        short_limit.knj_block_norm_test_stall(0)
    assert int(status) == 1
    bad = torch.isnan(got[0]).all(1).nonzero().flatten().tolist()
    assert bad[0] == 0 and len(bad) > 1 and bad == list(range(0, T, bad[1]))
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[bad] = False
    for a, b in zip(got, want):
        assert torch.isnan(a[~good]).all() and torch.equal(a[good], b[good])
    status.zero_()
    for a, b in zip(run(status), want):
        assert torch.equal(a, b)
    assert int(status) == 0


def test_status_words_that_are_refused():
    from kanjoos_b200 import ops
    x, w = torch.ones((2, 64), device="cuda"), torch.ones(64, device="cuda")
    for bad in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="status"):
            ops.block_norm(x, pre_w=w, status=bad)


def test_status_of_blocks_that_share_a_workspace(short_limit):
    """Each block answers for its own last run, whatever another block of other sizes and weights has run over the workspace since."""
    from kanjoos_b200._lib import KnjError
    from kanjoos_b200.moe import MoeBlock
    from test_gpu_moe_block import bank_of, on_device
    H = 256
    banks = [on_device(bank_of(kd, 8, H, 128, 10 + i)) for i, kd in enumerate((BF16, E4M3))]
    ws = torch.empty(1 << 25, dtype=torch.uint8, device="cuda")
    first, second = (MoeBlock(b, top_k=2, max_tokens=4000, workspace=ws) for b in banks)
    first.status()   # nothing has run
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    x = torch.randn((4000, H), device="cuda", generator=g).to(BF16)
    want = first.run(x[:7]).clone()
    second.run(x)
    second.status()
    first.status()
    assert int(first._status) == 0 and int(second._status) == 0
    short_limit.knj_block_norm_test_stall(1)
    try:
        out = first.run(x)      # 4000 rows: its norms go through the ring
    finally:
        short_limit.knj_block_norm_test_stall(0)
    second.run(x[:20])
    second.status()
    with pytest.raises(KnjError, match="gave up"):
        first.status()
    bad = torch.isnan(out.float()).all(1)
    assert bad[0] and 0 < int(bad.sum()) < 100
    assert torch.equal(first.run(x[:7]), want)
    first.status()


@pytest.fixture(params=[1, 2, 3], ids=["single", "pair", "split"])
def form(request):
    from kanjoos_b200 import _lib
    _lib.lib().knj_expert_tc_form(request.param)
    yield request.param
    _lib.lib().knj_expert_tc_form(0)


def stalled(L, what, call):
    """(outputs of an ordinary call, of one whose wait runs out, of an ordinary one behind it)"""
    want = call(None).float()
    torch.cuda.synchronize()
    L.knj_expert_tc_test_stall(what)
    try:
        status = word()
        got = call(status).float()
        torch.cuda.synchronize()
    finally:
        L.knj_expert_tc_test_stall(0)
    assert int(status) == 1
    status = word()
    again = call(status).float()
    assert int(status) == 0 and torch.equal(again, want)
    return want, got


@pytest.mark.parametrize("what", [1, 2, 3], ids=["accumulator", "operands", "last-accumulator"])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("kind", ["gateup", "proj"])
@pytest.mark.parametrize("size", ["few", "many"])
def test_expert_product_whose_wait_runs_out(kind, dtype, what, size, form, short_limit):
    """One tile per CTA (few) and several (many). NaN begins with a tile of the stalled CTA or of its pair or cluster; the rest is right and
    rows that no entry names stay as they were."""
    import block_ops_ref as ref
    from kanjoos_b200 import ops
    g = torch.Generator()
    g.manual_seed(7)
    E, N, K = (2, 256, 1024) if size == "few" else (6, 2048, 1024)
    counts = [20, 12] if size == "few" else [200, 0, 300, 64, 17, 120]
    P = sum(counts)
    idx, cnt = ref.tables(counts, g)
    mats = [ref.matrix((E, N, K), g, dtype) for _ in range(2)]
    md, sc = [m[0].cuda() for m in mats], [None if m[1] is None else m[1].cuda() for m in mats]
    x = torch.randn((P, K), generator=g).to(BF16).cuda()
    xs = None
    if dtype == E4M3:
        x, xs = ops.fp8_rows(x)
    idx, cnt = idx.cuda(), cnt.cuda()

    def call(status):
        out = torch.full((P + 3, N), 5.0, dtype=F32, device="cuda")
        if kind == "gateup":
            ops.expert_gateup(x, md[0], md[1], idx, cnt, P, 1, gate_scale=sc[0], up_scale=sc[1], x_scale=xs, out=out[:P], status=status)
        else:
            ops.expert_proj(x, md[0], idx, cnt, P, scale=sc[0], a_scale=xs, out=out[:P], status=status)
        return out
    want, got = stalled(short_limit, what, call)
    bad = torch.isnan(got)
    assert bad.any() and not bad.all() and not bad[P:].any()
    assert torch.equal(got[~bad], want[~bad])
    if what != 3:   # the first tile: the first outputs of the first expert's first rows
        assert bad[idx[0, 0].long(), 0]


@pytest.mark.parametrize("what", [1, 2, 3], ids=["accumulator", "operands", "last-accumulator"])
def test_dense_product_whose_wait_runs_out(what, form, short_limit):
    import block_ops_ref as ref
    from kanjoos_b200 import ops
    g = torch.Generator()
    g.manual_seed(8)
    w, sc = ref.matrix((1100, 1024), g, E4M3)
    w, sc, x = w.cuda(), sc.cuda(), torch.randn((600, 1024), generator=g).cuda()
    want, got = stalled(short_limit, what, lambda status: ops.fp8_matmul(w, sc, x, status=status))
    bad = torch.isnan(got)
    assert bad.any() and not bad.all() and torch.equal(got[~bad], want[~bad])


def test_block_whose_product_gives_up(form, short_limit):
    from kanjoos_b200._lib import KnjError
    from kanjoos_b200.moe import MoeBlock
    from test_gpu_moe_block import bank_of, on_device
    for kind in (BF16, E4M3):
        b = MoeBlock(on_device(bank_of(kind, 8, 256, 128, 3)), top_k=2, max_tokens=64)
        x = torch.randn((64, 256), device="cuda")
        want = b.run(x).clone()
        b.status()
        short_limit.knj_expert_tc_test_stall(1)
        try:
            b.run(x)
            with pytest.raises(KnjError, match="gave up"):
                b.status()
        finally:
            short_limit.knj_expert_tc_test_stall(0)
        assert torch.equal(b.run(x), want)
        b.status()


def test_status_words_of_products_that_are_refused():
    import block_ops_ref as ref
    from kanjoos_b200 import ops
    g = torch.Generator()
    w, sc = ref.matrix((64, 64), g, E4M3)
    x, idx, cnt = torch.ones((2, 64), device="cuda"), torch.tensor([[0, 1]], dtype=torch.int32).cuda(), torch.tensor([2], dtype=torch.int32).cuda()
    wb = torch.zeros((1, 64, 64), dtype=BF16, device="cuda")
    for bad in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        for call in (lambda: ops.fp8_matmul(w.cuda(), sc.cuda(), x, status=bad), lambda: ops.expert_proj(x.to(BF16), wb, idx, cnt, 2, status=bad),
                     lambda: ops.expert_gateup(x.to(BF16), wb, wb, idx, cnt, 2, 1, status=bad)):
            with pytest.raises(ValueError, match="status"):
                call()


@pytest.mark.parametrize("what", [1, 2, 3], ids=["accumulator", "operands", "last-accumulator"])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_a_cluster_with_several_tiles_whose_wait_runs_out(dtype, what, form, short_limit):
    """A table that names its pairs again and again makes more tiles than there are clusters, so that a split tile which gives up has
    others behind it. Which of a pair's many tiles wrote last is open: a right value, or NaN from a tile that was given up."""
    import block_ops_ref as ref
    from kanjoos_b200 import ops
    g = torch.Generator()
    g.manual_seed(11)
    E, N, K, P, stride = 2, 272, 1024, 40, 3000
    mats = [ref.matrix((E, N, K), g, dtype) for _ in range(2)]
    md, sc = [m[0].cuda() for m in mats], [None if m[1] is None else m[1].cuda() for m in mats]
    x, xs = torch.randn((P, K), generator=g).to(BF16).cuda(), None
    if dtype == E4M3:
        x, xs = ops.fp8_rows(x)
    idx = torch.zeros((E, stride), dtype=torch.int32)
    idx[1] = torch.arange(stride) % P
    idx, cnt = idx.cuda(), torch.tensor([0, stride], dtype=torch.int32).cuda()
    want, got = stalled(short_limit, what, lambda status: ops.expert_gateup(x, md[0], md[1], idx, cnt, P, 1, gate_scale=sc[0], up_scale=sc[1],
                                                                           x_scale=xs, out_dtype=F32, status=status))
    bad = torch.isnan(got)
    assert not torch.isnan(want).any() and torch.equal(got[~bad], want[~bad])
