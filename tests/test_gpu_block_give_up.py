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
