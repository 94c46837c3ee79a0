"""int8 rows, the dense int8 product and the products grouped by expert, against their definitions in 64 bits."""
import ctypes as C

import pytest
import torch

import block_ops_ref as ref
import int8_ref as i8
from test_gpu_block_ops import BF16, EXPERTS, F16, F32, form, gen, strided  # noqa: F401
from test_gpu_block_ops_use import far

pytestmark = pytest.mark.gpu
I8 = torch.int8


# ------------------------------------------------------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,pad", [(1, 1, 0), (1, 8, 0), (3, 7, 0), (9, 256, 0), (8, 1024, 8), (17, 1032, 0), (5, 2048, 3), (2, 4096, 0), (3, 8200, 0),
                                     (2, 32768, 0), (2, 32776, 0), (4, 5001, 0), (700, 208, 0), (3000, 2048, 0)])
def test_rows_are_the_definitions_bits(n, k, pad, dtype):
    from kanjoos_b200 import ops
    g = gen("rows8", n, k, dtype)
    x = (torch.randn((n, k), generator=g) * torch.randn((n, 1), generator=g).exp()).to(dtype)
    want, scale = i8.rows(x)
    xd = x.cuda()
    q, s = ops.int8_rows(strided(xd, pad) if pad else xd)
    assert q.dtype == I8 and torch.equal(s.cpu(), scale) and torch.equal(q.cpu(), want)


@pytest.mark.parametrize("k", [64, 2048, 2049])
def test_special_rows(k):
    """Zeros, values below the normal range of the scale, the largest values, ties, NaN and infinities; each row stands for itself."""
    from kanjoos_b200 import ops
    x = torch.randn((9, k), generator=gen("special8", k))
    x[0] = 0
    x[1] *= 2.0 ** -120
    x[2] *= 3e37
    x[3, 1] = float("nan")
    x[4, k - 1] = float("-inf")
    x[5] = torch.arange(k).remainder(127) - 63.5
    x[5, 0] = 127.0
    x[6] = -0.0
    x[7] = torch.finfo(F32).max
    want, scale = i8.rows(x)
    q, s = ops.int8_rows(x.cuda())
    q, s = q.cpu(), s.cpu()
    assert torch.equal(q, want) and torch.equal(torch.nan_to_num(s, nan=-7.0), torch.nan_to_num(scale, nan=-7.0))
    assert torch.isnan(s[3]) and torch.isinf(s[4]) and (q[3:5] == 0).all() and (q[7] == 127).all()


# ---------------------------------------------------------------------------------------------------- dense product

@pytest.mark.parametrize("m,n,k,dtype,out,pad", [(1, 2048, 2048, BF16, F32, 0), (1, 1, 16, F32, F32, 0), (2, 100, 144, F16, BF16, 0),
                                                 (17, 128, 128, BF16, F16, 8), (64, 1000, 2064, F32, F32, 4), (65, 257, 400, BF16, BF16, 0),
                                                 (301, 1000, 2048, F16, F16, 0), (513, 384, 256, F16, F32, 0), (3, 4096, 4096, BF16, F32, 0),
                                                 (130, 130, 32784, BF16, F32, 0), (33, 96, 4080, BF16, F32, 0)])
def test_int8_matmul(m, n, k, dtype, out, pad, form):
    from kanjoos_b200 import ops
    g = gen(m, n, k)
    w, s = i8.matrix((n, k), g)
    x = torch.randn((m, k), generator=g).to(dtype)
    codes, scale = i8.rows(x)
    want, err = i8.product(codes, scale, w, s)
    xd = x.cuda()
    got = ops.int8_matmul(w.cuda(), s.cuda(), strided(xd, pad) if pad else xd, out_dtype=out)
    assert got.dtype == out
    ref.check(got, want, err + ref.held(want.abs() + err, out), "product")
    q, qs = ops.int8_rows(xd)
    wide = torch.full((m, k + 32), 77, dtype=I8, device="cuda")
    wide[:, :k] = q
    for rows in (q, wide[:, :k]):
        assert torch.equal(got, ops.int8_matmul(w.cuda(), s.cuda(), rows, qs, out_dtype=out)), "of rows in codes"


@pytest.mark.parametrize("n,k,pad", [(1, 16, 0), (7, 160, 3), (2048, 2048, 0), (1000, 4096, 8), (20011, 512, 1), (33, 5120, 0), (64, 5136, 0), (5, 20480, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_few_rows_have_the_bits_of_many(n, k, pad, dtype):
    """Each number of rows that a kernel is built for and those between, strided and at odd addresses, outputs of every type; a row's result
    does not depend on the rows around it."""
    from kanjoos_b200 import ops
    g = gen("few8", n, k, dtype)
    w, s = i8.matrix((n, k), g)
    w, s = w.cuda(), s.cuda()
    x = torch.randn((9, k), generator=g).to(dtype)
    x[2] = 0.0
    x[4, k // 2] = 1e4
    x = strided(x.cuda(), pad) if pad else x.cuda()
    q, qs = ops.int8_rows(x)
    for out in (F32, BF16, F16):
        want = ops.int8_matmul(w, s, q, qs, out_dtype=out)
        for m in (1, 2, 3, 4, 5, 7, 8, 9):
            assert torch.equal(ops.int8_matmul(w, s, x[:m], out_dtype=out), want[:m]), m
        for at in (1, 3):
            assert torch.equal(ops.int8_matmul(w, s, x[at:at + 5], out_dtype=out), want[at:at + 5])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_rows_that_are_not_finite(dtype):
    from kanjoos_b200 import ops
    g = gen("few nan8")
    w, s = i8.matrix((100, 304), g)
    x = torch.randn((8, 304), generator=g).to(dtype)
    clean = ops.int8_matmul(w.cuda(), s.cuda(), x.cuda()).cpu()
    x[1, 303], x[3, 0], x[6, 5] = float("nan"), float("inf"), float("-inf")
    got = ops.int8_matmul(w.cuda(), s.cuda(), x.cuda()).cpu()
    bad = [1, 3, 6]
    keep = [i for i in range(8) if i not in bad]
    assert torch.isnan(got[bad]).all() and torch.equal(got[keep], clean[keep])


def test_few_rows_write_their_rows_alone():
    """An output with a row stride of its own through the entry point: nothing between and behind the rows is written."""
    from kanjoos_b200 import _lib
    g = gen("few ld8")
    w, s = (t.cuda() for t in i8.matrix((37, 64), g))
    x = torch.randn((3, 64), generator=g).cuda()
    y = torch.full((6, 50), -77.0, device="cuda")
    a = _lib.Int8MatmulArgs(w=w.data_ptr(), w_scale=s.data_ptr(), n_in=64, n_out=37, x=x.data_ptr(), ldx=64, m=3, y=y.data_ptr(), ldy=50)
    _lib.check(_lib.lib().knj_int8_matmul_launch(C.byref(a), torch.cuda.current_stream().cuda_stream))
    from kanjoos_b200 import ops
    assert torch.equal(y[:3, :37], ops.int8_matmul(w, s, x))
    assert (y[3:] == -77.0).all() and (y[:, 37:] == -77.0).all()


def test_few_rows_of_a_matrix_beyond_32_bits():
    from kanjoos_b200 import ops
    n, k = 525000, 4096
    assert (n - 3) * k > 1 << 31
    g = gen("few far8")
    few, s3 = i8.matrix((3, k), g)
    w = torch.zeros((n, k), dtype=I8, device="cuda")
    s = torch.ones(n, device="cuda")
    w[-3:], s[-3:] = few.cuda(), s3.cuda()
    x = torch.randn((2, k), generator=g).cuda()
    got = ops.int8_matmul(w, s, x)
    assert torch.equal(got[:, -3:], ops.int8_matmul(few.cuda(), s3.cuda(), x)) and (got[:, :-3] == 0).all()


def test_sums_of_the_largest_codes(form):
    """Sums next to the end of 32 bits: every product 16384 or -16256, as many as the entry points take."""
    from kanjoos_b200 import ops
    k = 131056
    w = torch.full((20, k), -128, dtype=I8)
    x = torch.full((3, k), -128, dtype=I8)
    x[1] = 127
    x[2, ::2] = 127
    s = torch.ones(20)
    want, err = i8.product(x, torch.ones(3), w, s)
    assert want.abs().max() == 16384.0 * k
    got = ops.int8_matmul(w.cuda(), s.cuda(), x.cuda(), torch.ones(3).cuda())
    ref.check(got, want, err, "largest")


def test_non_finite_rows_of_the_product(form):
    from kanjoos_b200 import ops
    g = gen("nan8")
    w, s = i8.matrix((256, 384), g)
    x = torch.randn((20, 384), generator=g).to(BF16)
    clean = ops.int8_matmul(w.cuda(), s.cuda(), x.cuda()).cpu()
    x[3, 17] = float("nan")
    x[4, 383] = float("inf")
    s2 = s.clone()
    s2[9] = float("nan")
    got = ops.int8_matmul(w.cuda(), s2.cuda(), x.cuda()).cpu()
    assert torch.isnan(got[3:5]).all() and torch.isnan(got[:, 9]).all()
    keep = [i for i in range(20) if i not in (3, 4)]
    cols = [i for i in range(256) if i != 9]
    assert torch.equal(got[keep][:, cols], clean[keep][:, cols])


# --------------------------------------------------------------------------------------------------- expert products

def run_expert(kind, E, N, K, counts, out_t, dtype=BF16):
    from kanjoos_b200 import ops
    g = gen("8", kind, E, N, K)
    P, top_k = sum(counts), 3
    idx, cnt = ref.tables(counts, g, stride=max(counts) + 3)
    mats = [i8.matrix((E, N, K), g) for _ in range(2 if kind == "gateup" else 1)]
    if kind == "gateup":   # gates of a few units, not of hundreds
        mats = [(w, s * 0.01) for w, s in mats]
    x = torch.randn((-(-P // top_k) if kind == "gateup" else P, K), generator=g).to(dtype)
    codes, scale = i8.rows(x)
    md = [(w.cuda(), s.cuda()) for w, s in mats]
    out = torch.full((P + 2, N + 5), -12345.0, dtype=out_t, device="cuda")
    part = out[:P, :N]
    if kind == "gateup":
        want, err = i8.gateup(codes, scale, *mats[0], *mats[1], idx, cnt, lambda p: p // top_k, P)
        got = ops.expert_gateup(x.cuda(), md[0][0], md[1][0], idx.cuda(), cnt.cuda(), P, top_k, gate_scale=md[0][1], up_scale=md[1][1], out=part)
        # the same rows as codes, into an output with whole sectors
        dense = ops.expert_gateup(codes.cuda(), md[0][0], md[1][0], idx.cuda(), cnt.cuda(), P, top_k, gate_scale=md[0][1], up_scale=md[1][1],
                                  x_scale=scale.cuda(), out_dtype=out_t)
    else:
        want, err = i8.proj(codes, scale, *mats[0], idx, cnt, lambda p: p, P)
        got = ops.expert_proj(x.cuda(), md[0][0], idx.cuda(), cnt.cuda(), P, scale=md[0][1], out=part)
        dense = ops.expert_proj(codes.cuda(), md[0][0], idx.cuda(), cnt.cuda(), P, scale=md[0][1], a_scale=scale.cuda(), out_dtype=out_t)
    assert got is part
    ref.check(part, want, err + ref.held(want.abs() + err, out_t), kind)
    assert torch.equal(part, dense)
    out = out.cpu()
    assert (out[P:] == -12345.0).all() and (out[:, N:] == -12345.0).all(), "something outside the output was written"


@pytest.mark.parametrize("E,N,K,counts", [c for c in EXPERTS if c[2] % 16 == 0])
@pytest.mark.parametrize("kind", ["gateup", "proj"])
def test_expert_products(kind, E, N, K, counts, form):
    run_expert(kind, E, N, K, counts, {"gateup": BF16, "proj": F32}[kind])


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["gateup", "proj"])
def test_expert_output_types(kind, out, form):
    run_expert(kind, 3, 264, 288, [70, 0, 9], out, F16)


def test_unnamed_rows_bad_entries_and_row_maps(form):
    from kanjoos_b200 import ops
    g = gen("unnamed8")
    E, N, K, P = 3, 136, 272, 40
    w, sc = i8.matrix((E, N, K), g)
    codes, scale = i8.rows(torch.randn((12, K), generator=g))
    idx = torch.tensor([[0, 7, 7, -1], [3, P, 1 << 30, -5], [11, 12, 13, 39]], dtype=torch.int32)
    cnt = torch.tensor([3, 4, 9], dtype=torch.int32)
    row_map = torch.randint(0, 12, (P,), generator=g, dtype=torch.int32)
    row_map[12], row_map[13] = 12, -1                      # outside x
    out = torch.full((P, N), 7.0, dtype=F32, device="cuda")
    wide = torch.full((12, K + 16), 127, dtype=I8, device="cuda")
    wide[:, :K] = codes.cuda()
    ops.expert_proj(wide[:, :K], w.cuda(), idx.cuda(), cnt.cuda(), P, pair_row=row_map.cuda(), scale=sc.cuda(), a_scale=scale.cuda(), out=out)
    out = out.cpu()
    named = {0: 0, 7: 0, 3: 1, 11: 2, 12: 2, 13: 2, 39: 2}
    for p in range(P):
        if p not in named:
            assert (out[p] == 7.0).all(), p
        elif p in (12, 13):
            assert (out[p] == 0).all(), p
        else:
            r = int(row_map[p])
            want, err = i8.product(codes[r:r + 1], scale[r:r + 1], w[named[p]], sc[named[p]])
            ref.check(out[p][None], want, err + ref.held(want.abs(), F32), f"pair {p}")


def test_no_pairs_at_all(form):
    from kanjoos_b200 import ops
    w, sc = i8.matrix((4, 128, 128), gen("empty8"))
    w, sc = w.cuda(), sc.cuda()
    idx, cnt = torch.full((4, 6), -1, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    out = torch.full((6, 128), 3.0, dtype=F32, device="cuda")
    x = torch.randn((6, 128), device="cuda")
    ops.expert_proj(x, w, idx, cnt, 6, scale=sc, out=out)
    assert (out == 3.0).all()
    assert ops.expert_proj(x[:0], w, idx, cnt, 0, scale=sc).shape == (0, 128)
    assert ops.int8_matmul(w[0], sc[0], x[:0]).shape == (0, 128) and ops.int8_rows(x[:0])[0].shape == (0, 128)


def test_experts_rows_and_outputs_beyond_32_bits(form):
    from kanjoos_b200 import ops
    g = gen("far8")
    E, N, K, P, ld = 130, 4096, 4096, 40, 1 << 26
    assert (E - 1) * N * K > 1 << 31 and (P - 1) * ld > 1 << 31
    w1, s1 = i8.matrix((N, K), g)
    w = torch.empty((E, N, K), dtype=I8, device="cuda")
    w[E - 1] = w1.cuda()
    sc = torch.zeros((E, N), device="cuda")
    sc[E - 1] = s1.cuda()
    codes, scale = i8.rows(torch.randn((P, K), generator=g))
    wide = far(P, K, ld, I8)
    wide.copy_(codes.cuda())
    idx = torch.zeros((E, P), dtype=torch.int32, device="cuda")
    idx[E - 1] = torch.arange(P)
    cnt = torch.zeros(E, dtype=torch.int32, device="cuda")
    cnt[E - 1] = P
    out = far(P, N, ld, BF16)
    ops.expert_proj(wide, w, idx, cnt, P, scale=sc, a_scale=scale.cuda(), out=out)
    want, err = i8.product(codes, scale, w1, s1)
    ref.check(out, want, err + ref.held(want.abs() + err, BF16), "far")


def test_captured_replayed_and_on_another_stream(form):
    """Rows, dense and grouped product in one graph, replayed over other inputs; the same bits as called, and from run to run."""
    from kanjoos_b200 import ops
    g = gen("graph8")
    E, H, T = 3, 512, 75
    w, sc = i8.matrix((E, H, H), g)
    w, sc = w.cuda(), sc.cuda() * 0.01
    idx, cnt = (t.cuda() for t in ref.tables([30, 0, 45], g, stride=T))
    x = torch.randn((T, H), generator=g).to(BF16).cuda()

    def step(x):
        a = ops.expert_gateup(x, w, w, idx, cnt, T, 1, gate_scale=sc, up_scale=sc)
        return ops.int8_matmul(w[1], sc[1], ops.expert_proj(a, w, idx, cnt, T, scale=sc, out_dtype=BF16))

    ins = [torch.randn((T, H), generator=g).to(BF16).cuda() for _ in range(3)]
    want = [step(v) for v in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(x)
        for v, y in list(zip(ins, want)) * 2:
            x.copy_(v)
            graph.replay()
            assert torch.equal(out, y)
    torch.cuda.current_stream().wait_stream(side)
