"""The operators around an MoE block in 64 bits on the CPU, with the error bounds that their f32 sums and roundings give."""
import torch

GROUP, SMALLEST = 128, 2.0 ** -100
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # half a step below the normal range


def held(v, dtype):
    """What rounding |v| to dtype may cost: half a step, relative in the normal range, absolute below it."""
    return U[dtype] * v.abs() + TINY[dtype]


def fp8_rows(x):
    """(codes, scale) by the definition, in f32 as it says; IEEE arithmetic gives the same bits everywhere."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % GROUP)).unflatten(-1, (-1, GROUP))
    most = v.abs().amax(-1)
    small = most < SMALLEST
    scale = torch.where(small, torch.zeros_like(most), most * torch.tensor(1.0 / 448.0, dtype=torch.float32))
    inverse = torch.where(small, torch.zeros_like(most), 1.0 / scale)
    codes = (v * inverse[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.flatten(-2)[..., :k].contiguous(), scale


def rows_value(codes, scale):
    return codes.double() * scale.double().repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]


def matrix(shape, g, dtype):
    """A matrix (or one per expert) and its scales, None for 16-bit types."""
    w = torch.randn(shape, generator=g) * 0.05
    if dtype != torch.float8_e4m3fn:
        return w.to(dtype), None
    n, k = shape[-2:]
    scale = torch.rand(shape[:-2] + (-(-n // GROUP), -(-k // GROUP)), generator=g) * 0.01 + 1e-3
    return (w * 400).to(dtype), scale


def matrix_value(w, scale):
    v = w.double()
    if scale is not None:
        n, k = w.shape[-2:]
        v = v * scale.double().repeat_interleave(GROUP, -1)[..., :k].repeat_interleave(GROUP, -2)[..., :n, :]
    return v


def product(x, w):
    """(x . w^T, bound of an f32 sum's error): a chain of K additions, each off by at most 2^-24 of the sum of magnitudes, or a
    tensor core's, which truncates at 2^-23 at most once per 8 products; the products are exact."""
    return x @ w.t(), (x.shape[-1] * 2.0 ** -24 + 2.0 ** -20) * (x.abs() @ w.abs().t())


def tables(counts, g, device="cpu", stride=None):
    """Tables of pairs 0 .. sum(counts)-1 shuffled over experts with these counts; one pair per row."""
    P = sum(counts)
    perm = torch.randperm(P, generator=g)
    idx = torch.full((len(counts), stride or max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    for e, c in enumerate(counts):
        idx[e, :c] = perm[at:at + c].sort().values.int()
        at += c
    return idx, torch.tensor(counts, dtype=torch.int32)


def gateup(x, wg, wu, idx, cnt, row_of, P):
    """(values, bound before the output's rounding, written)"""
    out, err, wrote = (torch.zeros((P, wg.shape[1]), dtype=torch.float64), torch.zeros((P, wg.shape[1]), dtype=torch.float64),
                       torch.zeros(P, dtype=torch.bool))
    for e, n in enumerate(cnt.tolist()):
        p = idx[e, :n].long()
        if n == 0:
            continue
        r = x[row_of(p)]
        gate, eg = product(r, wg[e])
        up, eu = product(r, wu[e])
        act = gate * torch.sigmoid(gate)
        out[p] = act * up
        # |d silu| <= 1.1 |d gate|; a fast exponential and division: 2^-20 relative together
        err[p] = 1.1 * eg * (up.abs() + eu) + act.abs() * eu + 2.0 ** -20 * (act * up).abs()
        wrote[p] = True
    return out, err, wrote


def proj(x, w, idx, cnt, row_of, P):
    out, err, wrote = (torch.zeros((P, w.shape[1]), dtype=torch.float64), torch.zeros((P, w.shape[1]), dtype=torch.float64),
                       torch.zeros(P, dtype=torch.bool))
    for e, n in enumerate(cnt.tolist()):
        p = idx[e, :n].long()
        if n:
            out[p], err[p] = product(x[row_of(p)], w[e])
            wrote[p] = True
    return out, err, wrote


def block_norm(x, y, post_w, gate, sigmoid, alpha, beta, pre_w, eps):
    """(s, bound of s, h, bound of h), before any rounding to an output type."""
    x = x.double()
    H = x.shape[1]
    s = beta * x
    size = s.abs()
    if y is not None:
        n = y.double()
        if post_w is not None:
            n = n / torch.sqrt(n.square().mean(1, keepdim=True) + eps) * post_w.double()
        if gate is not None:
            n = n * (torch.sigmoid(gate.double()) if sigmoid else gate.double())
        s = s + alpha * n
        size = size + (alpha * n).abs()
    # sums of squares: at most H / 32 + 32 additions deep, halved by the root; a handful of products and a division behind it
    rel = (H / 64 + 32) * 2.0 ** -24
    es = rel * size
    if pre_w is None:
        return s, es, None, None
    inv = 1.0 / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    h = s * inv * pre_w.double()
    root = es.square().mean(1, keepdim=True).sqrt() * inv     # relative change of the norm by s's own errors
    return s, es, h, (es * inv) * pre_w.double().abs() + (rel + root) * h.abs()


def check(got, want, bound, what=""):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off - bound).max()):.3e} above its bound at {bad.nonzero()[0].tolist()}"
