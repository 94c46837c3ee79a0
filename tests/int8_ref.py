"""int8 rows, matrices and products by their definitions, on the CPU."""
import torch

import block_ops_ref as ref


def rows(x):
    """(codes, scale) by the definition, in f32 as it says; IEEE arithmetic gives the same bits everywhere."""
    v = x.float()
    most = v.abs().amax(-1) if v.shape[-1] else v.new_zeros(v.shape[:-1])
    small = most < ref.SMALLEST
    scale = torch.where(small, torch.zeros_like(most), most * torch.tensor(1.0 / 127.0, dtype=torch.float32))
    inverse = torch.where(small, torch.zeros_like(most), 1.0 / scale)
    codes = torch.round(v * inverse[..., None])
    codes = torch.where(torch.isfinite(most)[..., None], codes, torch.zeros_like(codes))
    return codes.to(torch.int8), scale


def matrix(shape, g):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8), torch.rand(shape[:-1], generator=g) * 0.01 + 1e-4


# The sum is exact; what rounds is the sum's conversion to f32, the product of the two scales and that with the sum: half a step each.
REL = 3.01 * 2.0 ** -24


def product(codes, scale, w, w_scale):
    """(codes . w^T * scales, error of its f32 form before the output's rounding), in 64 bits: the sums stay below 2^53."""
    y = codes.double() @ w.double().t() * (scale.double()[:, None] * w_scale.double())
    return y, REL * y.abs()


def gateup(codes, scale, wg, sg, wu, su, idx, cnt, row_of, P):
    out, err = (torch.zeros((P, wg.shape[1]), dtype=torch.float64) for _ in range(2))
    for e, n in enumerate(cnt.tolist()):
        if n == 0:
            continue
        p = idx[e, :n].long()
        r = row_of(p)
        gate, eg = product(codes[r], scale[r], wg[e], sg[e])
        up, eu = product(codes[r], scale[r], wu[e], su[e])
        act = gate * torch.sigmoid(gate)
        out[p] = act * up
        # |d silu| <= 1.1 |d gate|; the fast exponential and division: 2^-21 (1 + |gate| / 3), and gates below -87 give 0
        err[p] = 1.1 * eg * (up.abs() + eu) + act.abs() * eu + (2.0 ** -21 * (1 + gate.abs() / 3) + 2.0 ** -22) * (act * up).abs() + \
            torch.where(gate < -80, 2.0 ** -100, 0.0) * up.abs()
    return out, err


def proj(codes, scale, w, s, idx, cnt, row_of, P):
    out, err = (torch.zeros((P, w.shape[1]), dtype=torch.float64) for _ in range(2))
    for e, n in enumerate(cnt.tolist()):
        if n:
            p = idx[e, :n].long()
            r = row_of(p)
            out[p], err[p] = product(codes[r], scale[r], w[e], s[e])
    return out, err
