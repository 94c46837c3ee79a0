"""The MoE block in 64 bits without any rounding between its stages, and the bound of an f32 evaluation's error."""
import torch

import block_ops_ref as ref

# what two planes of a value leave out: half a step of the second one on what half a step of the first one left
PLANES = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float8_e4m3fn: 2.0 ** -22, torch.int8: 2.0 ** -22}


def value(w, scale):
    if w.dtype == torch.int8:
        return w.double() * scale.double()[..., None]
    return ref.matrix_value(w, scale)


def _sum(x, ex, w, planes):
    """x . w^T of rows with error ex, and its error: ref.product's bound of an f32 sum and what the planes leave out."""
    K = x.shape[-1]
    return x @ w.t(), (K * 2.0 ** -24 + 2.0 ** -20 + planes) * ((x.abs() + ex) @ w.abs().t()) + ex @ w.abs().t()


def experts(b, x, pair_exp, pair_w, top_k, planes=None):
    """(weighted sum over the given experts, its error)"""
    T, H = x.shape
    planes = PLANES[b.gate.dtype] if planes is None else planes
    if b.pre_norm is None:
        h, eh = x.double(), torch.zeros((T, H), dtype=torch.float64)
    else:
        _, _, h, eh = ref.block_norm(x, None, None, None, False, 1.0, 1.0, b.pre_norm, b.rms_eps)
    y, ey = torch.zeros((T, H), dtype=torch.float64), torch.zeros((T, H), dtype=torch.float64)
    pe = pair_exp.view(T, top_k)
    for e in pe.unique().tolist():
        t, s = (pe == e).nonzero(as_tuple=True)
        mats = [value(getattr(b, n)[e], None if getattr(b, n + "_scale") is None else getattr(b, n + "_scale")[e]) for n in ("gate", "up", "down")]
        gate, eg = _sum(h[t], eh[t], mats[0], planes)
        up, eu = _sum(h[t], eh[t], mats[1], planes)
        act = gate * torch.sigmoid(gate)
        a = act * up
        # |d silu| <= 1.1 |d gate|; exponential, sum, division, product: 2^-20
        ea = 1.1 * eg * (up.abs() + eu) + act.abs() * eu + 2.0 ** -20 * a.abs()
        d, ed = _sum(a, ea, mats[2], planes)
        w = pair_w.view(T, top_k)[t, s].double()[:, None]
        y[t] += w * d
        ey[t] += w * ed + (top_k + 1) * 2.0 ** -24 * (w * d).abs()
    return y, ey


def block(b, x, pair_exp, pair_w, top_k, next_w=None, gate=None, planes=None):
    """(out, its bound, next rows, their bound) over the given routing, before they are rounded to their types."""
    y, ey = experts(b, x, pair_exp, pair_w, top_k, planes)
    H = b.hidden
    rel = (H / 64 + 32) * 2.0 ** -24
    n, en = y, ey
    if b.post_norm is not None:
        inv = 1.0 / torch.sqrt(y.square().mean(1, keepdim=True) + b.rms_eps)
        w = b.post_norm.double()
        n = y * inv * w
        en = ey * inv * w.abs() + (rel + ey.square().mean(1, keepdim=True).sqrt() * inv) * n.abs()
    gate = b.out_gate if gate is None else gate
    if gate is not None:
        g = torch.sigmoid(gate.double()) if b.gate_sigmoid else gate.double()
        n, en = n * g, en * g.abs() + 2.0 ** -20 * (n * g).abs()
    s = b.beta * x.double() + b.alpha * n
    es = abs(b.alpha) * en + 4 * 2.0 ** -24 * ((b.beta * x.double()).abs() + (b.alpha * n).abs())
    if next_w is None:
        return s, es, None, None
    inv = 1.0 / torch.sqrt(s.square().mean(1, keepdim=True) + b.rms_eps)
    h = s * inv * next_w.double()
    return s, es, h, es * inv * next_w.double().abs() + (rel + es.square().mean(1, keepdim=True).sqrt() * inv) * h.abs()


def logits(b, x):
    """The router's logits and their error."""
    if b.pre_norm is None:
        h, eh = x.double(), torch.zeros(x.shape, dtype=torch.float64)
    else:
        _, _, h, eh = ref.block_norm(x, None, None, None, False, 1.0, 1.0, b.pre_norm, b.rms_eps)
    v, e = _sum(h, eh, b.router.double(), 0.0)
    return (v, e) if b.router_bias is None else (v + b.router_bias.double(), e + 2.0 ** -24 * (v + b.router_bias.double()).abs())


def check_routing(b, x, pair_exp, pair_w, top_k):
    """k different experts a token, no other one is better by more than the logits' error, weights a softmax over them."""
    T = x.shape[0]
    v, e = logits(b, x)
    pe = pair_exp.view(T, top_k).long()
    assert (pe.sort(1).values.diff(dim=1) > 0).all() and (pe >= 0).all() and (pe < v.shape[1]).all()
    top = v.gather(1, pe)
    least = (top + e.gather(1, pe)).min(1).values
    rest = (v - e).scatter(1, pe, float("-inf")).max(1).values
    assert (rest <= least).all()
    shift = 2 * e.gather(1, pe).max(1, keepdim=True).values + (top_k + 8) * 2.0 ** -23
    want = top.softmax(1)
    assert ((pair_w.view(T, top_k).double() - want).abs() <= want * 2 * shift.clamp(max=0.5) + 2.0 ** -100).all()
