"""The norm between two blocks on values near both ends of the f32 range, in every kernel that forms it: 16-byte rows straight into
registers and through the ring, rows of any width, rows above 16384 values."""
import pytest
import torch

import block_ops_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16

# (T, H): one row per CTA, the ring, any width with two and with four groups a warp, above 16384 values
ROWS = [(3, 512), (3000, 512), (400, 2048), (2, 16384), (5, 1001), (3, 5003), (2, 16392), (3, 16385)]


def gen(*key):
    g = torch.Generator()
    g.manual_seed(sum((i + 1) * 104729 * ord(c) for i, c in enumerate(str(key))))
    return g


def check_both(got, x, y, **kw):
    s, es, h, eh = ref.block_norm(x, y, kw.get("post_w"), kw.get("gate"), kw.get("gate_sigmoid", False), kw.get("alpha", 1.0), kw.get("beta", 1.0),
                                  kw.get("pre_w"), 1e-6)
    ref.check(got[0], s, es + ref.held(s, F32), "stream")
    if h is not None:
        ref.check(got[1], h, eh + ref.held(h, F32), "normalised rows")


def run(x, y, **kw):
    from kanjoos_b200 import ops
    dev = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()}
    return ops.block_norm(x.cuda(), None if y is None else y.cuda(), norm_dtype=F32, **dev)


@pytest.mark.parametrize("T,H", ROWS)
def test_block_output_whose_squares_leave_the_range(T, H):
    """y around 1e30: its squares are infinite in f32, its norm is not. x is of order one, so that the stream shows n."""
    g = gen("post", T, H)
    x, y, w = torch.randn((T, H), generator=g), torch.randn((T, H), generator=g) * 1e30, 1 + 0.3 * torch.randn(H, generator=g)
    y[-1] *= 1e-30   # an ordinary row beside them
    check_both(run(x, y, post_w=w, alpha=2.0, pre_w=w), x, y, post_w=w, alpha=2.0, pre_w=w)


@pytest.mark.parametrize("T,H", ROWS)
def test_stream_whose_squares_leave_the_range(T, H):
    g = gen("pre", T, H)
    x, w = torch.randn((T, H), generator=g) * 1e30, 1 + 0.3 * torch.randn(H, generator=g)
    check_both(run(x, None, pre_w=w, stream_dtype=F32), x, None, pre_w=w)


@pytest.mark.parametrize("T,H", ROWS)
@pytest.mark.parametrize("gate", [None, "channel", "row", "full"])
def test_weights_and_gates_act_on_the_normalised_row(T, H, gate):
    """n = y * inverse norm is of order one whatever y is: neither y * w * g, which is infinite here, nor a tiny inverse times w, g or
    alpha, which has few bits left, may stand in its way."""
    g = gen("order", T, H, gate)
    x, y = torch.zeros((T, H)), torch.randn((T, H), generator=g) * 1e34
    w = (1 + 0.3 * torch.randn(H, generator=g).clamp(-2, 2)) * 1e6
    gt = None if gate is None else torch.randn({"channel": (H,), "row": (T, 1), "full": (T, H)}[gate], generator=g) * 1e5
    check_both(run(x, y, post_w=w, gate=gt, alpha=1e-3), x, y, post_w=w, gate=gt, alpha=1e-3)
    small = None if gt is None else gt * 1e-15
    check_both(run(x, y, post_w=w * 1e-6, gate=small, alpha=1e-3), x, y, post_w=w * 1e-6, gate=small, alpha=1e-3)


@pytest.mark.parametrize("T,H", ROWS)
def test_small_weights_in_front_of_the_next_block(T, H):
    """h = s * inverse norm * pre_w with s around 1e36 and weights around 1e-4: their product with the inverse norm alone is denormal."""
    g = gen("small", T, H)
    x, w = torch.randn((T, H), generator=g) * 1e36, (1 + 0.3 * torch.randn(H, generator=g)) * 1e-4
    check_both(run(x, None, pre_w=w, stream_dtype=F32), x, None, pre_w=w)
