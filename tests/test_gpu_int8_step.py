"""A decode step of layers in whole numbers, as a serving program runs it: the block of a layer, its norm for the next, a dense int8 product
of those rows added to the stream, through three layers, the blocks over one workspace, and the whole captured."""
import pytest
import torch

import block_ops_ref as ref
import int8_ref as i8
import moe_decode_ref as dr
from test_gpu_block_ops import BF16, F32, gen
from test_gpu_moe_block import on_device
from test_gpu_moe_decode import bank, compare, rows

pytestmark = pytest.mark.gpu
I8 = torch.int8
E, H, F, K, LAYERS = 24, 512, 208, 4, 3


def layers(kind):
    from kanjoos_b200.moe import MoeBlock
    out, workspace = [], None
    for i in range(LAYERS):
        host = bank(kind, E, H, F, 70 + i)
        blk = MoeBlock(on_device(host), top_k=K, max_tokens=16, workspace=workspace)
        workspace = blk.workspace
        w, s = i8.matrix((H, H), gen("step", i))
        out.append((host, blk, w.cuda(), s.cuda(), torch.linspace(0.5, 1.5, H, device="cuda").to(BF16)))
    return out


def step(net, x):
    from kanjoos_b200 import ops
    for _, blk, w, s, norm in net:
        out, h = blk.decode(x, next_norm=norm)
        x = out + ops.int8_matmul(w, s, h, out_dtype=x.dtype)
    return x


@pytest.mark.parametrize("kind", [I8, BF16])
@pytest.mark.parametrize("T", [1, 4, 5, 16])
def test_first_layer_against_64_bits(kind, T):
    from kanjoos_b200 import ops
    host, blk, w, s, norm = layers(kind)[0]
    x = rows(T, H, 80 + T)
    got = blk.decode(x.cuda(), next_norm=norm, return_routing=True)
    _, _, hs, eh = compare(host, x, K, got, norm.cpu())
    y = ops.int8_matmul(w, s, got[1])
    # a code is off its value by half a step of the row's scale, and by what the row itself is off
    matrix = dr.value(w.cpu(), s.cpu())
    off = 0.5 * got[1].abs().amax(1, keepdim=True).double().cpu() / 127.0 * (1.0 + 2.0 ** -20) + eh + ref.held(hs.abs() + eh, F32)
    want = hs @ matrix.t()
    bound = off @ matrix.abs().t()
    ref.check(y, want, bound + ref.held(want.abs() + bound, F32) + 2.0 ** -22 * (want.abs() + bound), "product of the next rows")


@pytest.mark.parametrize("kind", [I8, BF16])
@pytest.mark.parametrize("T", [1, 5, 16])
def test_captured_step(kind, T):
    """The captured step gives the bits of the launched one, whatever ran over its workspace in between; tokens stand for themselves."""
    net = layers(kind)
    ins = [rows(T, H, 90 + i, BF16).cuda() for i in range(3)]
    want = [step(net, v) for v in ins]
    assert all(torch.isfinite(v).all() for v in want)
    for t in {0, T - 1}:
        assert torch.equal(step(net, ins[0][t:t + 1]), want[0][t:t + 1])
    x = ins[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(net, x)
        for v, w in list(zip(ins, want)) * 2:
            x.copy_(v)
            graph.replay()
            assert torch.equal(out, w)
            net[0][1].run(v)
    torch.cuda.current_stream().wait_stream(side)
    for layer in net:
        layer[1].status()
