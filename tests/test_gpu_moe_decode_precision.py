"""What the MoE block of a decode step keeps of its f32 values: rows of which every sum has a single term, so that the planes in which
rows and activations reach the tensor core are all that can be missing.

    out[t][h] = d * silu(g * v[t]) * (u * v[t])        d, g, u values that the matrices hold, v of 24 bits

The bound, in units of 2^-24 of the result: each of the three products leaves out what its planes do (three bf16 planes nothing, two fp16
planes half a step of 11 bits of half a step of 11 bits: 4 units), rounds (2; of the up to three parts of a value, which a tensor core may
truncate) and, for codes, rounds once more under its scale (2): 8 units, of gate times |d ln silu / d ln gate| <= 1.3 for |gate| <= 2.
silu's exponential, sum and division 6, the product with up, the weight, the sum over the experts and the output 1 each: 8 * 3.3 + 10 < 38."""
import pytest
import torch

from moe_decode_ref import value
from test_gpu_moe_block import BF16, E4M3, F16, F32, on_device

pytestmark = pytest.mark.gpu
BOUND = 38 * 2.0 ** -24


def one_expert(kind, H, F, g):
    """One expert whose gate, up and down have one value throughout; down's rows are zero but for one place each."""
    from kanjoos_b200.moe import FloatExpertBank
    def full(n, k, v):
        return torch.full((1, n, k), v)
    d = torch.zeros((1, H, F))
    d[0, torch.arange(H), torch.randint(F, (H,), generator=g)] = 1.59375
    b = FloatExpertBank(gate=full(F, H, 0.8359375).to(F16 if kind == F16 else BF16), up=full(F, H, -1.2890625).to(F16 if kind == F16 else BF16),
                        down=d.to(F16 if kind == F16 else BF16), router=torch.zeros((1, H), dtype=BF16), beta=0.0)
    return b.to_e4m3() if kind == E4M3 else b.to_int8() if kind == torch.int8 else b


@pytest.mark.parametrize("kind", [BF16, F16, E4M3, torch.int8])
@pytest.mark.parametrize("H,F", [(256, 64), (512, 1024), (2048, 768), (2304, 2064), (4352, 48), (256, 12304)])
def test_no_bit_of_a_value_is_lost(kind, H, F):
    from kanjoos_b200.moe import MoeBlock
    g = torch.Generator().manual_seed(H + F)
    b = one_expert(kind, H, F, g)
    blk = MoeBlock(on_device(b), top_k=1, max_tokens=16)
    gate, up = (value(getattr(b, n)[0], None if getattr(b, n + "_scale") is None else getattr(b, n + "_scale")[0])[0, 0] for n in ("gate", "up"))
    down = value(b.down[0], None if b.down_scale is None else b.down_scale[0]).sum(1)
    for T in (1, 2, 3, 4, 5, 6, 8, 11, 16):
        for _ in range(4):
            v = (1.0 + torch.rand(T, generator=g)) * torch.where(torch.rand(T, generator=g) < 0.5, -1.0, 1.0)
            assert v.dtype == F32
            x = torch.zeros((T, H))
            x[torch.arange(T), torch.randint(H, (T,), generator=g)] = v
            out = blk.decode(x.cuda()).double().cpu()
            s = gate * v.double()
            want = (s * torch.sigmoid(s) * up * v.double())[:, None] * down
            off = ((out - want).abs() / want.abs()).max().item()
            assert off <= BOUND, (T, off / 2.0 ** -24)
    blk.status()
