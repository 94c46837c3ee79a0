"""The MoE block of a decode step against 64 bits where rows are longer than 2048 bytes (tiles of eight matrix rows) and than 4096 (slices), for
every type of experts; e4m3 blocks differ much in their scales and end inside rows and columns."""
from dataclasses import replace

import pytest
import torch

from test_gpu_moe_block import BF16, E4M3, F16, bank_of
from test_gpu_moe_decode import KINDS, compare, rows, run

pytestmark = pytest.mark.gpu


def uneven(w, g):
    """The matrices times a power of two for each block of 128 x 128."""
    E, n, k = w.shape
    f = torch.exp2(torch.randint(-3, 4, (E, -(-n // 128), -(-k // 128)), generator=g).float())
    return (w.float() * f.repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]).to(w.dtype)


def bank(kind, E, H, F, seed):
    g = torch.Generator().manual_seed(seed)
    b = bank_of(F16 if kind == F16 else BF16, E, H, F, seed, True, True)
    b = replace(b, **{n: uneven(getattr(b, n), g) for n in ("gate", "up", "down")})
    return b.to_e4m3() if kind == E4M3 else b.to_int8() if kind == torch.int8 else b


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("E,H,F,k", [(4, 2304, 2064, 2), (3, 256, 4176, 2), (3, 4352, 144, 2), (5, 1280, 1040, 3), (2, 6400, 48, 1)])
@pytest.mark.parametrize("T", [1, 4, 16])
def test_long_rows_against_64_bits(kind, E, H, F, k, T):
    b = bank(kind, E, H, F, E + T)
    x = rows(T, H, T + 1)
    compare(b, x, k, run(b, x.cuda(), k))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E,H,F,k", [(16, 2, 8192, 64, 1), (3, 2, 32768, 32, 2), (16, 2, 256, 8208, 2), (2, 1, 256, 40960, 1), (7, 2, 16384, 48, 1),
                                       (3, 1, 22784, 32, 1), (3, 1, 256, 22656, 1)])
def test_long_rows_in_passes(kind, T, E, H, F, k):
    b = bank(kind, E, H, F, 7)
    x = rows(T, H, 1)
    compare(b, x, k, run(b, x.cuda(), k))
