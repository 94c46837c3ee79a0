"""Sizes that pass 32 bits on their way to the library: a count that would be cut to its low word is refused. Tensors without memory and a
library that records what it is given; no device."""
import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.fixture
def ops(monkeypatch):
    from kanjoos_b200 import ops as module

    class Library:
        calls = []

        def __getattr__(self, name):
            def call(*args):
                self.calls.append((name, args))
                return 0
            return call
    Library.calls = []
    monkeypatch.setattr(module, "_cur", lambda: torch.empty(0, device="meta").get_device())
    monkeypatch.setattr(module, "lib", Library)
    monkeypatch.setattr(module, "_raw_stream", lambda: 0)
    module.calls = Library.calls
    yield module
    del module.calls
    module._fp8_matmul_scratch.cache_clear()


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_an_ordinary_call_gets_through(ops):
    ops.fp8_rows(meta(3, 256))
    assert ops.calls and ops.calls[-1][1][3:5] == (3, 256)


@pytest.mark.parametrize("rows", [1 << 31, (1 << 32) + 3])
def test_rows_beyond_32_bits(ops, rows):
    for call in (lambda: ops.fp8_rows(meta(rows, 1)), lambda: ops.block_norm(meta(rows, 1), pre_w=meta(1)),
                 lambda: ops.fp8_matmul(meta(8, 16, dtype=E4M3), meta(1, 1, dtype=torch.float32), meta(rows, 16)),
                 lambda: ops.fp8_matmul(meta(rows, 16, dtype=E4M3), meta(-(-rows // 128), 1, dtype=torch.float32), meta(2, 16)),
                 lambda: ops.fp8_rows(meta(2, rows))):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    assert not ops.calls
