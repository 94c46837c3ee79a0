"""Host-side objects of the MoE expert path: an expert bank resident in HBM, one
MoE-FFN layer (the reference's Model::moe, src/model/model.cpp:399-510, with the
ffn RMSNorm before it and the residual add after it) and the resident
whole-stack decode loop (tools/bench/q4k_stream_ffn.hip:1233-1325 run_resident).
All arithmetic is done by libknj_device.so."""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, replace

import numpy as np
import torch

from . import synth
from ._lib import (DT_BF16, DT_E4M3, DT_F16, DT_F32, GATE_CHANNEL, GATE_FULL, GATE_ROW, MoeBlockArgs, MoeFfnArgs, check, lib)

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16}
_DT_FLOAT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}
_DT_EXPERT = {torch.bfloat16: DT_BF16, torch.float16: DT_F16, torch.float8_e4m3fn: DT_E4M3}


@dataclass
class ExpertBank:
    """Weights of one MoE layer, all on one device.

    gate, up: uint8 [E][F][H/256][144]; down: uint8 [E][H][F/256][144] (Q4_K) or [...][210] (Q6_K);
    router: bf16 [E][H]; router_bias: f32 [E] or None; norm_w: bf16 [H] or None.
    """
    gate: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    router: torch.Tensor
    router_bias: torch.Tensor | None = None
    norm_w: torch.Tensor | None = None
    rms_eps: float = synth.RMS_EPS

    @property
    def n_experts(self) -> int:
        return self.gate.shape[0]

    @property
    def ffn(self) -> int:
        return self.gate.shape[1]

    @property
    def hidden(self) -> int:
        return self.gate.shape[2] * 256

    def nbytes(self) -> int:
        return self.gate.numel() + self.up.numel() + self.down.numel()

    @staticmethod
    def from_numpy(bank: dict, router_bits: np.ndarray, bias: np.ndarray | None = None,
                   norm_bits: np.ndarray | None = None, device="cuda") -> "ExpertBank":
        def bf(bits):
            return torch.from_numpy(bits.view(np.int16).copy()).view(torch.bfloat16).to(device)
        return ExpertBank(
            gate=torch.from_numpy(bank["gate"]).to(device), up=torch.from_numpy(bank["up"]).to(device),
            down=torch.from_numpy(bank["down"]).to(device), router=bf(router_bits),
            router_bias=None if bias is None else torch.from_numpy(bias).to(device),
            norm_w=None if norm_bits is None else bf(norm_bits))

    @staticmethod
    def random(n_experts: int = synth.N_EXPERTS, hidden: int = synth.HIDDEN, ffn: int = synth.FFN, seed: int = 0,
               with_norm: bool = True, device="cuda") -> "ExpertBank":
        """Random-init bank drawn on the device (for large resident stacks): same
        value distributions as synth.q4k_rows, torch's CUDA generator."""
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def q4k(rows, n_in):
            nb = n_in // 256
            blk = torch.randint(0, 256, (n_experts, rows, nb, 144), dtype=torch.uint8, device=device, generator=g)
            dd = (torch.randn((n_experts, rows, nb, 2), device=device, generator=g).abs() * 0.01).to(torch.float16)
            blk[..., 0:4] = dd.view(torch.uint8).reshape(n_experts, rows, nb, 4)
            return blk
        router = (torch.randn((n_experts, hidden), device=device, generator=g) * 0.02).to(torch.bfloat16)
        norm = (1.0 + 0.02 * torch.randn(hidden, device=device, generator=g)).to(torch.bfloat16) if with_norm else None
        return ExpertBank(gate=q4k(ffn, hidden), up=q4k(ffn, hidden), down=q4k(hidden, ffn), router=router, norm_w=norm)


class MoeFfnLayer:
    """One MoE-FFN layer bound to a maximum token count (workspace is allocated
    once here; calls allocate nothing)."""

    def __init__(self, bank: ExpertBank, top_k: int = synth.TOP_K, max_tokens: int = 64, residual: bool = False,
                 use_norm: bool = True, workspace: torch.Tensor | None = None):
        self.bank, self.top_k, self.max_tokens, self.residual = bank, top_k, max_tokens, residual
        self.use_norm = use_norm and bank.norm_w is not None
        need = max(lib().knj_moe_ffn_workspace_bytes(max_tokens, bank.hidden, bank.ffn, bank.n_experts, top_k, mode)
                   for mode in (0, 1))
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=bank.gate.device)
        assert workspace.numel() >= need and workspace.data_ptr() % 256 == 0
        self.workspace = workspace
        self._need = need

    def _args(self, x: torch.Tensor, out: torch.Tensor, taps=None, fused_combine: bool = False) -> MoeFfnArgs:
        b = self.bank
        T, H = x.shape
        assert H == b.hidden and T <= self.max_tokens and x.is_contiguous() and out.is_contiguous()
        a = MoeFfnArgs()
        a.n_tokens, a.hidden, a.ffn, a.n_experts, a.top_k = T, H, b.ffn, b.n_experts, self.top_k
        a.x_dtype, a.x, a.ldx = _DT[x.dtype], x.data_ptr(), H
        a.w_router = b.router.data_ptr()
        a.router_bias = b.router_bias.data_ptr() if b.router_bias is not None else None
        a.w_gate, a.w_up, a.w_down = b.gate.data_ptr(), b.up.data_ptr(), b.down.data_ptr()
        a.down_format = 1 if b.down.shape[-1] == 210 else 0  # Q6_K down matrices of a mixed-format layer
        a.norm_w = b.norm_w.data_ptr() if self.use_norm else None
        a.rms_eps = b.rms_eps
        a.residual = 1 if self.residual else 0
        a.fused_combine = 1 if fused_combine else 0
        a.out, a.out_dtype, a.ldo = out.data_ptr(), _DT[out.dtype], H
        a.workspace, a.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
        if taps is not None:
            a.tap_pair_exp, a.tap_pair_w = taps[0].data_ptr(), taps[1].data_ptr()
        return a

    def _run(self, fn, x, out, out_dtype, return_routing, fused_combine=False):
        if out is None:
            out = torch.empty(x.shape, dtype=out_dtype or torch.float32, device=x.device)
        taps = None
        if return_routing:
            P = x.shape[0] * self.top_k
            taps = (torch.empty(P, dtype=torch.int32, device=x.device), torch.empty(P, dtype=torch.float32, device=x.device))
        args = self._args(x, out, taps, fused_combine)
        check(fn(C.byref(args), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return (out, taps[0], taps[1]) if return_routing else out

    def decode(self, x, out=None, out_dtype=None, return_routing=False):
        """f32-accurate path (batch <= 64 is the intended use)."""
        return self._run(lib().knj_moe_ffn_decode_launch, x, out, out_dtype, return_routing)

    def prefill(self, x, out=None, out_dtype=None, return_routing=False, fused_combine=False):
        """Grouped-GEMM path over per-expert token buckets. fused_combine=False: per-pair rows + the ordered combine
        kernel (reproducible, and the faster form); True: the weighted sum fused into the down GEMM's epilogue
        (f32 reductions, unordered)."""
        return self._run(lib().knj_moe_ffn_prefill_launch, x, out, out_dtype, return_routing, fused_combine)


class MoeStack:
    """The resident whole-stack loop: L layers, each RMSNorm -> MoE -> residual
    add, the residual stream kept in bf16 between layers."""

    def __init__(self, banks: list[ExpertBank], top_k: int = synth.TOP_K, max_tokens: int = 64):
        need = max(lib().knj_moe_ffn_workspace_bytes(max_tokens, b.hidden, b.ffn, b.n_experts, top_k, 0) for b in banks)
        self.workspace = torch.empty(need, dtype=torch.uint8, device=banks[0].gate.device)
        self.layers = [MoeFfnLayer(b, top_k, max_tokens, residual=True, use_norm=True, workspace=self.workspace)
                       for b in banks]
        self.max_tokens = max_tokens
        self._buf = None
        self._graph = None

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """x bf16 [B][H] -> residual stream after the last layer (bf16). Eager launches."""
        B, H = x.shape
        if self._buf is None or self._buf[0].shape != x.shape:
            self._buf = (torch.empty_like(x), torch.empty_like(x))
            self._graph = None
        cur = x
        for i, layer in enumerate(self.layers):
            nxt = self._buf[i & 1]
            layer.decode(cur, out=nxt)
            cur = nxt
        return cur

    def capture(self, x: torch.Tensor):
        """Capture one whole-stack step over the static input buffer `x` into a
        CUDA graph; returns (graph, output tensor). Replays read x in place."""
        self.step(x)  # warm-up: set function attributes, allocate ping-pong buffers
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = self.step(x)
        return g, out


class FusedMoeStack:
    """The resident stack for a decode batch of 1..64 tokens as ONE cooperative launch (knj_moe_stack_*): the per-layer loop,
    its routing and its hand-offs run inside a single kernel with grid barriers between the stages. Buffers are
    static: write the step's rows into `self.x` (or pass them to step) and read `self.out` after the launch."""

    def __init__(self, banks: list[ExpertBank], top_k: int = synth.TOP_K, n_tokens: int = 1, dtype=torch.bfloat16,
                 residual: bool = True, use_norm: bool = True, taps: bool = False,
                 layer_inputs: list[torch.Tensor] | None = None, keep_outputs: bool = False):
        """layer_inputs: one [n_tokens][H] tensor per layer that the layer reads INSTEAD of its predecessor's output
        (independent layers, e.g. to drive every layer with fresh rows); default: the layers form a chain.
        keep_outputs: every layer writes a buffer of its own (self.outs[l]) instead of two alternating ones."""
        dev = banks[0].gate.device
        H = banks[0].hidden
        self.x = torch.zeros((n_tokens, H), dtype=dtype, device=dev)
        self._buf = (torch.zeros_like(self.x), torch.zeros_like(self.x))
        self.outs = [torch.zeros_like(self.x) for _ in banks] if keep_outputs else None
        ws = torch.empty(256, dtype=torch.uint8, device=dev)
        self._layers = [MoeFfnLayer.__new__(MoeFfnLayer) for _ in banks]
        P = n_tokens * top_k
        self.taps = [(torch.empty(P, dtype=torch.int32, device=dev), torch.empty(P, dtype=torch.float32, device=dev))
                     for _ in banks] if taps else None
        arr = (MoeFfnArgs * len(banks))()
        cur = self.x
        for l, (layer, b) in enumerate(zip(self._layers, banks)):
            layer.bank, layer.top_k, layer.max_tokens, layer.residual = b, top_k, n_tokens, residual
            layer.use_norm = use_norm and b.norm_w is not None
            layer.workspace = ws
            nxt = self.outs[l] if keep_outputs else self._buf[l & 1]
            if layer_inputs is not None:
                cur = layer_inputs[l]
            arr[l] = layer._args(cur, nxt, self.taps[l] if taps else None)
            cur = nxt
        self.out = cur
        self._banks, self._inputs = banks, layer_inputs  # keep the weights and the rows alive
        h = C.c_void_p()
        check(lib().knj_moe_stack_create(arr, len(banks), C.byref(h)))
        self._h = h

    def step(self, x: torch.Tensor | None = None) -> torch.Tensor:
        if x is not None:
            self.x.copy_(x)
        check(lib().knj_moe_stack_decode_launch(self._h, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return self.out

    def status(self) -> None:
        """Waits for the stream; raises if a grid barrier of the last launches gave up."""
        check(lib().knj_moe_stack_status(self._h, C.c_void_p(torch.cuda.current_stream().cuda_stream)))

    def set_wait(self, wait_cycles: int = 0, stall_first_barrier: int = 0) -> None:
        """Limit of the kernel's bounded waits (SM cycles; 0 = default) and the test hook that makes the first
        grid barrier unreachable."""
        check(lib().knj_moe_stack_set_wait(self._h, wait_cycles, stall_first_barrier))

    def close(self):
        if self._h:
            lib().knj_moe_stack_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def e4m3_blocks(w: torch.Tensor):
    """A matrix [..., N, K] as e4m3 codes and one f32 scale (largest magnitude / 448) for each block of 128 x 128, the form in
    which ops.fp8_matmul and the expert products take it. Done once, when weights are loaded."""
    n, k = w.shape[-2:]
    nb, kb = -(-n // 128), -(-k // 128)
    v = torch.nn.functional.pad(w.float(), (0, kb * 128 - k, 0, nb * 128 - n)).unflatten(-1, (kb, 128)).unflatten(-3, (nb, 128))
    scale = v.abs().amax(dim=(-3, -1)) / 448.0
    q = torch.where(scale[..., :, None, :, None] > 0, v / scale[..., :, None, :, None], torch.zeros_like(v)).clamp_(-448.0, 448.0)
    return q.flatten(-2).flatten(-3, -2)[..., :n, :k].to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


@dataclass
class FloatExpertBank:
    """Weights of one MoE block whose experts are bf16, f16 or e4m3, all on one device.

    gate, up [E][F][H]; down [E][H][F]; for e4m3 their scales f32 [E][ceil(rows/128)][ceil(cols/128)]; router bf16 [E][H];
    router_bias f32 [E] or None; pre_norm, post_norm: norm weights [H] in front of the block and behind it (one type), or None;
    out_gate [H]: what the block's output is multiplied with (through a sigmoid with gate_sigmoid), or None; router_exact: False where
    the router's bf16 weights were rounded from a file that holds more bits."""
    gate: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    router: torch.Tensor
    gate_scale: torch.Tensor | None = None
    up_scale: torch.Tensor | None = None
    down_scale: torch.Tensor | None = None
    router_bias: torch.Tensor | None = None
    pre_norm: torch.Tensor | None = None
    post_norm: torch.Tensor | None = None
    out_gate: torch.Tensor | None = None
    gate_sigmoid: bool = False
    alpha: float = 1.0
    beta: float = 1.0
    rms_eps: float = synth.RMS_EPS
    router_exact: bool = True

    @property
    def n_experts(self) -> int:
        return self.gate.shape[0]

    @property
    def ffn(self) -> int:
        return self.gate.shape[1]

    @property
    def hidden(self) -> int:
        return self.gate.shape[2]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.gate, self.up, self.down))

    def to_e4m3(self) -> "FloatExpertBank":
        """The same block with its experts as e4m3 codes under block scales."""
        parts = {}
        for name in ("gate", "up", "down"):
            parts[name], parts[name + "_scale"] = e4m3_blocks(getattr(self, name))
        return replace(self, **parts)


class MoeBlock:
    """One MoE block of a residual stream (knj_moe_block_launch): norm, routing, experts, ordered combine, norm behind the block, gate,
    scaled residual add and, on request, the norm in front of the next block. Bound to a maximum token count: the workspace is
    allocated once here."""

    def __init__(self, bank: FloatExpertBank, top_k: int = synth.TOP_K, max_tokens: int = 64, workspace: torch.Tensor | None = None):
        E, F, H = bank.gate.shape
        kind = bank.gate.dtype
        if kind not in _DT_EXPERT or bank.up.dtype != kind or bank.down.dtype != kind:
            raise ValueError("experts are bf16, f16 or float8_e4m3fn, all three matrices of one type")
        want = {"gate": (E, F, H), "up": (E, F, H), "down": (E, H, F), "router": (E, H)}
        if kind == torch.float8_e4m3fn:
            want.update(gate_scale=(E, -(-F // 128), -(-H // 128)), up_scale=(E, -(-F // 128), -(-H // 128)), down_scale=(E, -(-H // 128), -(-F // 128)))
        for name, shape in want.items():
            t = getattr(bank, name)
            if t is None or tuple(t.shape) != shape or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{name}: expected a contiguous CUDA tensor of shape {shape}")
            if name.endswith("_scale") and t.dtype != torch.float32:
                raise ValueError(f"{name}: scales are f32")
        if bank.router.dtype != torch.bfloat16:
            raise ValueError("the router's weights are bf16")
        for name in (*want, "pre_norm", "post_norm", "out_gate", "router_bias"):
            t = getattr(bank, name)
            if t is not None and t.device != bank.gate.device:
                raise ValueError(f"{name} lives on {t.device}, the block on {bank.gate.device}")
        norms = [w for w in (bank.pre_norm, bank.post_norm) if w is not None]
        if any(tuple(w.shape) != (H,) or w.dtype not in _DT_FLOAT or w.dtype != norms[0].dtype or not w.is_contiguous() for w in norms):
            raise ValueError(f"norm weights are contiguous [{H}] of one type")
        if bank.out_gate is not None and (tuple(bank.out_gate.shape) != (H,) or bank.out_gate.dtype not in _DT_FLOAT or not bank.out_gate.is_contiguous()):
            raise ValueError(f"out_gate is contiguous [{H}]")
        if bank.router_bias is not None and (tuple(bank.router_bias.shape) != (E,) or bank.router_bias.dtype != torch.float32 or not bank.router_bias.is_contiguous()):
            raise ValueError(f"router_bias is contiguous f32 [{E}]")
        self.bank, self.top_k, self.max_tokens = bank, top_k, max_tokens
        need = lib().knj_moe_block_workspace_bytes(max_tokens, H, F, E, top_k, _DT_EXPERT[kind])
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=bank.gate.device)
        if workspace.dtype != torch.uint8 or workspace.numel() < need or workspace.data_ptr() % 256 or workspace.device != bank.gate.device or \
                not workspace.is_contiguous():
            raise ValueError(f"workspace of {need} contiguous uint8 values on the block's device, 256-byte aligned, needed")
        self.workspace = workspace
        self._status = torch.empty(1, dtype=torch.int32, device=bank.gate.device)   # of this block alone; a launch clears it
        self._last = None

    def _args(self, x, out, gate, next_norm, h_next, h_scale, taps) -> MoeBlockArgs:
        b = self.bank
        T, H = x.shape
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        a = MoeBlockArgs(n_tokens=T, hidden=H, ffn=b.ffn, n_experts=b.n_experts, top_k=self.top_k, x_dtype=_DT_FLOAT[x.dtype],
                         out_dtype=_DT_FLOAT[out.dtype], w_dtype=_DT_EXPERT[b.gate.dtype], alpha=b.alpha, beta=b.beta, eps=b.rms_eps,
                         gate_sigmoid=1 if b.gate_sigmoid else 0, x=x.data_ptr(), ldx=x.stride(0) if T > 1 else H, out=out.data_ptr(),
                         ldo=out.stride(0) if T > 1 else H, pre_w=ptr(b.pre_norm), post_w=ptr(b.post_norm), next_w=ptr(next_norm),
                         w_router=b.router.data_ptr(), router_bias=ptr(b.router_bias), w_gate=b.gate.data_ptr(), w_up=b.up.data_ptr(),
                         w_down=b.down.data_ptr(), gate_scale=ptr(b.gate_scale), up_scale=ptr(b.up_scale), down_scale=ptr(b.down_scale),
                         h_next=ptr(h_next), ld_h_next=H, h_next_scale=ptr(h_scale), workspace=self.workspace.data_ptr(),
                         workspace_bytes=self.workspace.numel(), status=self._status.data_ptr())
        for w in (b.pre_norm, b.post_norm, next_norm):
            if w is not None:
                a.w_norm_dtype = _DT_FLOAT[w.dtype]
        if gate is not None:
            a.gate, a.gate_dtype = gate.data_ptr(), _DT_FLOAT[gate.dtype]
            a.gate_kind = GATE_CHANNEL if gate.dim() == 1 else GATE_ROW if gate.shape[1] == 1 and H > 1 else GATE_FULL
            a.ldg = 0 if gate.dim() == 1 else gate.stride(0) if T > 1 else gate.shape[1]
        if h_next is not None:
            a.h_next_dtype = DT_E4M3 if h_next.dtype == torch.float8_e4m3fn else _DT_FLOAT[h_next.dtype]
        if taps is not None:
            a.tap_pair_exp, a.tap_pair_w = taps[0].data_ptr(), taps[1].data_ptr()
        return a

    def run(self, x, out=None, gate=None, next_norm=None, next_dtype=None, return_routing=False):
        """x [T][H] f32 / bf16 / f16 -> the stream behind the block, in x's type or into `out` (which may be x). gate: the rows' own
        gate [T][1] or [T][H] in place of the bank's. next_norm [H], in the type of the bank's norms (any float type where those are
        f32): also returns h = norm(out; next_norm) in next_dtype (default: x's type; float8_e4m3fn: (codes, scale)). Returns out, or
        a tuple (out[, h][, pair_exp, pair_w])."""
        b = self.bank
        if x.dim() != 2 or x.shape[1] != b.hidden or x.shape[0] > self.max_tokens or x.dtype not in _DT_FLOAT or x.stride(1) != 1:
            raise ValueError(f"x is {x.dtype} {tuple(x.shape)}, expected rows of {b.hidden} values, at most {self.max_tokens}")
        if x.device != b.gate.device or x.get_device() != torch.cuda.current_device():
            raise ValueError(f"x lives on {x.device}, the block on {b.gate.device}; the current device is {torch.cuda.current_device()}")
        T, H = x.shape
        if out is None:
            out = torch.empty((T, H), dtype=x.dtype, device=x.device)
        elif out.shape != x.shape or out.dtype not in _DT_FLOAT or out.device != x.device or out.stride(1) != 1:
            raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, expected rows like x")
        gate = b.out_gate if gate is None else gate
        if gate is not None and gate.dim() == 2 and (gate.shape[0] != T or gate.shape[1] not in (1, H) or gate.device != x.device or
                                                     gate.dtype not in _DT_FLOAT or (gate.shape[1] > 1 and gate.stride(1) != 1)):
            raise ValueError(f"gate is {gate.dtype} {tuple(gate.shape)}, expected [{T}][1] or [{T}][{H}]")
        if gate is not None and gate.dim() != 2 and gate is not b.out_gate:
            raise ValueError("a call's gate has a row for each token")
        h = scale = None
        if next_norm is not None:
            norms = [w for w in (b.pre_norm, b.post_norm) if w is not None]
            if norms and norms[0].dtype == torch.float32 and next_norm.dtype in _DT_FLOAT:
                next_norm = next_norm.float()   # the same values
            if tuple(next_norm.shape) != (H,) or next_norm.dtype not in _DT_FLOAT or any(w.dtype != next_norm.dtype for w in norms) or \
                    next_norm.device != x.device or not next_norm.is_contiguous():
                raise ValueError(f"next_norm is {next_norm.dtype} {tuple(next_norm.shape)}, expected [{H}] in the block's norm type (or narrower than f32 ones)")
            if next_dtype not in (None, torch.float8_e4m3fn, *_DT_FLOAT):
                raise ValueError(f"next_dtype is {next_dtype}, expected f32, bf16, f16 or float8_e4m3fn")
            h = torch.empty((T, H), dtype=next_dtype or x.dtype, device=x.device)
            if h.dtype == torch.float8_e4m3fn:
                scale = torch.empty((T, -(-H // 128)), dtype=torch.float32, device=x.device)
        taps = None
        if return_routing:
            taps = (torch.empty(T * self.top_k, dtype=torch.int32, device=x.device), torch.empty(T * self.top_k, dtype=torch.float32, device=x.device))
        a = self._args(x, out, gate, next_norm, h, scale, taps)
        check(lib().knj_moe_block_launch(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        self._last = a
        result = (out,) + (() if h is None else ((h, scale) if scale is not None else h,)) + (taps or ())
        return result if len(result) > 1 else out

    def status(self) -> None:
        """Waits for the stream; raises if a bounded wait of the last run gave up."""
        if self._last is None:
            return
        check(lib().knj_moe_block_status(C.byref(self._last), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
