"""Thin typed wrappers over the C-ABI for torch CUDA tensors (torch supplies
device memory and streams only; every computation is a kernel of
libknj_device.so). Names follow the C entry points."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import (DT_BF16, DT_E4M3, DT_F16, DT_F32, GATE_CHANNEL, GATE_FULL, GATE_NONE, GATE_ROW, BlockNormArgs, ExpertGemmArgs, check,
                   lib, packed)

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}
_E4M3 = torch.float8_e4m3fn
_DT_ALL = {**_DT, _E4M3: DT_E4M3}


def _p(t: torch.Tensor | None):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _raw_stream() -> int:
    """The current device's current stream, without a torch.cuda.Stream object around it."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


@functools.lru_cache(maxsize=None)
def _noalloc_scratch() -> int:
    return int(lib().knj_q4k_matmul_noalloc_max_scratch())


def _need(t: torch.Tensor, dtype=None):
    if not t.is_cuda:
        raise ValueError("tensor must live on a CUDA device")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"expected {dtype}, got {t.dtype}")
    return t


def device_caps(idx: int = 0) -> _lib.DeviceCapsC:
    caps = _lib.DeviceCapsC()
    check(lib().knj_dev_caps(idx, C.byref(caps)))
    return caps


def control(seed: int, n_threads: int = 64, n_blocks: int = 1) -> torch.Tensor:
    out = torch.full((2,), 0xABABABAB - (1 << 32), dtype=torch.int32, device="cuda")
    check(lib().knj_control_launch(_p(out), seed, n_threads, n_blocks, _stream()))
    return out


def probe_caps(inp: torch.Tensor | None = None) -> torch.Tensor:
    cap = torch.zeros(8, dtype=torch.int32, device="cuda")
    check(lib().knj_probe_caps_launch(_p(cap), _p(inp), _stream()))
    return cap


def build_asum(act: torch.Tensor, M: int, K: int, n_threads: int = 64, n_blocks: int | None = None) -> torch.Tensor:
    _need(act, torch.int32)
    asum = torch.full((M, K // 128), 0x5A5A5A5A, dtype=torch.int32, device="cuda")
    if n_blocks is None:
        n_blocks = max(1, (M * (K // 128) + n_threads - 1) // n_threads)
    check(lib().knj_build_asum_launch(_p(act), _p(asum), M, K, n_threads, n_blocks, _stream()))
    return asum


def gemm_w4_i8(Bq: torch.Tensor, act: torch.Tensor, asum: torch.Tensor, M: int, N: int, K: int, n_threads: int = 64,
               n_blocks: int | None = None) -> torch.Tensor:
    _need(Bq, torch.uint8), _need(act, torch.int32), _need(asum, torch.int32)
    Cm = torch.full((M, N), -12345.0, dtype=torch.float32, device="cuda")
    if n_blocks is None:
        n_blocks = max(1, (M * N + n_threads - 1) // n_threads)
    check(lib().knj_gemm_w4_i8_launch(_p(Bq), _p(act), _p(asum), _p(Cm), M, N, K, n_threads, n_blocks, _stream()))
    return Cm


def dot_helpers(a: torch.Tensor, b: torch.Tensor, acc: torch.Tensor):
    """int32 [n] x 3 -> (dot4_i8, dot8_i4, dot2_i16) computed by include/knj_dot.h on the device."""
    _need(a, torch.int32), _need(b, torch.int32), _need(acc, torch.int32)
    outs = [torch.full_like(a, 0x5A5A5A5A) for _ in range(3)]
    check(lib().knj_dot_helpers_launch(_p(a), _p(b), _p(acc), _p(outs[0]), _p(outs[1]), _p(outs[2]), a.numel(), _stream()))
    return outs


def q4k_dequant(blocks: torch.Tensor) -> torch.Tensor:
    """uint8 [..., 144] -> f32 [..., 256]."""
    _need(blocks, torch.uint8)
    assert blocks.shape[-1] == 144
    nb = blocks.numel() // 144
    out = torch.full(blocks.shape[:-1] + (256,), -12345.0, dtype=torch.float32, device="cuda")
    check(lib().knj_q4k_dequant_launch(_p(blocks), _p(out), nb, _stream()))
    return out


def q6k_dequant(blocks: torch.Tensor) -> torch.Tensor:
    _need(blocks, torch.uint8)
    assert blocks.shape[-1] == 210
    nb = blocks.numel() // 210
    out = torch.full(blocks.shape[:-1] + (256,), -12345.0, dtype=torch.float32, device="cuda")
    check(lib().knj_q6k_dequant_launch(_p(blocks), _p(out), nb, _stream()))
    return out


def rmsnorm(x: torch.Tensor, w_bf16: torch.Tensor, eps: float) -> torch.Tensor:
    _need(x), _need(w_bf16, torch.bfloat16)
    T, H = x.shape
    out = torch.empty((T, H), dtype=torch.float32, device="cuda")
    check(lib().knj_rmsnorm_launch(_p(x), _DT[x.dtype], H, _p(w_bf16), eps, T, H, _p(out), _stream()))
    return out


def router_topk(x: torch.Tensor, Wr: torch.Tensor, k: int, bias: torch.Tensor | None = None):
    """x [T][H] (f32/bf16), Wr bf16 [E][H] -> (logits [T][E], pair_exp [T*k], pair_w [T*k])."""
    _need(x), _need(Wr, torch.bfloat16)
    T, H = x.shape
    E = Wr.shape[0]
    logits = torch.empty((T, E), dtype=torch.float32, device="cuda")
    pair_exp = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    pair_w = torch.full((T * k,), -12345.0, dtype=torch.float32, device="cuda")
    check(lib().knj_router_topk_launch(_p(x), _DT[x.dtype], H, _p(Wr), _p(bias), T, H, E, k, _p(logits), _p(pair_exp),
                                       _p(pair_w), _stream()))
    return logits, pair_exp, pair_w


def moe_permute(pair_exp: torch.Tensor, E: int, idx_stride: int):
    _need(pair_exp, torch.int32)
    P = pair_exp.numel()
    pair_idx = torch.empty((E, idx_stride), dtype=torch.int32, device="cuda")
    pair_cnt = torch.empty((E,), dtype=torch.int32, device="cuda")
    exp_list = torch.empty((E,), dtype=torch.int32, device="cuda")
    n_active = torch.empty((4,), dtype=torch.int32, device="cuda")
    if P >= 8192 and E <= 256:
        nbytes = int(lib().knj_moe_permute_scratch_bytes(P, E))
        scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        check(lib().knj_moe_permute_ws_launch(_p(pair_exp), P, E, idx_stride, _p(pair_idx), _p(pair_cnt), _p(exp_list),
                                              _p(n_active), _p(scratch), nbytes, _stream()))
    else:
        check(lib().knj_moe_permute_launch(_p(pair_exp), P, E, idx_stride, _p(pair_idx), _p(pair_cnt), _p(exp_list),
                                           _p(n_active), _stream()))
    return pair_idx, pair_cnt, exp_list, n_active


def q4k_gateup(x, Wg, Wu, pair_idx, pair_cnt, exp_list, n_active, P: int, top_k: int, want=("G", "U", "A"),
               pair_tok=None):
    """x [T][K] activation rows (f32/bf16/f16) -> dict of f32 [P][N] outputs (G, U, A = silu(G)*U)."""
    _need(x)
    E, N, nsb, _ = Wg.shape
    K = nsb * 256
    outs = {n: (torch.full((P, N), -12345.0, dtype=torch.float32, device="cuda") if n in want else None)
            for n in ("G", "U", "A")}
    check(lib().knj_q4k_gateup_launch(_p(x), _DT[x.dtype], x.shape[1], _p(Wg), _p(Wu), _p(pair_idx), _p(pair_cnt),
                                      _p(pair_tok), _p(exp_list), _p(n_active), _p(outs["G"]), _p(outs["U"]),
                                      _p(outs["A"]), N, K, nsb * 144, pair_idx.shape[1], E, top_k, None, _stream()))
    return outs


def q4k_proj(a, W, pair_idx, pair_cnt, exp_list, n_active, P: int, pair_row=None):
    """a [rows][K] activation rows (one per pair unless pair_row maps them) -> Y f32 [P][N]."""
    _need(a)
    E, N, nsb, _ = W.shape
    K = nsb * 256
    Y = torch.full((P, N), -12345.0, dtype=torch.float32, device="cuda")
    check(lib().knj_q4k_proj_launch(_p(a), _DT[a.dtype], a.shape[1], _p(W), _p(pair_idx), _p(pair_cnt), _p(pair_row),
                                    _p(exp_list), _p(n_active), _p(Y), N, K, nsb * 144, pair_idx.shape[1], E, None,
                                    _stream()))
    return Y


def q6k_proj(A: torch.Tensor, W6: torch.Tensor, pair_idx, pair_cnt, exp_list, n_active, P: int) -> torch.Tensor:
    """A f32 [P][K], W6 uint8 [E][N][K/256][210] -> Y f32 [P][N] (rows of pairs of inactive experts stay poisoned)."""
    _need(A, torch.float32), _need(W6, torch.uint8)
    E, N, nblk, _ = W6.shape
    Y = torch.full((P, N), -12345.0, dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(lib().knj_q6k_proj_launch(_p(A), _p(W6), _p(pair_idx), _p(pair_cnt), _p(exp_list), _p(n_active), _p(Y), N,
                                    nblk * 256, pair_idx.shape[1], E, _p(status), _stream()))
    if int(status.item()):
        raise RuntimeError("knj_q6k_proj_launch: a bounded wait for a weight block gave up")
    return Y


def fuse_gateup_silu(G: torch.Tensor, U: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    _need(G, torch.float32), _need(U, torch.float32)
    A = torch.empty(G.shape, dtype=dtype, device="cuda")
    check(lib().knj_fuse_gateup_silu_launch(_p(G), _p(U), _p(A), _DT[dtype], G.numel(), _stream()))
    return A


def moe_combine(Y, pair_exp, pair_w, T: int, k: int, resid=None, out_dtype=torch.float32, pair_row=None):
    H = Y.shape[1]
    out = torch.empty((T, H), dtype=out_dtype, device="cuda")
    check(lib().knj_moe_combine_launch(_p(Y), _p(pair_row), _p(pair_exp), _p(pair_w), _p(resid),
                                       _DT[resid.dtype] if resid is not None else 0, H, _p(out), _DT[out_dtype], H, T, H,
                                       k, _stream()))
    return out


def q4k_matmul(W: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """W uint8 [n_out][n_in/256][144], x [m][n_in] -> f32 [m][n_out] (Model::matmul)."""
    _need(W, torch.uint8), _need(x)
    n_out, nsb, _ = W.shape
    m, n_in = x.shape
    assert nsb * 256 == n_in
    y = torch.empty((m, n_out), dtype=torch.float32, device="cuda")  # every element is written (NaN where a bounded wait gave up)
    L = lib()
    nbytes = L.knj_q4k_matmul_workspace_bytes(m, n_in)
    # The kernel needs no scratch: up to the limit of the entry point that takes none, nothing is allocated for it. A one-row
    # product of 768 x 2048 takes the device 5 us and this function more: 15.8 us a call with a workspace and stream objects, 9.3 so.
    if 0 < nbytes <= _noalloc_scratch():
        check(L.knj_q4k_matmul_noalloc_launch(W.data_ptr(), n_in, n_out, x.data_ptr(), _DT[x.dtype], n_in, m, y.data_ptr(), n_out, _raw_stream()))
        return y
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    check(L.knj_q4k_matmul_launch(_p(W), n_in, n_out, _p(x), _DT[x.dtype], n_in, m, _p(y), n_out, _p(ws), nbytes, _stream()))
    return y


def to_f16(x: torch.Tensor) -> torch.Tensor:
    _need(x)
    rows, K = x.shape
    out = torch.empty((rows, K), dtype=torch.float16, device="cuda")
    check(lib().knj_to_f16_launch(_p(x), _DT[x.dtype], K, rows, K, _p(out), _stream()))
    return out


def q4k_gateup_tc(xh, Wg, Wu, pair_idx, pair_cnt, P: int, top_k: int, pair_tok=None, poison: bool = True):
    """Tensor-core grouped gate+up: returns (A fp16 [P][N] scaled by 2^-6, status int32[1]).
    poison=True pre-fills A with NaN so that tests can see unwritten rows."""
    _need(xh, torch.float16)
    E, N, nsb, _ = Wg.shape
    A = (torch.full((P, N), float("nan"), dtype=torch.float16, device="cuda") if poison
         else torch.empty((P, N), dtype=torch.float16, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(lib().knj_q4k_gateup_tc_launch(_p(xh), _p(Wg), _p(Wu), _p(pair_idx), _p(pair_cnt), _p(pair_tok), _p(A), N,
                                         nsb * 256, nsb * 144, pair_idx.shape[1], E, top_k, P, _p(status), _stream()))
    return A, status


def q6k_down_tc(ah, W6, pair_idx, pair_cnt, P: int, pair_row=None):
    """Grouped down GEMM over Q6_K weights [E][N][K/256][210] (K <= 1024): fp16 activations as the gate+up GEMM
    writes them -> Y f32 [P][N]."""
    _need(ah, torch.float16), _need(W6, torch.uint8)
    E, N, nsb, _ = W6.shape
    Y = torch.full((P, N), -12345.0, dtype=torch.float32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(lib().knj_q6k_down_tc_launch(_p(ah), _p(W6), _p(pair_idx), _p(pair_cnt), _p(pair_row), _p(Y), N, nsb * 256,
                                       pair_idx.shape[1], E, P, _p(status), _stream()))
    return Y, status


def q4k_down_tc(ah, Wd, pair_idx, pair_cnt, P: int, pair_row=None, poison: bool = True):
    _need(ah, torch.float16)
    E, N, nsb, _ = Wd.shape
    Y = (torch.full((P, N), -12345.0, dtype=torch.float32, device="cuda") if poison
         else torch.empty((P, N), dtype=torch.float32, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(lib().knj_q4k_down_tc_launch(_p(ah), _p(Wd), _p(pair_idx), _p(pair_cnt), _p(pair_row), _p(Y), N, nsb * 256,
                                       nsb * 144, pair_idx.shape[1], E, P, _p(status), _stream()))
    return Y, status


# ---- experts in bf16, fp16 and e4m3, and what stands between two blocks -------------------------------------------
# These calls are made once or a few times per layer and decode step, so their host work counts: attributes are read once, outputs
# come from new_empty / empty_like (1.4 us against torch.empty's 2.4).

_cur = torch._C._cuda_getDevice
_OPERAND = {torch.bfloat16: DT_BF16, torch.float16: DT_F16, _E4M3: DT_E4M3}
_norm_args, _expert_args = packed(BlockNormArgs), packed(ExpertGemmArgs)
_ONLY_F32, _ONLY_I32, _ONLY_E4M3 = {torch.float32: DT_F32}, {torch.int32: 0}, {_E4M3: DT_E4M3}


def _refuse(t: torch.Tensor, what: str, cur: int, shape, types):
    if t.get_device() != cur:
        raise ValueError(f"{what} lives on {t.device}, not on the current CUDA device")
    raise ValueError(f"{what} is {t.dtype} {tuple(t.shape)} with strides {t.stride()}, expected {' / '.join(str(d) for d in types)} "
                     f"{'rows' if shape is None else tuple(shape)}, dense inside a row and without overlap")


def _refuse_count(what: str, shape):
    """The library counts in 32 bits, and ctypes would hand it a larger number's low word."""
    raise ValueError(f"{what} is {tuple(shape)}: rows and columns have to stay below 2^31")


def _rows(t: torch.Tensor, what: str, cur: int, shape=None, types=_DT):
    """A matrix of rows, dense inside a row, any row stride, on the current device: (address, type code, row stride)."""
    code, s = types.get(t.dtype), t.shape
    if code is None or len(s) != 2 or t.get_device() != cur or (shape is not None and s != shape):
        _refuse(t, what, cur, shape, types)
    n, k = s
    if (n | k) >> 31:
        _refuse_count(what, s)
    ld, one = t.stride()
    if n <= 1:
        ld = k
    if (one != 1 and k > 1) or ld < k:
        _refuse(t, what, cur, shape, types)
    return t.data_ptr(), code, ld


def _dense(t: torch.Tensor, what: str, cur: int, shape, types) -> int:
    """A contiguous tensor of this shape on the current device: its address."""
    if t.dtype not in types or t.shape != shape or t.get_device() != cur or not t.is_contiguous():
        _refuse(t, what, cur, shape, types)
    return t.data_ptr()


def fp8_rows(x: torch.Tensor):
    """x [rows][K] (f32 / bf16 / f16) -> (codes float8_e4m3fn [rows][K], scale f32 [rows][ceil(K/128)])."""
    ptr, code, ld = _rows(x, "x", _cur())
    n, k = x.shape
    q = x.new_empty(n, k, dtype=_E4M3)
    scale = x.new_empty(n, (k + 127) // 128, dtype=torch.float32)
    check(lib().knj_fp8_rows_launch(ptr, code, ld, n, k, q.data_ptr(), scale.data_ptr(), _raw_stream()))
    return q, scale


@functools.lru_cache(maxsize=1024)
def _fp8_matmul_scratch(m: int, k: int) -> int:
    return int(lib().knj_fp8_matmul_workspace_bytes(m, k))


def fp8_matmul(W: torch.Tensor, W_scale: torch.Tensor, x: torch.Tensor, out_dtype=torch.float32, status=None) -> torch.Tensor:
    """W float8_e4m3fn [n_out][n_in] with W_scale f32 [ceil(n_out/128)][ceil(n_in/128)], x [m][n_in] (f32 / bf16 / f16, turned
    into e4m3 rows as fp8_rows does) -> [m][n_out] in out_dtype. status as for expert_gateup."""
    cur = _cur()
    ptr, code, ld = _rows(x, "x", cur)
    m, k = x.shape
    n, out_code = W.shape[0], _DT.get(out_dtype)
    if out_code is None:
        raise ValueError(f"out_dtype is {out_dtype}")
    if n >> 31:
        _refuse_count("W", W.shape)
    w = _dense(W, "W", cur, (n, k), _ONLY_E4M3)
    ws = _dense(W_scale, "W_scale", cur, ((n + 127) // 128, (k + 127) // 128), _ONLY_F32)
    y = x.new_empty(m, n, dtype=out_dtype)
    nbytes = _fp8_matmul_scratch(m, k)
    work = x.new_empty(nbytes, dtype=torch.uint8)
    check(lib().knj_fp8_matmul_launch(w, ws, k, n, ptr, code, ld, m, y.data_ptr(), out_code, n, work.data_ptr(), nbytes,
                                      None if status is None else _dense(status, "status", cur, (1,), _ONLY_I32), _raw_stream()))
    return y


def _expert(launch, x, x_scale, w, w1, s0, s1, pair_idx, pair_cnt, P, row_map, row_div, out, out_dtype, out_scale, status):
    cur = _cur()
    if w.dim() != 3 or w.dtype not in _OPERAND:
        raise ValueError(f"expert matrices are bf16, f16 or float8_e4m3fn [E][N][K], got {w.dtype} {tuple(w.shape)}")
    shape = w.shape
    E, N, K = shape
    types = (w.dtype,)
    w_ptr = _dense(w, "an expert matrix", cur, shape, types)
    w1_ptr = 0 if w1 is None else _dense(w1, "an expert matrix", cur, shape, types)
    xs = s0_ptr = s1_ptr = 0
    if w.dtype == _E4M3:
        if s0 is None or (w1 is not None and s1 is None):
            raise ValueError("e4m3 expert matrices need their scales")
        sshape = (E, (N + 127) // 128, (K + 127) // 128)
        s0_ptr = _dense(s0, "a matrix's scales", cur, sshape, _ONLY_F32)
        if w1 is not None:
            s1_ptr = _dense(s1, "a matrix's scales", cur, sshape, _ONLY_F32)
        if x.dtype != _E4M3:
            if x_scale is not None:
                raise ValueError("x_scale belongs to e4m3 rows")
            x, x_scale = fp8_rows(x)
        elif x_scale is None:
            raise ValueError("e4m3 rows need x_scale")
        xs = _dense(x_scale, "x_scale", cur, (x.shape[0], sshape[2]), _ONLY_F32)
    elif s0 is not None or s1 is not None or x_scale is not None:
        raise ValueError("scales belong to e4m3 matrices and rows")
    x_ptr, x_code, ld = _rows(x, "x", cur, (x.shape[0], K), {w.dtype: _OPERAND[w.dtype]})
    idx_shape = pair_idx.shape
    if len(idx_shape) != 2:
        raise ValueError(f"pair_idx has shape {tuple(idx_shape)}")
    idx = _dense(pair_idx, "pair_idx", cur, (E, idx_shape[1]), _ONLY_I32)
    cnt = _dense(pair_cnt, "pair_cnt", cur, (E,), _ONLY_I32)
    rmap = 0 if row_map is None else _dense(row_map, "the row map", cur, (P,), _ONLY_I32)
    if out is None:
        out_code = _DT.get(out_dtype)
        if out_code is None:
            raise ValueError(f"out_dtype is {out_dtype}")
        out = x.new_empty(P, N, dtype=out_dtype)
        out_ptr, ldo = out.data_ptr(), N
    else:
        out_ptr, out_code, ldo = _rows(out, "out", cur, (P, N))
    a = _expert_args(x_ptr, xs, ld, w_ptr, w1_ptr, s0_ptr, s1_ptr, idx, cnt, rmap, idx_shape[1], out_ptr, ldo,
                     0 if status is None else _dense(status, "status", cur, (1,), _ONLY_I32), x.shape[0], P, N, K, E,
                     row_div, x_code, x_code, out_code, out_scale)
    check(launch(a, _raw_stream()))
    return out


def expert_gateup(x, Wg, Wu, pair_idx, pair_cnt, P: int, top_k: int, pair_tok=None, gate_scale=None, up_scale=None, x_scale=None,
                  out_dtype=None, out=None, out_scale: float = 1.0, status=None):
    """silu(x . Wg[e]) * (x . Wu[e]) * out_scale for every routed pair: [P][N] in out_dtype (default: the matrices' type, bf16
    for e4m3 ones). Wg, Wu [E][N][K] bf16 / f16 (x in the same type) or float8_e4m3fn with gate_scale and up_scale f32
    [E][ceil(N/128)][ceil(K/128)] (x e4m3 with x_scale, or f32 / bf16 / f16, which fp8_rows turns into e4m3 rows). x [T][K];
    pair p reads row pair_tok[p], or p // top_k. Rows of pairs that no table entry names are left as they were. status: an i32 tensor of
    one element that is set to 1 when a bounded wait gave up (outputs concerned are NaN), otherwise left as it is."""
    if out_dtype is None:
        out_dtype = torch.bfloat16 if Wg.dtype == _E4M3 else Wg.dtype
    return _expert(lib().knj_expert_gateup_launch, x, x_scale, Wg, Wu, gate_scale, up_scale, pair_idx, pair_cnt, P, pair_tok, top_k, out,
                   out_dtype, out_scale, status)


def expert_proj(a, W, pair_idx, pair_cnt, P: int, pair_row=None, scale=None, a_scale=None, out_dtype=torch.float32, out=None,
                out_scale: float = 1.0, status=None):
    """a . W[e] * out_scale for every routed pair: [P][N] in out_dtype. a holds one row per pair (row pair_row[p] when given,
    else p); types, scales, unnamed rows and status as for expert_gateup."""
    return _expert(lib().knj_expert_proj_launch, a, a_scale, W, None, scale, None, pair_idx, pair_cnt, P, pair_row, 1, out, out_dtype, out_scale,
                   status)


def block_norm(x, y=None, *, post_w=None, gate=None, gate_sigmoid: bool = False, alpha: float = 1.0, beta: float = 1.0, pre_w=None,
               eps: float = 1e-6, stream_dtype=None, norm_dtype=torch.bfloat16, stream_out=None, status=None):
    """What stands between two blocks: s = beta * x + alpha * gate * norm(y; post_w), h = norm(s; pre_w).
    x [T][H] the residual stream, y [T][H] the block's output or None, post_w / pre_w [H] norm weights or None (one type),
    gate [H], [T][1] or [T][H] (through a sigmoid with gate_sigmoid). Returns (s, h): s in stream_dtype (default: x's type;
    None without y unless stream_out or stream_dtype asks for it), h in norm_dtype (None without pre_w), for
    torch.float8_e4m3fn as (codes, scale). stream_out may be x or y and otherwise overlaps neither. status: an i32 tensor of one
    element that is set to 1 when a bounded wait gave up (rows concerned are NaN), otherwise left as it is."""
    cur = _cur()
    x_ptr, x_code, ldx = _rows(x, "x", cur)
    shape = x.shape
    T, H = shape
    s = h = scale = None
    y_ptr = gate_ptr = s_ptr = h_ptr = scale_ptr = post = pre = 0
    y_code = w_code = gate_code = s_code = h_code = ldy = ldg = lds = 0
    kind = GATE_NONE
    if y is not None:
        y_ptr, y_code, ldy = _rows(y, "y", cur, shape)
    if post_w is not None:
        post, w_code = _dense(post_w, "post_w", cur, (H,), _DT), _DT[post_w.dtype]
    if pre_w is not None:
        pre = _dense(pre_w, "pre_w", cur, (H,), _DT)
        if post_w is not None and w_code != _DT[pre_w.dtype]:
            raise ValueError("post_w and pre_w are of one type")
        w_code = _DT[pre_w.dtype]
        h_code = _DT_ALL.get(norm_dtype)
        if h_code is None:
            raise ValueError(f"norm_dtype is {norm_dtype}")
        h = torch.empty_like(x, dtype=norm_dtype, memory_format=torch.contiguous_format)
        h_ptr = h.data_ptr()
        if h_code == DT_E4M3:
            scale = x.new_empty(T, (H + 127) // 128, dtype=torch.float32)
            scale_ptr = scale.data_ptr()
    if gate is not None:
        if gate.dim() == 1:
            gate_ptr, gate_code, kind = _dense(gate, "gate", cur, (H,), _DT), _DT[gate.dtype], GATE_CHANNEL
        else:
            rows_only = gate.shape[1] == 1 and H > 1
            gate_ptr, gate_code, ldg = _rows(gate, "gate", cur, (T, 1) if rows_only else shape)
            kind = GATE_ROW if rows_only else GATE_FULL
    if stream_out is not None:
        s = stream_out
        s_ptr, s_code, lds = _rows(s, "the stream", cur, shape)
    elif y is not None or stream_dtype is not None:
        s_code = x_code if stream_dtype is None else _DT.get(stream_dtype)
        if s_code is None:
            raise ValueError(f"stream_dtype is {stream_dtype}")
        s = torch.empty_like(x, dtype=stream_dtype, memory_format=torch.contiguous_format)
        s_ptr, lds = s.data_ptr(), H
    a = _norm_args(T, H, x_ptr, ldx, y_ptr, ldy, post, pre, gate_ptr, ldg, s_ptr, lds, h_ptr, H, scale_ptr, x_code, y_code, w_code, gate_code,
                   s_code, h_code, kind, 1 if gate_sigmoid else 0, alpha, beta, eps, 0 if status is None else _dense(status, "status", cur, (1,), _ONLY_I32))
    check(lib().knj_block_norm_launch(a, _raw_stream()))
    return s, (h if scale is None else (h, scale))
