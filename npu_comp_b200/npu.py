"""Operator surface of the B200 build, named after the reference's
`b_program_examples/npu.py` (fp16, matmul, run) and the Llama-layer macros of
`b_program_examples/llama_layer.py:71-152` (rmsnorm, rope, attention, FFN).

Where the reference's functions *emit NPU instructions* that mysim later
executes (npu.py:41-47 appends an m_mul program; npu.py:62-71 runs it), these
functions *compute*: they take CUDA tensors, launch the sm_100a kernels of
libnpub.so on the current stream and return CUDA tensors.  Every op calls the
C ABI of include/npub.h through ctypes; there is no CPU or PyTorch fallback.

Errors: invalid shapes/dtypes raise ValueError (the reference raises
CodegenError, d_compiler/npu_compiler/codegen.py:21-22); a failing CUDA call
raises NpubError (the reference's CalledProcessError from run()).
"""
from __future__ import annotations

import functools
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import NpubError  # noqa: F401  (re-exported)

__all__ = [
    "fp16", "quantize_w8", "matmul", "rmsnorm", "add", "swiglu", "softmax", "rope", "attention",
    "attention_decode", "kv_append", "rope_kv_append", "rope_kv_store", "matmul_swiglu", "interleave_gate_up",
    "matmul_rms", "rmsnorm_parts",
    "rope_paged_append", "attention_packed", "attention_paged", "attention_paged_decode",
    "embed", "argmax", "isa_vector", "f32_to_f16_bits", "f16_bits_to_f32", "device_error", "NpubError",
]


def fp16(x: float) -> float:
    """Round a python float through FP16 (b_program_examples/npu.py:7-8)."""
    return struct.unpack('<e', struct.pack('<e', float(x)))[0]


# ----------------------------------------------------------------- helpers

def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _mat(t: torch.Tensor, name: str, dtype: torch.dtype) -> int:
    """Validate a row-major CUDA matrix and return its leading dimension."""
    _need(isinstance(t, torch.Tensor), f"{name} must be a torch.Tensor")
    _need(t.is_cuda, f"{name} must be a CUDA tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(t.dim() == 2, f"{name} must be 2-D, got shape {tuple(t.shape)}")
    _need(t.stride(1) == 1 or t.shape[1] == 1, f"{name} must have unit stride along its last dim")
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device) -> Tuple[Optional[torch.Tensor], int]:
    if nbytes <= 0:
        return None, 0
    ws = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    off = (-ws.data_ptr()) % 256
    return ws[off:off + nbytes], nbytes


# A W8A16 workspace starts with 64 KiB of tile counters for the few-token
# (stream-K) kernel; they must start at zero and every call leaves them at
# zero.  One zero-filled buffer per (device, stream) serves every W8A16 call;
# a grown buffer replaces the old one, which is kept alive for CUDA graphs
# that captured its address.
_zeroed_ws = {}
_retired_ws = []


def device_error(clear: bool = False) -> int:
    """The current device's error word: non-zero when a bounded device-side wait
    gave up (NPUB_ERR_DEVICE_TIMEOUT cases; synchronises the device).

    With clear=True the word is reset, and so are the tile counters of every
    W8A16 workspace this module hands out and of the library's allocation-free
    scratch: a stream-K call whose wait gave up may have left counts there,
    which the next call would take for pieces already written."""
    lib = _lib.load()
    v = int(lib.npub_device_error(1 if clear else 0))
    if v == _lib.NPUB_ERR_CUDA:
        raise NpubError("npub_device_error", v, lib.npub_strerror(v).decode())
    if clear:
        dev = torch.cuda.current_device()
        for (d, _), buf in _zeroed_ws.items():
            if d == dev:
                buf.zero_()
        torch.cuda.synchronize()
    return v


def _zeroed_workspace(nbytes: int, device) -> Tuple[Optional[torch.Tensor], int]:
    if nbytes <= 0:
        return None, 0
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    buf = _zeroed_ws.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _retired_ws.append(buf)
        buf = torch.zeros(max(nbytes, 4 << 20), dtype=torch.uint8, device=device)
        _zeroed_ws[key] = buf
    return buf, buf.numel()


# -------------------------------------------------------------- W8A16 matmul

# When a list, every matmul() call appends (start_event, end_event, flops, int8)
# recorded on the launching stream -- used by bench.py to time the GEMM kernels
# inside a step.
gemm_events = None



def quantize_w8(W: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Symmetric per-output-channel int8 quantisation of W [K, N] fp32 (x @ W).

    Returns (Wq int8 [N, K] K-major, scale fp16 [N]) with
    scale[n] = fp16(max_k |W[k, n]| / 127) and Wq[n, k] = clip(rint(W[k, n] / scale[n]), +-127).
    """
    ldw = _mat(W, "W", torch.float32)
    K, N = W.shape
    q = torch.empty((N, K), dtype=torch.int8, device=W.device)
    s = torch.empty((N,), dtype=torch.float16, device=W.device)
    _lib.call("npub_quantize_w8", W.data_ptr(), ldw, K, N, q.data_ptr(), K, s.data_ptr(), _stream())
    return q, s


def matmul(A: torch.Tensor, W: torch.Tensor, scale: Optional[torch.Tensor] = None, *,
           out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           alpha: float = 1.0) -> torch.Tensor:
    """C[M, N] = fp16(alpha * scale[n] * sum_k A[m, k] W[n, k]) (+ residual[m, n]).

    The reference's matmul (npu.py:41-47) computes C = A @ B with B [K, N]; here
    the weight is packed K-major as W [N, K] -- int8 (W8A16, from quantize_w8)
    or fp16 (W = B.T.contiguous()).  A is fp16 [M, K]; K must be a multiple of 16.
    """
    lda = _mat(A, "A", torch.float16)
    _need(W.dtype in (torch.int8, torch.float16), "W must be int8 or float16")
    ldw = _mat(W, "W", W.dtype)
    M, K = A.shape
    N, K2 = W.shape
    _need(K == K2, f"K mismatch: A {tuple(A.shape)} vs W {tuple(W.shape)}")
    if scale is not None:
        _need(scale.is_cuda and scale.dtype == torch.float16 and scale.numel() == N and scale.is_contiguous(),
              "scale must be a contiguous fp16 CUDA tensor of N elements")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    ldc = _mat(out, "out", torch.float16)
    _need(tuple(out.shape) == (M, N), "out must be [M, N]")
    ldr = 0
    if residual is not None:
        ldr = _mat(residual, "residual", torch.float16)
        _need(tuple(residual.shape) == (M, N), "residual must be [M, N]")
    int8 = W.dtype == torch.int8
    wsq = "npub_w8a16_gemm_workspace" if int8 else "npub_f16_gemm_workspace"
    if int8:
        ws, wsb = _zeroed_workspace(_lib.query(wsq, M, N, K), A.device)
    else:
        ws, wsb = _workspace(_lib.query(wsq, M, N, K), A.device)
    fn = "npub_w8a16_gemm" if int8 else "npub_f16_gemm"
    ev = gemm_events
    if ev is not None:
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
    _lib.call(fn, A.data_ptr(), lda, W.data_ptr(), ldw, _ptr(scale), out.data_ptr(), ldc, _ptr(residual), ldr,
              M, N, K, float(alpha), _ptr(ws), wsb, _stream())
    if ev is not None:
        e1.record()
        ev.append((e0, e1, 2.0 * M * N * K, int8))
    return out


def interleave_gate_up(wq: torch.Tensor, scale: torch.Tensor):
    """[gate rows (F) | up rows (F)] -> rows 2c = gate c, 2c + 1 = up c, the
    layout matmul_swiglu takes (int8 [2F, K] and fp16 [2F])."""
    F2, K = wq.shape
    _need(F2 % 2 == 0 and scale.numel() == F2, "gate|up weights need an even row count and one scale per row")
    F = F2 // 2
    w = wq.view(2, F, K).transpose(0, 1).reshape(F2, K).contiguous()
    s = scale.view(2, F).t().reshape(F2).contiguous()
    return w, s


def matmul_swiglu(A: torch.Tensor, Wgu: torch.Tensor, scale: torch.Tensor, *,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[M, F] = fp16(silu(g) * u) with g, u the fp16 W8A16 projections of A
    on the gate and up rows of Wgu (int8 [2F, K], interleaved by
    interleave_gate_up; scale fp16 [2F]): matmul() then swiglu(), fused."""
    lda = _mat(A, "A", torch.float16)
    ldw = _mat(Wgu, "Wgu", torch.int8)
    M, K = A.shape
    F2, K2 = Wgu.shape
    _need(K == K2 and F2 % 2 == 0, f"shape mismatch: A {tuple(A.shape)} vs Wgu {tuple(Wgu.shape)}")
    _need(scale.is_cuda and scale.dtype == torch.float16 and scale.numel() == F2 and scale.is_contiguous(),
          "scale must be a contiguous fp16 CUDA tensor of 2F elements")
    F = F2 // 2
    if out is None:
        out = torch.empty((M, F), dtype=torch.float16, device=A.device)
    ldo = _mat(out, "out", torch.float16)
    _need(tuple(out.shape) == (M, F), "out must be [M, F]")
    ws, wsb = _zeroed_workspace(_lib.query("npub_w8a16_gemm_workspace", M, F2, K), A.device)
    ev = gemm_events
    if ev is not None:
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
    _lib.call("npub_w8a16_gemm_swiglu", A.data_ptr(), lda, Wgu.data_ptr(), ldw, scale.data_ptr(), out.data_ptr(),
              ldo, M, F, K, _ptr(ws), wsb, _stream())
    if ev is not None:
        e1.record()
        ev.append((e0, e1, 2.0 * M * F2 * K, True))
    return out


def matmul_rms(A: torch.Tensor, Wq: torch.Tensor, scale: torch.Tensor, *, out: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, swiglu: bool = False,
               rs: Optional[Tuple[torch.Tensor, int]] = None, eps: float = 1e-5,
               gamma: Optional[torch.Tensor] = None, g_out: Optional[torch.Tensor] = None,
               ss_out: Optional[torch.Tensor] = None, prefetch_next: Optional[torch.Tensor] = None):
    """W8A16 GEMM of a decode step (M <= 64) with an RMSNorm folded in
    (npub_w8a16_gemm_rms): the RMSNorm -> projection pairs of a decode layer
    without the normalised activations' round trip or their own launch.

    rs=(ss, d): A is fp16(h * gamma) of a residual stream h (rmsnorm_parts or a
    producer call below) and row t of the result is scaled by
    1 / sqrt(sum(ss[:, t]) / d + eps) before rounding (before SwiGLU with
    swiglu=True, where Wq holds interleaved gate/up rows and out is [M, N/2]).
    gamma: also return (out, g_out, ss_out) -- g_out = fp16(out * gamma) and
    ss_out [N/32, M] fp32, the next call's rs.  prefetch_next: the int8 weights
    of the next GEMM of a decode chain (same M), whose first tiles go to L2
    while this GEMM runs.  Raises NpubError for M > 64."""
    lda = _mat(A, "A", torch.float16)
    ldw = _mat(Wq, "Wq", torch.int8)
    M, K = A.shape
    N, K2 = Wq.shape
    _need(K == K2, f"K mismatch: A {tuple(A.shape)} vs Wq {tuple(Wq.shape)}")
    _need(scale.is_cuda and scale.dtype == torch.float16 and scale.numel() == N and scale.is_contiguous(),
          "scale must be a contiguous fp16 CUDA tensor of N elements")
    NC = N // 2 if swiglu else N
    if out is None:
        out = torch.empty((M, NC), dtype=torch.float16, device=A.device)
    ldc = _mat(out, "out", torch.float16)
    _need(tuple(out.shape) == (M, NC), f"out must be [{M}, {NC}]")
    ldr = 0
    if residual is not None:
        ldr = _mat(residual, "residual", torch.float16)
        _need(tuple(residual.shape) == (M, N), "residual must be [M, N]")
    rs_p, rs_n, rs_ld, rs_d = None, 0, 0, 0
    if rs is not None:
        ss, rs_d = rs
        _need(ss.is_cuda and ss.dtype == torch.float32 and ss.dim() == 2 and ss.shape[1] >= M and ss.stride(1) == 1,
              "rs[0] must be fp32 CUDA [parts, >= M] with unit column stride")
        rs_p, rs_n, rs_ld = ss, ss.shape[0], ss.stride(0)
    ldg = ss_ld = 0
    if gamma is not None:
        _need(gamma.is_cuda and gamma.dtype == torch.float16 and gamma.numel() == N and gamma.is_contiguous(),
              "gamma must be a contiguous fp16 CUDA tensor of N elements")
        if g_out is None:
            g_out = torch.empty((M, N), dtype=torch.float16, device=A.device)
        if ss_out is None:
            ss_out = torch.empty((N // 32, M), dtype=torch.float32, device=A.device)
        ldg = _mat(g_out, "g_out", torch.float16)
        _need(ss_out.dtype == torch.float32 and ss_out.dim() == 2 and ss_out.shape[0] == N // 32 and
              ss_out.shape[1] >= M and ss_out.stride(1) == 1, "ss_out must be fp32 [N/32, >= M]")
        ss_ld = ss_out.stride(0)
    ws, wsb = _zeroed_workspace(_lib.query("npub_w8a16_gemm_rms_workspace", M, N, K), A.device)
    _lib.call("npub_w8a16_gemm_rms", A.data_ptr(), lda, Wq.data_ptr(), ldw, scale.data_ptr(), out.data_ptr(), ldc,
              _ptr(residual), ldr, M, N, K, 1 if swiglu else 0, _ptr(rs_p), rs_n, rs_ld, int(rs_d), float(eps),
              _ptr(gamma), _ptr(g_out if gamma is not None else None), ldg,
              _ptr(ss_out if gamma is not None else None), ss_ld, _ptr(prefetch_next),
              prefetch_next.stride(0) if prefetch_next is not None else 0,
              prefetch_next.shape[0] if prefetch_next is not None else 0,
              prefetch_next.shape[1] if prefetch_next is not None else 0, _ptr(ws), wsb, _stream())
    return out if gamma is None else (out, g_out, ss_out)


def rmsnorm_parts(x: torch.Tensor, gamma: torch.Tensor, *, g_out: Optional[torch.Tensor] = None,
                  ss_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The (g, ss) that matmul_rms(rs=(ss, d)) takes for an RMSNorm of x
    (fp16 [rows, d], d % 32 == 0): g = fp16(x * gamma), ss [d/32, rows] fp32
    the sums of x^2 over every 32 columns."""
    ldx = _mat(x, "x", torch.float16)
    rows, d = x.shape
    _need(gamma.is_cuda and gamma.dtype == torch.float16 and gamma.numel() == d and gamma.is_contiguous(),
          "gamma must be a contiguous fp16 CUDA tensor of d elements")
    if g_out is None:
        g_out = torch.empty((rows, d), dtype=torch.float16, device=x.device)
    if ss_out is None:
        ss_out = torch.empty((d // 32, rows), dtype=torch.float32, device=x.device)
    ldg = _mat(g_out, "g_out", torch.float16)
    _need(ss_out.dtype == torch.float32 and ss_out.dim() == 2 and ss_out.shape[0] == d // 32 and
          ss_out.shape[1] >= rows and ss_out.stride(1) == 1, "ss_out must be fp32 [d/32, >= rows]")
    _lib.call("npub_rmsnorm_parts", x.data_ptr(), ldx, gamma.data_ptr(), g_out.data_ptr(), ldg, ss_out.data_ptr(),
              ss_out.stride(0), rows, d, _stream())
    return g_out, ss_out


# ---------------------------------------------------------------- vector ops

def rmsnorm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5, *, residual: Optional[torch.Tensor] = None,
            residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """y = fp16(x / sqrt(mean(x^2) + eps) * gamma) per row (legalize.py:30-47).

    With `residual`, h = fp16(x + residual) is formed first (llama_layer.py:139),
    written to `residual_out` (default: a new tensor) and normalised; returns (y, h).
    """
    ldx = _mat(x, "x", torch.float16)
    rows, d = x.shape
    _need(gamma.is_cuda and gamma.dtype == torch.float16 and gamma.numel() == d and gamma.is_contiguous(),
          "gamma must be a contiguous fp16 CUDA tensor of d elements")
    if out is None:
        out = torch.empty((rows, d), dtype=torch.float16, device=x.device)
    ldy = _mat(out, "out", torch.float16)
    ldr = ldxo = 0
    if residual is not None:
        ldr = _mat(residual, "residual", torch.float16)
        _need(tuple(residual.shape) == (rows, d), "residual must match x")
        if residual_out is None:
            residual_out = torch.empty((rows, d), dtype=torch.float16, device=x.device)
        ldxo = _mat(residual_out, "residual_out", torch.float16)
    _lib.call("npub_rmsnorm", x.data_ptr(), ldx, _ptr(residual), ldr, _ptr(residual_out), ldxo, gamma.data_ptr(),
              out.data_ptr(), ldy, rows, d, float(eps), _stream())
    return out if residual is None else (out, residual_out)


def add(a: torch.Tensor, b: torch.Tensor, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = fp16(a + b), the residual add of llama_layer.py:139,152 (fp16 [rows, cols])."""
    lda = _mat(a, "a", torch.float16)
    ldb = _mat(b, "b", torch.float16)
    _need(a.shape == b.shape, "a and b must have the same shape")
    rows, cols = a.shape
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.float16, device=a.device)
    ldo = _mat(out, "out", torch.float16)
    _lib.call("npub_add", a.data_ptr(), lda, b.data_ptr(), ldb, out.data_ptr(), ldo, rows, cols, _stream())
    return out


def swiglu(g: torch.Tensor, u: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h = fp16(g / (1 + exp(-g)) * u) (legalize.py:130-149).  With u=None, g is
    [rows, 2F] holding the gate in its first F columns and up in the last F."""
    if u is None:
        _need(g.dim() == 2 and g.shape[1] % 2 == 0, "g must be [rows, 2F] when u is None")
        F = g.shape[1] // 2
        g, u = g[:, :F], g[:, F:]
    ldg = _mat(g, "g", torch.float16)
    ldu = _mat(u, "u", torch.float16)
    _need(g.shape == u.shape, "g and u must have the same shape")
    rows, cols = g.shape
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.float16, device=g.device)
    ldh = _mat(out, "out", torch.float16)
    _lib.call("npub_swiglu", g.data_ptr(), ldg, u.data_ptr(), ldu, out.data_ptr(), ldh, rows, cols, _stream())
    return out


def softmax(s: torch.Tensor, *, causal: bool = False, scale: float = 1.0, causal_offset: int = 0,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Row softmax of scale*s over the last dim (legalize.py:97-114); causal rows
    r see columns c <= r + causal_offset and get exact zeros elsewhere."""
    _need(s.is_cuda and s.dtype == torch.float16 and s.dim() >= 2 and s.is_contiguous(),
          "s must be a contiguous fp16 CUDA tensor with >= 2 dims")
    rows, cols = s.shape[-2], s.shape[-1]
    batch = s.numel() // max(1, rows * cols)
    _need(cols % 8 == 0, "the row length must be a multiple of 8")
    if out is None:
        out = torch.empty_like(s)
    _need(out.shape == s.shape and out.is_contiguous() and out.dtype == torch.float16, "bad out")
    _lib.call("npub_softmax_rows", s.data_ptr(), out.data_ptr(), cols, rows * cols, batch, rows, cols, float(scale),
              int(causal_offset) if causal else _lib.NPUB_NO_CAUSAL, 1, _stream())
    return out


def _freq_table(inv_freq: Optional[torch.Tensor], head_dim: int, dev) -> Optional[int]:
    if inv_freq is None:
        return None
    _need(inv_freq.is_cuda and inv_freq.device == dev and inv_freq.dtype == torch.float32
          and inv_freq.is_contiguous() and inv_freq.numel() == head_dim // 2,
          "inv_freq must be contiguous fp32 CUDA [head_dim/2] on the tensor's device")
    return inv_freq.data_ptr()


def rope_freqs(head_dim: int, theta: float = 10000.0, *, llama3_scaling=None, device=None) -> torch.Tensor:
    """Per-frequency rates [head_dim/2] (fp32) for the *_freqs RoPE paths:
    theta^(-2i/head_dim), with the Llama-3 frequency scaling of
    legalize.py:50-64 when llama3_scaling is True (the reference's factor 32,
    low 1, high 4, old context 8192) or a tuple (factor, low, high, old_ctx).
    Built on the host by npub_rope_llama3_freqs, then copied to `device`."""
    import ctypes
    if llama3_scaling is True:
        llama3_scaling = (32.0, 1.0, 4.0, 8192.0)
    factor, low, high, old = llama3_scaling if llama3_scaling else (0.0, 1.0, 4.0, 8192.0)
    out = (ctypes.c_float * (head_dim // 2))()
    _lib.call("npub_rope_llama3_freqs", ctypes.addressof(out), int(head_dim), float(theta), float(factor), float(low),
              float(high), float(old))
    t = torch.tensor(list(out), dtype=torch.float32)
    return t.to(device) if device is not None else t


def rope(x: torch.Tensor, heads: int, head_dim: int, *, pos0: int = 0, positions: Optional[torch.Tensor] = None,
         theta: float = 10000.0, inv_freq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """In-place RoPE on the first heads*head_dim columns of x [tokens, >=heads*head_dim]
    (rotate_half convention, llama_layer.py:33-40,96-112).  inv_freq (fp32
    CUDA [head_dim/2], from rope_freqs) replaces theta's frequencies, e.g.
    the Llama-3 scaled ones.  Returns x."""
    ldx = _mat(x, "x", torch.float16)
    tokens = x.shape[0]
    _need(x.shape[1] >= heads * head_dim, "x is narrower than heads*head_dim")
    pos_ptr = None
    if positions is not None:
        _need(positions.is_cuda and positions.dtype == torch.int32 and positions.numel() == tokens
              and positions.is_contiguous(), "positions must be contiguous int32 CUDA [tokens]")
        pos_ptr = positions.data_ptr()
    fp = _freq_table(inv_freq, head_dim, x.device)
    if fp is None:
        _lib.call("npub_rope", x.data_ptr(), ldx, tokens, heads, head_dim, pos_ptr, int(pos0), float(theta),
                  _stream())
    else:
        _lib.call("npub_rope_freqs", x.data_ptr(), ldx, tokens, heads, head_dim, pos_ptr, int(pos0), fp, _stream())
    return x


# ------------------------------------------------------- embedding / argmax

def embed(ids: torch.Tensor, table: torch.Tensor, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of the fp16 embedding table [vocab, d] for int32 token ids [n]."""
    _need(ids.is_cuda and ids.dtype == torch.int32 and ids.is_contiguous(), "ids must be contiguous int32 CUDA")
    ldt = _mat(table, "table", torch.float16)
    vocab, d = table.shape
    n = ids.numel()
    if out is None:
        out = torch.empty((n, d), dtype=torch.float16, device=table.device)
    ldo = _mat(out, "out", torch.float16)
    _lib.call("npub_embed", ids.data_ptr(), n, table.data_ptr(), ldt, vocab, d, out.data_ptr(), ldo, _stream())
    return out


def argmax(x: torch.Tensor, *, idx: Optional[torch.Tensor] = None, val: Optional[torch.Tensor] = None):
    """Per-row (index, value) of the largest fp16 logit (smallest index on ties)."""
    ldx = _mat(x, "x", torch.float16)
    rows, cols = x.shape
    if idx is None:
        idx = torch.empty((rows,), dtype=torch.int32, device=x.device)
    if val is None:
        val = torch.empty((rows,), dtype=torch.float32, device=x.device)
    _lib.call("npub_argmax_rows", x.data_ptr(), ldx, rows, cols, idx.data_ptr(), val.data_ptr(), _stream())
    return idx, val


def argmax_keys(x: torch.Tensor, index_offset: int = 0, *, keys: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-row greedy key (int64 [rows]) of fp16 logits x: the largest value and
    its smallest index + index_offset in one orderable word (npub_argmax_keys);
    select_keys over the keys of every vocabulary shard gives the global argmax."""
    ldx = _mat(x, "x", torch.float16)
    rows, cols = x.shape
    if keys is None:
        keys = torch.empty((rows,), dtype=torch.int64, device=x.device)
    _need(keys.is_cuda and keys.dtype == torch.int64 and keys.numel() == rows and keys.is_contiguous(),
          "keys must be contiguous int64 CUDA [rows]")
    _lib.call("npub_argmax_keys", x.data_ptr(), ldx, rows, cols, int(index_offset), keys.data_ptr(), _stream())
    return keys


def select_keys(keys: torch.Tensor, ranks: int, *, ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ids[b] = index of the largest of keys[r * rows + b] over r < ranks (int32)."""
    _need(keys.is_cuda and keys.dtype == torch.int64 and keys.is_contiguous() and keys.numel() % ranks == 0,
          "keys must be contiguous int64 CUDA [ranks * rows]")
    rows = keys.numel() // ranks
    if ids is None:
        ids = torch.empty((rows,), dtype=torch.int32, device=keys.device)
    _need(ids.is_cuda and ids.dtype == torch.int32 and ids.numel() == rows and ids.is_contiguous(),
          "ids must be contiguous int32 CUDA [rows]")
    _lib.call("npub_select_keys", keys.data_ptr(), int(ranks), rows, ids.data_ptr(), _stream())
    return ids


# ----------------------------------------------------------------- attention

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int, kv_heads: Optional[int] = None, *,
              head_dim: Optional[int] = None, batch: int = 1, causal: bool = True, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal (GQA) attention of llama_layer.py:114-137 for `batch` sequences of
    equal length stacked along rows: q [batch*T, heads*hd], k/v [batch*T, kv_heads*hd]."""
    kv_heads = kv_heads or heads
    ldq = _mat(q, "q", torch.float16)
    ldk = _mat(k, "k", torch.float16)
    ldv = _mat(v, "v", torch.float16)
    hd = head_dim or q.shape[1] // heads
    rows = q.shape[0]
    _need(rows % batch == 0, "rows must be a multiple of batch")
    T = rows // batch
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    if out is None:
        out = torch.empty((rows, heads * hd), dtype=torch.float16, device=q.device)
    ldo = _mat(out, "out", torch.float16)
    ws, wsb = _workspace(_lib.query("npub_attention_workspace", batch, T, heads, hd), q.device)
    _lib.call("npub_attention_prefill", q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo,
              batch, T, heads, kv_heads, hd, float(scale), 1 if causal else 0, _ptr(ws), wsb, _stream())
    return out


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, heads: int,
                     kv_heads: Optional[int] = None, lens: Optional[torch.Tensor] = None, ctx_len: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token per sequence against fp16 caches [batch, kv_heads, cap, 128]."""
    kv_heads = kv_heads or heads
    ldq = _mat(q, "q", torch.float16)
    batch = q.shape[0]
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.is_contiguous() and
          v_cache.is_contiguous() and k_cache.dtype == torch.float16, "caches must be contiguous fp16 [B, KVH, cap, hd]")
    B, KVH, cap, hd = k_cache.shape
    _need(B == batch and KVH == kv_heads, "cache shape does not match q / kv_heads")
    lens_ptr = None
    if lens is not None:
        _need(lens.is_cuda and lens.dtype == torch.int32 and lens.numel() == batch and lens.is_contiguous(),
              "lens must be contiguous int32 CUDA [batch]")
        lens_ptr = lens.data_ptr()
        ctx = int(ctx_len) if ctx_len else cap
    else:
        ctx = int(ctx_len)
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    if out is None:
        out = torch.empty((batch, heads * hd), dtype=torch.float16, device=q.device)
    ldo = _mat(out, "out", torch.float16)
    ws, wsb = _workspace(_lib.query("npub_attention_decode_workspace", batch, heads, ctx, hd), q.device)
    _lib.call("npub_attention_decode", q.data_ptr(), ldq, k_cache.data_ptr(), v_cache.data_ptr(), cap, lens_ptr, ctx,
              out.data_ptr(), ldo, batch, heads, kv_heads, hd, float(scale), _ptr(ws), wsb, _stream())
    return out


def kv_append(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
              pos: Optional[torch.Tensor] = None, pos0: int = 0) -> None:
    """cache[b, h, pos[b], :] = new[b, h*hd:(h+1)*hd] for K and V."""
    ldk = _mat(k_new, "k_new", torch.float16)
    ldv = _mat(v_new, "v_new", torch.float16)
    B, KVH, cap, hd = k_cache.shape
    pos_ptr = None
    if pos is not None:
        _need(pos.is_cuda and pos.dtype == torch.int32 and pos.numel() == B and pos.is_contiguous(),
              "pos must be contiguous int32 CUDA [batch]")
        pos_ptr = pos.data_ptr()
    _lib.call("npub_kv_append", k_new.data_ptr(), ldk, v_new.data_ptr(), ldv, k_cache.data_ptr(), v_cache.data_ptr(),
              cap, pos_ptr, int(pos0), B, KVH, hd, _stream())


# ------------------------------------------------------------ paged KV cache
#
# A paged cache is a pool k_pages / v_pages [n_pages, kv_heads, page_size,
# head_dim] and a table page_table [batch, max_pages] of page ids: key p of
# sequence b is slot p % page_size of page page_table[b, p // page_size].
# Packed rows are the sequences' new rows one after the other, sequence b at
# rows cu_seqlens[b] .. cu_seqlens[b + 1]; rows outside
# cu_seqlens[0] .. cu_seqlens[-1] are neither computed nor written.

# These ops run between two launches of a decode step, where 10 us of Python
# are more than the kernels take: their checks build no message unless they
# fail, and read the stream's handle without making a Stream object (a decode
# step's append: 30 us per call with the checks of the ops above, 12 us so, of
# which 5 us are the C call).

_Tensor, _f16, _i32 = torch.Tensor, torch.float16, torch.int32


class _Here:
    """The context of a tensor on the current device: nothing to do."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_here = _Here()


def _device(dev: int):
    """A context in which device index dev is current."""
    return _here if torch._C._cuda_getDevice() == dev else torch.cuda.device(dev)


def _first16(t: torch.Tensor, name: str):
    """(device index, rows, columns, leading dimension) of an op's first fp16 matrix."""
    if isinstance(t, _Tensor) and t.dtype is _f16 and t.is_cuda:
        s = t.stride()
        if len(s) == 2:
            n, c = t.shape
            if s[1] == 1 or c == 1:
                return t.get_device(), n, c, s[0] if n > 1 else max(s[0], c)
    _mat(t, name, torch.float16)  # raises
    raise ValueError(f"{name} must be a row-major fp16 CUDA matrix")


def _rows16(t: torch.Tensor, name: str, dev: int):
    """(rows, columns, leading dimension) of a further one, on the same device."""
    d, n, c, ld = _first16(t, name)
    if d != dev:
        raise ValueError(f"{name} must be on the same device as the first argument")
    return n, c, ld


def _ints(t: torch.Tensor, name: str, n: int, dev: int) -> int:
    if not (isinstance(t, _Tensor) and t.dtype is _i32 and t.get_device() == dev and t.dim() == 1 and t.numel() == n
            and t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous int32 CUDA [{n}] on the same device as the first argument")
    return t.data_ptr()


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, dev: int):
    """Validate a paged cache; returns ((n_pages, kv_heads, page_size, head_dim), batch, max_pages, ldt)."""
    if not (isinstance(k_pages, _Tensor) and k_pages.dtype is _f16 and k_pages.get_device() == dev
            and k_pages.dim() == 4 and k_pages.is_contiguous() and isinstance(v_pages, _Tensor)
            and v_pages.dtype is _f16 and v_pages.get_device() == dev and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous fp16 CUDA [n_pages, kv_heads, page_size, head_dim] on "
                         "the same device as the first argument")
    shape = k_pages.shape
    if v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must have the same shape")
    if not (isinstance(page_table, _Tensor) and page_table.dtype is _i32 and page_table.get_device() == dev):
        raise ValueError("page_table must be int32 CUDA [batch, max_pages] on the same device as the first argument")
    s = page_table.stride()
    if len(s) != 2 or (s[1] != 1 and page_table.shape[1] != 1):
        raise ValueError("page_table must be [batch, max_pages] with unit stride along its last dim")
    B, W = page_table.shape
    return shape, B, W, s[0] if B > 1 else max(s[0], W)


def _out16(out: Optional[torch.Tensor], like: torch.Tensor, rows: int, cols: int, dev: int):
    """(output [rows, cols], its leading dimension)"""
    if out is None:
        return like.new_empty(rows, cols), cols
    n, c, ld = _rows16(out, "out", dev)
    if n != rows or c != cols:
        raise ValueError(f"out must be [{rows}, {cols}]")
    return out, ld


def _context(ctx_len: int, width: int) -> int:
    """The keys that a call's split is planned for, as the C entries take them (a table may be wider than an int)."""
    return min(int(ctx_len) if ctx_len > 0 else width, width, 2 ** 31 - 1)


@functools.lru_cache(maxsize=4096)
def _paged_query(dev: int, name: str, *sizes: int) -> int:
    with torch.cuda.device(dev):
        return _lib.query(name, *sizes)  # a function of the sizes and the device's SM count


def _paged_workspace(like: torch.Tensor, dev: int, name: str, *sizes: int):
    """(tensor that holds the workspace or None, its address or None, its size)"""
    n = _paged_query(dev, name, *sizes)
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=like.device)
    p = ws.data_ptr()
    if p % 256:
        ws, _ = _workspace(n, like.device)
        p = ws.data_ptr()
    return ws, p, n


def rope_paged_append(qkv: torch.Tensor, q_heads: int, kv_heads: int, head_dim: int, positions: torch.Tensor,
                      inv_freq: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      page_table: torch.Tensor, *, cu_seqlens: Optional[torch.Tensor] = None,
                      rot_dim: Optional[int] = None, interleaved: bool = False,
                      q_gamma: Optional[torch.Tensor] = None, k_gamma: Optional[torch.Tensor] = None,
                      eps: float = 1e-5, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The step between the QKV projection and the attention over a paged cache,
    in one kernel: an RMSNorm of every q / k head (with q_gamma / k_gamma), RoPE
    (llama_layer.py:96-112) of the q and k heads of the fused rows qkv
    [tokens, (q_heads + 2 kv_heads) * head_dim], k and v written to the pages at
    positions[t].  Returns q [tokens, q_heads * head_dim] (out; may be the q
    columns of qkv).

    cu_seqlens (int32 [batch + 1]): packed prompts; None: row t is sequence t's.
    inv_freq (fp32 [rot_dim / 2], from rope_freqs): the rotation's rates;
    rot_dim < head_dim rotates the first rot_dim columns only; interleaved
    pairs columns (2i, 2i + 1) instead of (i, i + rot_dim / 2).  A position
    outside the table, or a page id outside the pool, is rotated but not stored.
    Rows with the same slot leave columns of several of them in it."""
    dev, T, cols, ldx = _first16(qkv, "qkv")
    R = head_dim if rot_dim is None else int(rot_dim)
    if cols < (q_heads + 2 * kv_heads) * head_dim:
        raise ValueError("qkv has too few columns")
    (n_pages, kvh, ps, hd), B, W, ldt = _pool(k_pages, v_pages, page_table, dev)
    if kvh != kv_heads or hd != head_dim:
        raise ValueError("the pages' kv_heads and head_dim must match")
    pos = _ints(positions, "positions", T, dev)
    if not (isinstance(inv_freq, _Tensor) and inv_freq.dtype is torch.float32 and inv_freq.get_device() == dev
            and inv_freq.is_contiguous() and inv_freq.numel() * 2 == R):
        raise ValueError("inv_freq must be contiguous fp32 CUDA [rot_dim/2]")
    gq = gk = None
    if q_gamma is not None or k_gamma is not None:
        for g in (q_gamma, k_gamma):
            if g is not None and not (isinstance(g, _Tensor) and g.dtype is _f16 and g.get_device() == dev
                                      and g.numel() == head_dim and g.is_contiguous()):
                raise ValueError("q_gamma and k_gamma must be contiguous fp16 CUDA tensors of head_dim elements")
        gq, gk = _ptr(q_gamma), _ptr(k_gamma)
    if cu_seqlens is None:
        if B != T:
            raise ValueError("without cu_seqlens the table needs one row per token")
        cu = None
    else:
        cu = _ints(cu_seqlens, "cu_seqlens", B + 1, dev)
    out, ldq = _out16(out, qkv, T, q_heads * head_dim, dev)
    with _device(dev):
        st = _lib.bound("npub_rope_paged_append")(
            qkv.data_ptr(), ldx, out.data_ptr(), ldq, T, q_heads, kv_heads, head_dim, R,
            1 if interleaved else 0, pos, inv_freq.data_ptr(), gq, gk, eps, k_pages.data_ptr(), v_pages.data_ptr(),
            n_pages, ps, page_table.data_ptr(), ldt, W, cu, B, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.fail("npub_rope_paged_append", st)
    return out


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, heads: int,
                     kv_heads: Optional[int] = None, *, head_dim: Optional[int] = None, causal: bool = True,
                     scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention() (llama_layer.py:114-137) over packed prompts of different
    lengths: q [total, heads*hd], k/v [total, kv_heads*hd], sequence b at rows
    cu_seqlens[b] .. cu_seqlens[b + 1] (int32 [batch + 1]).  head_dim a multiple
    of 16 up to 128."""
    kv_heads = kv_heads or heads
    _need(heads > 0 and kv_heads > 0, "heads and kv_heads must be positive")
    dev, T, qc, ldq = _first16(q, "q")
    Tk, kc, ldk = _rows16(k, "k", dev)
    Tv, vc, ldv = _rows16(v, "v", dev)
    hd = head_dim or qc // heads
    if Tk != T or Tv != T:
        raise ValueError("q, k and v must have the same number of rows")
    if qc < heads * hd or kc < kv_heads * hd or vc < kv_heads * hd:
        raise ValueError("q, k or v is narrower than its heads")
    B = (cu_seqlens.numel() if isinstance(cu_seqlens, _Tensor) else 0) - 1
    if B < 0:
        raise ValueError("cu_seqlens must hold batch + 1 offsets")
    cu = _ints(cu_seqlens, "cu_seqlens", B + 1, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(max(hd, 1))
    out, ldo = _out16(out, q, T, heads * hd, dev)
    with _device(dev):
        st = _lib.bound("npub_attention_packed")(
            q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo,
            cu, B, T, heads, kv_heads, hd, scale, 1 if causal else 0, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.fail("npub_attention_packed", st)
    return out


def attention_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    lens: torch.Tensor, cu_seqlens: torch.Tensor, *, heads: int, max_new: int = 0, ctx_len: int = 0,
                    causal: bool = True, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed new rows q [total, heads*hd] over a paged cache that
    holds them already: sequence b's keys are positions 0 .. lens[b] - 1 (int32
    [batch]) and its new rows (cu_seqlens) the last of them.  Prompt chunks,
    prompts behind a cached prefix, drafted tokens.

    max_new: at least the new rows of any sequence (0: not known); up to
    r = 16 * kv_heads / heads of them run on the kernel for few rows, where a
    sequence that has more than r rows all the same gets zeros for those past
    its first r.  ctx_len: the largest lens expected (0: the table's width),
    which only decides how keys are split over CTAs.  page_size 16 .. 256."""
    dev, T, qc, ldq = _first16(q, "q")
    (n_pages, kv_heads, ps, hd), B, W, ldt = _pool(k_pages, v_pages, page_table, dev)
    if qc != heads * hd:
        raise ValueError("q must be [total, heads * head_dim]")
    ln = _ints(lens, "lens", B, dev)
    cu = _ints(cu_seqlens, "cu_seqlens", B + 1, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(max(hd, 1))
    max_new = min(int(max_new), 2 ** 31 - 1)
    ctx = _context(ctx_len, W * ps)
    out, ldo = _out16(out, q, T, heads * hd, dev)
    ws, wsp, wsb = _paged_workspace(q, dev, "npub_attention_paged_workspace", B, T, max_new, ctx, heads, kv_heads, hd)
    with _device(dev):
        st = _lib.bound("npub_attention_paged")(
            q.data_ptr(), ldq, k_pages.data_ptr(), v_pages.data_ptr(), n_pages, ps,
            page_table.data_ptr(), ldt, W, ln, cu, B, T, max_new, ctx, out.data_ptr(), ldo, heads, kv_heads, hd, scale,
            1 if causal else 0, wsp, wsb, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.fail("npub_attention_paged", st)
    return out


def attention_paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lens: torch.Tensor, *, heads: int, shared_len: int = 0, ctx_len: int = 0,
                           scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention_decode() over a paged cache: q [batch, heads*hd], one new row
    per sequence, keys 0 .. lens[b] - 1.

    shared_len (a multiple of page_size): the first shared_len keys of every
    sequence are in the same pages (a common prefix); they are read through the
    table's first row, where it pays once for the batch.  The result is that of
    shared_len=0 up to rounding, also for sequences shorter than shared_len.
    ctx_len: the largest lens expected (0: the table's width)."""
    dev, n, qc, ldq = _first16(q, "q")
    (n_pages, kv_heads, ps, hd), B, W, ldt = _pool(k_pages, v_pages, page_table, dev)
    if n != B or qc != heads * hd:
        raise ValueError("q must be [batch, heads * head_dim]")
    ln = _ints(lens, "lens", B, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(max(hd, 1))
    shared_len = int(shared_len)
    if not 0 <= shared_len <= min(W * ps, 2 ** 31 - 1):
        raise ValueError("shared_len must lie within the table, below 2^31")
    ctx = _context(ctx_len, W * ps)
    out, ldo = _out16(out, q, B, heads * hd, dev)
    ws, wsp, wsb = _paged_workspace(q, dev, "npub_attention_paged_decode_workspace", B, ctx, shared_len, heads,
                                    kv_heads, hd)
    with _device(dev):
        st = _lib.bound("npub_attention_paged_decode")(
            q.data_ptr(), ldq, k_pages.data_ptr(), v_pages.data_ptr(), n_pages, ps,
            page_table.data_ptr(), ldt, W, ln, B, ctx, shared_len, out.data_ptr(), ldo, heads, kv_heads, hd, scale,
            wsp, wsb, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.fail("npub_attention_paged_decode", st)
    return out


# --------------------------------------------------------- NPU ISA semantics

def rope_kv_append(qkv: torch.Tensor, q_heads: int, kv_heads: int, head_dim: int, positions: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor, *, theta: float = 10000.0,
                   lens: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None) -> None:
    """Decode step: rope() on the q and k heads of the fused QKV rows (in place)
    and kv_append() of the rotated k and the v heads at positions[t], in one
    kernel; lens (int32 [tokens], optional) receives positions + 1."""
    ldx = _mat(qkv, "qkv", torch.float16)
    T = qkv.shape[0]
    _need(qkv.shape[1] >= (q_heads + 2 * kv_heads) * head_dim, "qkv has too few columns")
    _need(positions.is_cuda and positions.dtype == torch.int32 and positions.numel() == T
          and positions.is_contiguous(), "positions must be contiguous int32 CUDA [tokens]")
    for c, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(c.is_cuda and c.dtype == torch.float16 and c.is_contiguous() and c.dim() == 4
              and tuple(c.shape[:2]) == (T, kv_heads) and c.shape[3] == head_dim,
              f"{n} must be contiguous fp16 CUDA [tokens, kv_heads, cap, head_dim]")
    if lens is not None:
        _need(lens.is_cuda and lens.dtype == torch.int32 and lens.numel() == T and lens.is_contiguous(),
              "lens must be contiguous int32 CUDA [tokens]")
    fp = _freq_table(inv_freq, head_dim, qkv.device)
    if fp is None:
        _lib.call("npub_rope_kv_append", qkv.data_ptr(), ldx, T, q_heads, kv_heads, head_dim, positions.data_ptr(),
                  float(theta), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[2], _ptr(lens), _stream())
    else:
        _lib.call("npub_rope_kv_append_freqs", qkv.data_ptr(), ldx, T, q_heads, kv_heads, head_dim,
                  positions.data_ptr(), fp, k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[2], _ptr(lens),
                  _stream())


def rope_kv_store(qkv: torch.Tensor, q_heads: int, kv_heads: int, head_dim: int, positions: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, *, tokens_per_seq: int,
                  theta: float = 10000.0, inv_freq: Optional[torch.Tensor] = None) -> None:
    """Prefill: rope() on the q and k heads of the fused QKV rows of `batch`
    prompts (rows r = b * tokens_per_seq + i, in place) and the rotated k and the
    v heads written to the caches [batch, kv_heads, cap, head_dim] at
    positions[r], in one kernel."""
    ldx = _mat(qkv, "qkv", torch.float16)
    T = qkv.shape[0]
    _need(tokens_per_seq > 0 and T % tokens_per_seq == 0, "rows must be a whole number of sequences")
    _need(qkv.shape[1] >= (q_heads + 2 * kv_heads) * head_dim, "qkv has too few columns")
    _need(positions.is_cuda and positions.dtype == torch.int32 and positions.numel() == T
          and positions.is_contiguous(), "positions must be contiguous int32 CUDA [tokens]")
    batch = T // tokens_per_seq
    for c, nm in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(c.is_cuda and c.dtype == torch.float16 and c.is_contiguous() and c.dim() == 4
              and tuple(c.shape[:2]) == (batch, kv_heads) and c.shape[3] == head_dim,
              f"{nm} must be contiguous fp16 CUDA [batch, kv_heads, cap, head_dim]")
    fp = _freq_table(inv_freq, head_dim, qkv.device)
    if fp is None:
        _lib.call("npub_rope_kv_store", qkv.data_ptr(), ldx, T, tokens_per_seq, q_heads, kv_heads, head_dim,
                  positions.data_ptr(), float(theta), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[2],
                  _stream())
    else:
        _lib.call("npub_rope_kv_store_freqs", qkv.data_ptr(), ldx, T, tokens_per_seq, q_heads, kv_heads, head_dim,
                  positions.data_ptr(), fp, k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[2], _stream())


def isa_vector(word: int, in1: torch.Tensor, in2: Optional[torch.Tensor] = None,
               prev_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Execute one elementwise NPU compute instruction (_poc/mysim.cpp:114-141)
    over fp32 PE buffers; returns the PE output buffer (fp32)."""
    for t, nm in ((in1, "in1"), (in2, "in2"), (prev_out, "prev_out")):
        if t is not None:
            _need(t.is_cuda and t.dtype == torch.float32 and t.is_contiguous(), f"{nm} must be contiguous fp32 CUDA")
    n = in1.numel()
    out = torch.empty(n, dtype=torch.float32, device=in1.device)
    _lib.call("npub_isa_vector", int(word) & 0xFFFFFFFF, in1.data_ptr(), _ptr(in2), _ptr(prev_out), out.data_ptr(), n,
              _stream())
    return out


def f32_to_f16_bits(x: torch.Tensor) -> torch.Tensor:
    """The cmodel's store rounding (mysim.cpp:19-38): fp32 -> fp16 bit patterns (int16)."""
    _need(x.is_cuda and x.dtype == torch.float32 and x.is_contiguous(), "x must be contiguous fp32 CUDA")
    y = torch.empty(x.shape, dtype=torch.int16, device=x.device)
    _lib.call("npub_f32_to_f16", x.data_ptr(), y.data_ptr(), x.numel(), _stream())
    return y


def f16_bits_to_f32(x: torch.Tensor) -> torch.Tensor:
    _need(x.is_cuda and x.dtype in (torch.int16, torch.float16) and x.is_contiguous(), "x must be 16-bit CUDA")
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    _lib.call("npub_f16_to_f32", x.data_ptr(), y.data_ptr(), x.numel(), _stream())
    return y
