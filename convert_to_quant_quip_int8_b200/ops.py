"""torch-facing wrappers of the libqi8 kernels.

Outputs are allocated here with the PyTorch caching allocator (the C library
never allocates); every launch goes on ``torch.cuda.current_stream()``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L


def _next_pow2(n: int) -> int:
    return 1 if n <= 1 else 1 << (n - 1).bit_length()


def _rows2d(x: torch.Tensor) -> torch.Tensor:
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    return x2


def _sign(s: Optional[torch.Tensor], n: int, device) -> Optional[torch.Tensor]:
    if s is None:
        return None
    s = s.to(device=device, dtype=torch.float32).contiguous().reshape(-1)
    assert s.numel() == n, f"sign vector has {s.numel()} entries, expected {n}"
    return s


def quant_rows(x: torch.Tensor, mode: int = L.QI8_Q_TOKEN, block: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-token (mode TOKEN) or per-128-block (mode BLOCK) int8 quantization of
    the last dimension.  Returns ``(q int8 [..., n], scale fp32 [...] or [..., n/128])``."""
    L.require_cuda(x)
    x2 = _rows2d(x)
    rows, n = x2.shape
    q = torch.empty((rows, n), dtype=torch.int8, device=x.device)
    base_mode = mode & 0xFF
    ns = 1 if base_mode == L.QI8_Q_TOKEN else n // block
    s = torch.empty((rows, ns), dtype=torch.float32, device=x.device)
    lib = L.load()
    L.check(lib.qi8_quant_rows(L.ptr(x2), L.dtype_code(x2.dtype), rows, n, x2.stride(0), mode, block,
                               L.ptr(q), n, L.ptr(s), L.stream_ptr(x.device)), "qi8_quant_rows")
    q = q.reshape(x.shape)
    if base_mode == L.QI8_Q_TOKEN:
        return q, s.reshape(*x.shape[:-1], 1)
    return q, s.reshape(*x.shape[:-1], ns)


def rotate_quant_rows(x: torch.Tensor, sign: Optional[torch.Tensor], n_pad: Optional[int] = None,
                      normalize: bool = True, mode: int = L.QI8_Q_TOKEN) -> Tuple[torch.Tensor, torch.Tensor]:
    """K1: ``quant(FWHT(pad(x, n_pad) * sign))``.  Returns ``(q [rows, n_pad], scale)``."""
    L.require_cuda(x)
    x2 = _rows2d(x)
    rows, n = x2.shape
    n_pad = n_pad or _next_pow2(n)
    if n_pad & (n_pad - 1):
        raise ValueError(f"Last dimension must be a power of 2, got {n_pad}")
    q = torch.empty((rows, n_pad), dtype=torch.int8, device=x.device)
    ns = 1 if mode == L.QI8_Q_TOKEN else n_pad // 128
    s = torch.empty((rows, ns), dtype=torch.float32, device=x.device)
    sg = _sign(sign, n_pad, x.device)
    lib = L.load()
    L.check(lib.qi8_rotate_quant_rows(L.ptr(x2), L.dtype_code(x2.dtype), rows, n, x2.stride(0), n_pad,
                                      L.ptr(sg), int(normalize), mode, L.ptr(q), L.ptr(s),
                                      L.stream_ptr(x.device)), "qi8_rotate_quant_rows")
    return q, s


def fwht_rows(x: torch.Tensor, n_pad: Optional[int] = None, pre_sign: Optional[torch.Tensor] = None,
              post_sign: Optional[torch.Tensor] = None, normalize: bool = True,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """FWHT of every row (last dim) to fp32 ``[..., n_pad]``."""
    L.require_cuda(x)
    x2 = _rows2d(x)
    rows, n = x2.shape
    n_pad = n_pad or n
    if n_pad & (n_pad - 1) or n_pad < 1:
        raise ValueError(f"Last dimension must be a power of 2, got {n_pad}")
    if out is None:
        out = torch.empty((rows, n_pad), dtype=torch.float32, device=x.device)
    lib = L.load()
    L.check(lib.qi8_fwht_rows(L.ptr(x2), L.dtype_code(x2.dtype), rows, n, x2.stride(0), n_pad,
                              L.ptr(_sign(pre_sign, n_pad, x.device)), L.ptr(_sign(post_sign, n_pad, x.device)),
                              int(normalize), L.ptr(out), L.stream_ptr(x.device)), "qi8_fwht_rows")
    return out.reshape(*x.shape[:-1], n_pad)


def fwht_cols_(x: torch.Tensor, final_mode: int = 0, factor: float = 1.0) -> torch.Tensor:
    """In-place FWHT down the columns of a contiguous fp32 matrix ``[rows, cols]``."""
    L.require_cuda(x)
    assert x.dtype == torch.float32 and x.dim() == 2 and x.stride(1) == 1, "x must be a row-major fp32 matrix"
    rows, cols = x.shape
    if rows & (rows - 1):
        raise ValueError(f"Second-to-last dimension must be power of 2, got {rows}")
    lib = L.load()
    L.check(lib.qi8_fwht_cols(L.ptr(x), rows, cols, x.stride(0), final_mode, float(factor),
                              L.stream_ptr(x.device)), "qi8_fwht_cols")
    return x


def unrotate_rows(y_had: torch.Tensor, sign_u: Optional[torch.Tensor], n_out: int,
                  bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """K3: ``(FWHT(y_had) * sign_u)[:, :n_out] + bias`` -> ``out_dtype``."""
    L.require_cuda(y_had)
    assert y_had.dtype == torch.float32 and y_had.is_contiguous(), "y_had must be contiguous fp32"
    rows, n_pad = y_had.reshape(-1, y_had.shape[-1]).shape
    out = torch.empty((rows, n_out), dtype=out_dtype, device=y_had.device)
    b = None if bias is None else bias.contiguous()
    lib = L.load()
    L.check(lib.qi8_unrotate_rows(L.ptr(y_had), rows, n_pad, L.ptr(_sign(sign_u, n_pad, y_had.device)),
                                  L.ptr(b), L.dtype_code(b.dtype) if b is not None else 0, n_out, L.ptr(out),
                                  L.dtype_code(out_dtype), n_out, L.stream_ptr(y_had.device)),
            "qi8_unrotate_rows")
    return out


def scale_kind(scale: Optional[torch.Tensor], rows: int, K: int, is_weight: bool, block: int = 128) -> int:
    """Classify a scale tensor for ``gemm_i8`` by its element count."""
    if scale is None:
        return L.QI8_S_NONE
    n = scale.numel()
    kb = K // block
    if n == 1 and not (rows == 1 and kb == 1 and scale.dim() >= 2):
        return L.QI8_S_SCALAR
    if n == rows:
        return L.QI8_S_ROW
    if n == rows * kb:
        return L.QI8_S_ROW_KBLOCK
    if is_weight and n == ((rows + block - 1) // block) * kb:
        return L.QI8_S_TILE128
    raise AssertionError(f"cannot interpret scale of shape {tuple(scale.shape)} for rows={rows}, K={K}")


def gemm_i8(a: torch.Tensor, b: torch.Tensor, a_scale: Optional[torch.Tensor] = None, a_kind: Optional[int] = None,
            b_scale: Optional[torch.Tensor] = None, b_kind: Optional[int] = None,
            bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
            act: int = L.QI8_ACT_NONE, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """K2: ``a [M, K] int8 . b [N, K]^T int8`` with the fused epilogue."""
    L.require_cuda(a, b)
    assert a.dtype == torch.int8 and b.dtype == torch.int8, "int8 operands required"
    a2 = a.reshape(-1, a.shape[-1])
    assert a2.is_contiguous() and b.is_contiguous() and b.dim() == 2, "Input tensors must be contiguous"
    M, K = a2.shape
    N = b.shape[0]
    assert b.shape[1] == K, f"Shape mismatch: b.shape={tuple(b.shape)}, expected [N, {K}]"
    if a_scale is not None:
        a_scale = a_scale.to(torch.float32).contiguous()
        a_kind = scale_kind(a_scale, M, K, False) if a_kind is None else a_kind
    else:
        a_kind = L.QI8_S_NONE
    if b_scale is not None:
        b_scale = b_scale.to(torch.float32).contiguous()
        b_kind = scale_kind(b_scale, N, K, True) if b_kind is None else b_kind
    else:
        b_kind = L.QI8_S_NONE
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    bb = None if bias is None else bias.contiguous()
    lib = L.load()
    # small output grids split K (int32 partials in a workspace, identical results)
    ws_bytes = _gemm_ws_bytes(M, N, K, a_kind, b_kind)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=a.device) if ws_bytes else None
    L.check(lib.qi8_gemm_i8_ws(L.ptr(a2), L.ptr(b), M, N, K, L.ptr(a_scale), a_kind, L.ptr(b_scale), b_kind,
                               L.ptr(bb), L.dtype_code(bb.dtype) if bb is not None else 0, L.ptr(out),
                               L.dtype_code(out.dtype), out.stride(0), act, L.ptr(ws), ws_bytes,
                               L.stream_ptr(a.device)), "qi8_gemm_i8")
    return out.reshape(*a.shape[:-1], N)


def gemm_i8_quant(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
                  bias: Optional[torch.Tensor] = None, out_block: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """K2 with the output requantized per (row, 128-column block) in the
    epilogue: ``a [..., K]`` int8 with block scales ``[..., K/128]``, ``b [N, K]``
    with ``[N/128, K/128]`` tile or ``[N, K/128]`` row-block scales.  Returns
    ``(q int8 [..., N], scale fp32 [..., N/128])``."""
    L.require_cuda(a, b)
    assert a.dtype == torch.int8 and b.dtype == torch.int8, "int8 operands required"
    a2 = a.reshape(-1, a.shape[-1])
    assert a2.is_contiguous() and b.is_contiguous() and b.dim() == 2, "Input tensors must be contiguous"
    M, K = a2.shape
    N = b.shape[0]
    assert b.shape[1] == K, f"Shape mismatch: b.shape={tuple(b.shape)}, expected [N, {K}]"
    assert N % out_block == 0, f"N={N} must be divisible by out_block_size={out_block}"
    a_scale = a_scale.to(torch.float32).contiguous()
    b_scale = b_scale.to(torch.float32).contiguous()
    assert a_scale.numel() == M * (K // 128), f"activation scales of shape {tuple(a_scale.shape)}"
    b_kind = L.QI8_S_ROW_KBLOCK if b_scale.numel() == N * (K // 128) else scale_kind(b_scale, N, K, True)
    q = torch.empty((M, N), dtype=torch.int8, device=a.device)
    s = torch.empty((M, N // out_block), dtype=torch.float32, device=a.device)
    bb = None if bias is None else bias.contiguous()
    L.check(L.load().qi8_gemm_i8_quant(L.ptr(a2), L.ptr(b), M, N, K, L.ptr(a_scale), L.QI8_S_ROW_KBLOCK,
                                       L.ptr(b_scale), b_kind, L.ptr(bb), L.dtype_code(bb.dtype) if bb is not None else 0,
                                       L.ptr(q), N, L.ptr(s), out_block, L.stream_ptr(a.device)), "qi8_gemm_i8_quant")
    return q.reshape(*a.shape[:-1], N), s.reshape(*a.shape[:-1], N // out_block)


def int8_gelu(q: torch.Tensor, scale: torch.Tensor, block: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """GELU of a block-quantized int8 activation, requantized per block."""
    L.require_cuda(q, scale)
    assert q.dtype == torch.int8 and q.is_contiguous() and scale.is_contiguous(), "Input tensors must be contiguous"
    n = q.shape[-1]
    rows = q.numel() // n
    q_out = torch.empty_like(q)
    s_out = torch.empty(scale.shape, dtype=torch.float32, device=q.device)
    L.check(L.load().qi8_int8_gelu(L.ptr(q), L.ptr(scale.to(torch.float32)), rows, n, block, L.ptr(q_out),
                                   L.ptr(s_out), L.stream_ptr(q.device)), "qi8_int8_gelu")
    return q_out, s_out


_WS_CACHE = {}


def _gemm_ws_bytes(M: int, N: int, K: int, a_kind: int, b_kind: int) -> int:
    key = (torch.cuda.current_device(), M, N, K, a_kind, b_kind)
    v = _WS_CACHE.get(key)
    if v is None:
        v = _WS_CACHE[key] = int(L.load().qi8_gemm_workspace_bytes(M, N, K, a_kind, b_kind))
    return v


def dequant(q: torch.Tensor, scale: torch.Tensor, kind: int, block: int = 128,
            out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    out = _fast("dequant", q, scale, kind, block, out_dtype)
    if out is not None:
        return out
    L.require_cuda(q, scale)
    q2 = q.reshape(-1, q.shape[-1]).contiguous()
    rows, n = q2.shape
    out = torch.empty((rows, n), dtype=out_dtype, device=q.device)
    lib = L.load()
    L.check(lib.qi8_dequant(L.ptr(q2), rows, n, L.ptr(scale.to(torch.float32).contiguous()), kind, block,
                            L.ptr(out), L.dtype_code(out_dtype), L.stream_ptr(q.device)), "qi8_dequant")
    return out.reshape(q.shape)


def quant_weight(w: torch.Tensor, kind: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tensorwise (SCALAR), per-row (ROW) or Triton-style 128x128 tile (TILE128) weight quantization."""
    L.require_cuda(w)
    w2 = w.reshape(-1, w.shape[-1]).contiguous()
    rows, n = w2.shape
    q = torch.empty((rows, n), dtype=torch.int8, device=w.device)
    if kind == L.QI8_S_SCALAR:
        s = torch.empty((), dtype=torch.float32, device=w.device)
    elif kind == L.QI8_S_ROW:
        s = torch.empty((rows, 1), dtype=torch.float32, device=w.device)
    else:
        s = torch.empty((rows // 128, n // 128), dtype=torch.float32, device=w.device)
    ws = torch.empty(64, dtype=torch.uint8, device=w.device)
    lib = L.load()
    L.check(lib.qi8_quant_weight(L.ptr(w2), L.dtype_code(w2.dtype), rows, n, kind, L.ptr(q), L.ptr(s), L.ptr(ws),
                                 ws.numel(), L.stream_ptr(w.device)), "qi8_quant_weight")
    return q.reshape(w.shape), s


def quip_workspace_bytes(M: int, N: int) -> int:
    return int(L.load().qi8_quip_workspace_bytes(M, N))


def quip_convert(w: torch.Tensor, s_u: torch.Tensor, s_v: torch.Tensor, store_transformed: bool = False,
                 requant: int = L.QI8_REQ_ROW, block: int = 128, want_dequant: bool = True,
                 workspace: Optional[torch.Tensor] = None):
    """K4: QuIP Hadamard conversion of one weight.  Returns ``(q, scale, dequantized_weight or None)``."""
    L.require_cuda(w)
    assert w.dim() == 2, "weight must be 2-D"
    w = w.contiguous()
    M, N = w.shape
    Mp, Np = _next_pow2(M), _next_pow2(N)
    su = _sign(s_u, Mp, w.device)
    sv = _sign(s_v, Np, w.device)
    nbytes = quip_workspace_bytes(M, N)
    if workspace is None or workspace.numel() < nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
    if store_transformed:
        q = torch.empty((Mp, Np), dtype=torch.int8, device=w.device)
        s = torch.empty((Mp, 1), dtype=torch.float32, device=w.device)
    else:
        q = torch.empty((M, N), dtype=torch.int8, device=w.device)
        if requant == L.QI8_REQ_BLOCK and N % block == 0:
            s = torch.empty((M, N // block, 1), dtype=torch.float32, device=w.device)
        elif requant == L.QI8_REQ_GLOBAL:
            s = torch.empty((), dtype=torch.float32, device=w.device)
        else:
            s = torch.empty((M, 1), dtype=torch.float32, device=w.device)
    deq = torch.empty((M, N), dtype=torch.float32, device=w.device) if want_dequant else None
    lib = L.load()
    L.check(lib.qi8_quip_convert(L.ptr(w), L.dtype_code(w.dtype), M, N, L.ptr(su), L.ptr(sv), int(store_transformed),
                                 requant, block, L.ptr(q), L.ptr(s), L.ptr(deq), L.ptr(workspace), workspace.numel(),
                                 L.stream_ptr(w.device)), "qi8_quip_convert")
    return q, s, deq


def weight_rotate2d(w: torch.Tensor, s_u: torch.Tensor, s_v: torch.Tensor, inverse: bool = False,
                    shape: Optional[tuple] = None) -> torch.Tensor:
    """Two-sided signed Hadamard rotation of a weight (the converter's
    incoherence step, converters/quip_int8.py:523-551 / :1489-1506).

    Forward: ``w`` [M, N] -> fp32 [M_pad, N_pad] = FHT_N(FHT_M(pad(w) s_u s_v^T)).
    Inverse: ``w`` [M_pad, N_pad] -> fp32 ``shape`` (default [M_pad, N_pad]) =
    slice(FHT_M(FHT_N(w)) s_u s_v^T).  Pads are ``len(s_u)``, ``len(s_v)``.
    """
    L.require_cuda(w)
    assert w.dim() == 2, "weight must be 2-D"
    w = w.contiguous()
    Mp, Np = int(s_u.numel()), int(s_v.numel())
    su = _sign(s_u, Mp, w.device)
    sv = _sign(s_v, Np, w.device)
    lib = L.load()
    if not inverse:
        M, N = w.shape
        out = torch.empty((Mp, Np), dtype=torch.float32, device=w.device)
        ws, nws = None, 0
    else:
        assert tuple(w.shape) == (Mp, Np), f"inverse rotation takes a [{Mp}, {Np}] matrix, got {tuple(w.shape)}"
        M, N = shape if shape is not None else (Mp, Np)
        out = torch.empty((M, N), dtype=torch.float32, device=w.device)
        ws = torch.empty((Mp, Np), dtype=torch.float32, device=w.device)
        nws = ws.numel() * 4
    L.check(lib.qi8_weight_rotate2d(L.ptr(w), L.dtype_code(w.dtype), M, N, Mp, Np, L.ptr(su), L.ptr(sv),
                                    int(bool(inverse)), L.ptr(out), L.ptr(ws), nws, L.stream_ptr(w.device)),
            "qi8_weight_rotate2d")
    return out


def allgather_cols(y_local: torch.Tensor, nccl_comm: int, world: int,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """All-gather of column shards ``[T, n_loc]`` into ``[T, world * n_loc]``
    over a caller-created NCCL communicator (``ncclComm_t`` as an integer)."""
    L.require_cuda(y_local)
    y_local = y_local.contiguous()
    T, n_loc = y_local.shape
    if out is None:
        out = torch.empty((T, world * n_loc), dtype=y_local.dtype, device=y_local.device)
    scratch = torch.empty((world, T, n_loc), dtype=y_local.dtype, device=y_local.device)
    lib = L.load()
    L.check(lib.qi8_allgather_cols(L.ptr(y_local), L.dtype_code(y_local.dtype), T, n_loc, L.ptr(out), out.stride(0),
                                   ctypes.c_void_p(nccl_comm), L.ptr(scratch), scratch.numel() * scratch.element_size(),
                                   L.stream_ptr(y_local.device)), "qi8_allgather_cols")
    return out


def gather_layout(gathered: torch.Tensor, world: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[world, T, n_loc]`` (or ``[world * T, n_loc]``) all-gather result ->
    ``[T, world * n_loc]``; ``out`` may be a row-strided view."""
    L.require_cuda(gathered)
    assert gathered.is_contiguous(), "gathered must be contiguous"
    n_loc = gathered.shape[-1]
    T = gathered.numel() // (world * n_loc)
    if out is None:
        out = torch.empty((T, world * n_loc), dtype=gathered.dtype, device=gathered.device)
    assert out.shape == (T, world * n_loc) and out.stride(1) == 1, "out must be [T, world * n_loc] row-major"
    L.check(L.load().qi8_gather_layout(L.ptr(gathered), L.dtype_code(gathered.dtype), world, T, n_loc, L.ptr(out),
                                       out.stride(0), L.stream_ptr(gathered.device)), "qi8_gather_layout")
    return out


def requant_weight(w: torch.Tensor, requant: int = L.QI8_REQ_ROW, block: int = 128):
    """QuIP requant rule without rotation (converters/quip_int8.py:1614-1669)."""
    L.require_cuda(w)
    assert w.dim() == 2 and w.stride(1) == 1, "weight must be a row-major 2-D tensor"
    M, N = w.shape
    q = torch.empty((M, N), dtype=torch.int8, device=w.device)
    if requant == L.QI8_REQ_BLOCK and N % block == 0:
        s = torch.empty((M, N // block, 1), dtype=torch.float32, device=w.device)
    elif requant == L.QI8_REQ_GLOBAL:
        s = torch.empty((), dtype=torch.float32, device=w.device)
    else:
        s = torch.empty((M, 1), dtype=torch.float32, device=w.device)
    ws = torch.empty(64, dtype=torch.uint8, device=w.device)
    lib = L.load()
    L.check(lib.qi8_requant_weight(L.ptr(w), L.dtype_code(w.dtype), M, N, w.stride(0), requant, block, L.ptr(q),
                                   L.ptr(s), L.ptr(ws), ws.numel(), L.stream_ptr(w.device)), "qi8_requant_weight")
    return q, s


# ---------------------------------------------------------------------------
# QuIP with the reference's defaults (diagonal rescaling, random permutation,
# damping, act-order, fp64 Hessian factorization, blocked LDLQ)
# ---------------------------------------------------------------------------

def col_sumsq(w: torch.Tensor) -> torch.Tensor:
    """``(W ** 2).sum(dim=0)`` in fp32, summed in torch's CPU order
    (converters/quip_int8.py:266)."""
    L.require_cuda(w)
    assert w.dim() == 2 and w.stride(1) == 1, "weight must be a row-major 2-D tensor"
    M, N = w.shape
    out = torch.empty(N, dtype=torch.float32, device=w.device)
    L.check(L.load().qi8_col_sumsq(L.ptr(w), L.dtype_code(w.dtype), M, N, w.stride(0), L.ptr(out),
                                   L.stream_ptr(w.device)), "qi8_col_sumsq")
    return out


def scale2d(x: Optional[torch.Tensor], shape: tuple, row: Optional[torch.Tensor] = None,
            col: Optional[torch.Tensor] = None, divide: bool = False, device=None) -> torch.Tensor:
    """``(x * col[None, :]) * row[:, None]`` or ``x / col[None, :]`` in fp32
    (converters/quip_int8.py:280-285, 303); ``x=None`` is the identity."""
    dev = x.device if x is not None else device
    if x is not None:
        L.require_cuda(x)
        assert x.stride(1) == 1, "x must be row-major"
    M, N = shape
    out = torch.empty((M, N), dtype=torch.float32, device=dev)
    L.check(L.load().qi8_scale2d(L.ptr(x), L.dtype_code(x.dtype) if x is not None else 0, M, N,
                                 x.stride(0) if x is not None else N, L.ptr(row), L.ptr(col), int(bool(divide)),
                                 L.ptr(out), N, L.stream_ptr(dev)), "qi8_scale2d")
    return out


def ldlq_prepare(w_rot: torch.Tensor, h_rot: torch.Tensor, cols: torch.Tensor, dead: torch.Tensor,
                 diag: torch.Tensor):
    """Gather W' and H' into LDLQ column order ``cols`` (dead columns zeroed,
    damped diagonal ``diag``), the per-row scale, and the Hessian reversed
    for the factorization.  Returns ``(W_p fp32 [M, N], scale [M, 1], H_rev fp64 [N, N])``."""
    M, N = w_rot.shape
    dev = w_rot.device
    wp = torch.empty((M, N), dtype=torch.float32, device=dev)
    sc = torch.empty((M, 1), dtype=torch.float32, device=dev)
    hrev = torch.empty((N, N), dtype=torch.float64, device=dev)
    L.check(L.load().qi8_ldlq_prepare(L.ptr(w_rot), L.ptr(h_rot), M, N, L.ptr(cols), L.ptr(dead), L.ptr(diag),
                                      L.ptr(wp), L.ptr(sc), L.ptr(hrev), L.stream_ptr(dev)), "qi8_ldlq_prepare")
    return wp, sc, hrev


def hinv_upper(h_rev: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Upper Cholesky factor of H^-1 from the reversed damped Hessian (fp64,
    overwritten); returns ``(U fp32 [N, N], info int32 device scalar)`` --
    info != 0 marks a non-positive pivot (the reference then uses the
    identity, converters/quip_int8.py:1211-1216)."""
    N = h_rev.shape[0]
    dev = h_rev.device
    lib = L.load()
    hinv = torch.empty((N, N), dtype=torch.float32, device=dev)
    info = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = torch.empty(int(lib.qi8_hinv_workspace_bytes(N)), dtype=torch.uint8, device=dev)
    L.check(lib.qi8_hinv_upper(L.ptr(h_rev), N, L.ptr(hinv), L.ptr(info), L.ptr(ws), ws.numel(),
                               L.stream_ptr(dev)), "qi8_hinv_upper")
    return hinv, info


def eye_f32(n: int, device) -> torch.Tensor:
    out = torch.empty((n, n), dtype=torch.float32, device=device)
    L.check(L.load().qi8_eye_f32(L.ptr(out), n, L.stream_ptr(device)), "qi8_eye_f32")
    return out


def ldlq(w: torch.Tensor, hinv: torch.Tensor, scale: torch.Tensor, block: int = 128) -> torch.Tensor:
    """The LDLQ pass (converters/quip_int8.py:813-945); ``w`` fp32 [M, N] is
    consumed (updated in place).  Returns ``Q'`` int8 [M, N]."""
    M, N = w.shape
    dev = w.device
    lib = L.load()
    q = torch.empty((M, N), dtype=torch.int8, device=dev)
    ws = torch.empty(int(lib.qi8_ldlq_workspace_bytes(M, N, block)), dtype=torch.uint8, device=dev)
    L.check(lib.qi8_ldlq(L.ptr(w), M, N, L.ptr(hinv), L.ptr(scale), block, L.ptr(q), L.ptr(ws), ws.numel(),
                         L.stream_ptr(dev)), "qi8_ldlq")
    return q


def ldlq_finish(q: torch.Tensor, scale: torch.Tensor, cols: torch.Tensor, want_deq: bool = True,
                want_q: bool = False):
    """Scatter LDLQ columns back to rotated order: ``(deq fp32 or None, q int8 or None)``."""
    M, N = q.shape
    dev = q.device
    deq = torch.empty((M, N), dtype=torch.float32, device=dev) if want_deq else None
    qs = torch.empty((M, N), dtype=torch.int8, device=dev) if want_q else None
    L.check(L.load().qi8_ldlq_finish(L.ptr(q), M, N, L.ptr(scale), L.ptr(cols), L.ptr(deq), L.ptr(qs),
                                     L.stream_ptr(dev)), "qi8_ldlq_finish")
    return deq, qs


# ---------------------------------------------------------------------------
# weights of 4 bits with group scales (format: include/qi8.h)
# ---------------------------------------------------------------------------

_I4_GROUPS = (32, 64, 128)


def _i4_padded(k: int) -> int:
    """Features per row of a 4-bit weight: ``k`` rounded up to whole 128s."""
    return -(-k // 128) * 128


def _one_device(x: torch.Tensor, *tensors: Optional[torch.Tensor]) -> torch.device:
    dev = x.device
    for t in (x, *tensors):
        if t is not None and (not t.is_cuda or t.device != dev):
            L.require_cuda(x, *tensors)
            raise AssertionError(f"tensors on {dev} and {t.device}")
    return dev


def _fast(name: str, *args):
    """The shortcut's result for arguments that need no conversion; ``None`` for all others, errors among them."""
    fast = L.fast_call() if L._call is None else L._call
    return getattr(fast, name)(*args) if fast else None


# the current stream of a device as a plain pointer: a tenth of the cost of a Stream object
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(dev: torch.device, what: str, fn, *args) -> None:
    """Calls a libqi8 entry point on ``dev`` and its current stream."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(index))
    if rc:
        L.check(rc, what)


def _check_i4(q: torch.Tensor, scale: torch.Tensor, k: int, group: int, dims: int) -> None:
    """``q`` uint8 [..., N, Kp/2] and ``scale`` bf16 [..., N, Kp/group] of a weight with ``k`` input features."""
    if q.dtype != torch.uint8 or scale.dtype != torch.bfloat16:
        raise TypeError(f"4-bit weights are uint8 codes and bfloat16 scales, got {q.dtype} and {scale.dtype}")
    assert group in _I4_GROUPS, f"group_size must be 32, 64 or 128, got {group}"
    assert k > 0, f"a weight of {k} features"
    kp = _i4_padded(k)
    shape = q.shape
    assert len(shape) == dims and shape[-1] * 2 == kp, \
        f"4-bit codes of shape {tuple(shape)}: expected {dims} dimensions and {kp // 2} bytes a row for {k} features"
    assert scale.shape == (*shape[:-1], kp // group), \
        f"scales of shape {tuple(scale.shape)} for codes of shape {tuple(shape)} and group_size {group}"
    assert q.is_contiguous() and scale.is_contiguous(), "4-bit codes and scales must be contiguous"


def _no_grad(*tensors: Optional[torch.Tensor], what: str = "4-bit operators") -> None:
    """Inference only: a result without a gradient (or a tangent of forward mode, which no_grad does not turn off) must
    not pass for one with it."""
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and ((grad and t.requires_grad) or forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"{what} have no backward pass and no forward mode: call them on detached "
                               "tensors, or under torch.no_grad() if no input has a tangent")


def quant_weight_i4(w: torch.Tensor, group: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """4-bit codes and group scales of ``w`` [..., N, K] (a parameter is read as it is, like the int8 quantizers do):
    ``(q uint8 [..., N, Kp/2], scale bf16 [..., N, Kp/group])``."""
    pair = _fast("quant_weight_i4", w, group)
    if pair is not None:
        return pair
    dev = _one_device(w)
    dt = L.dtype_code(w.dtype)
    if dt not in (L.QI8_BF16, L.QI8_F16, L.QI8_F32):
        raise TypeError(f"weights must be bfloat16, float16 or float32, got {w.dtype}")
    assert w.dim() >= 2 and w.shape[-1] > 0, f"weight of shape {tuple(w.shape)}: expected [..., N, K] with K > 0"
    assert group in _I4_GROUPS, f"group_size must be 32, 64 or 128, got {group}"
    w2 = w if w.dim() == 2 else w.reshape(-1, w.shape[-1])
    if w2.stride(1) != 1 or w2.stride(0) < w2.shape[1]:
        w2 = w2.contiguous()
    rows, k = w2.shape
    kp = _i4_padded(k)
    q = torch.empty(*w.shape[:-1], kp // 2, dtype=torch.uint8, device=dev)
    s = torch.empty(*w.shape[:-1], kp // group, dtype=torch.bfloat16, device=dev)
    _launch(dev, "qi8_quant_weight_i4", L.load().qi8_quant_weight_i4, w2.data_ptr(), dt, rows, k,
            max(w2.stride(0), k), group, q.data_ptr(), s.data_ptr())
    return q, s


def dequant_i4(q: torch.Tensor, scale: torch.Tensor, k: int, group: int = 128,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The weight [..., N, k] that 4-bit codes and scales stand for."""
    out = _fast("dequant_i4", q, scale, k, group, out_dtype)
    if out is not None:
        return out
    dev = _one_device(q, scale)
    _no_grad(scale)
    _check_i4(q, scale, k, group, q.dim())
    assert q.dim() >= 2, f"4-bit codes of shape {tuple(q.shape)}: expected [..., N, Kp/2]"
    dt = L.dtype_code(out_dtype)
    if dt not in (L.QI8_BF16, L.QI8_F16, L.QI8_F32):
        raise TypeError(f"output dtype must be bfloat16, float16 or float32, got {out_dtype}")
    out = torch.empty(*q.shape[:-1], k, dtype=out_dtype, device=dev)
    _launch(dev, "qi8_dequant_i4", L.load().qi8_dequant_i4, q.data_ptr(), scale.data_ptr(), out.numel() // k, k,
            group, out.data_ptr(), dt, k)
    return out


def gemm_w4(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, group: int = 128,
            bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x [..., K] W^T + bias`` with the 4-bit weight ``q`` [N, Kp/2], ``scale`` [N, Kp/group]."""
    if out_dtype is None:
        out = _fast("gemm_w4", x, q, scale, group, bias)
        if out is not None:
            return out
    dev = _one_device(x, q, scale, bias)
    _no_grad(x, scale, bias)
    shape = x.shape
    k = shape[-1]
    _check_i4(q, scale, k, group, 2)
    n = q.shape[0]
    x2 = x if len(shape) == 2 else x.reshape(-1, k)
    m = x2.shape[0]
    ld, inner = x2.stride()
    if inner != 1 or ld < k:
        if m > 1 or inner != 1:
            x2 = x2.contiguous()
        ld = k
    bias_ptr, bias_dt = None, 0
    if bias is not None:
        assert bias.dim() == 1 and bias.shape[0] == n, f"Bias must be 1D with length {n}, got shape {tuple(bias.shape)}"
        bias = bias.contiguous()
        bias_ptr, bias_dt = bias.data_ptr(), L.dtype_code(bias.dtype)
    out = torch.empty(m, n, dtype=out_dtype or x.dtype, device=dev)
    lib = L.load()
    x_ptr, ws_ptr, nbytes = x2.data_ptr(), None, 0
    if k & 7 or ld & 7 or x_ptr & 15:
        nbytes = lib.qi8_gemm_w4_workspace_bytes(x_ptr, m, k, ld)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ws_ptr = ws.data_ptr()
    _launch(dev, "qi8_gemm_w4", lib.qi8_gemm_w4, x_ptr, L.dtype_code(x.dtype), m, k, ld, q.data_ptr(),
            scale.data_ptr(), n, group, bias_ptr, bias_dt, out.data_ptr(), L.dtype_code(out.dtype), n, ws_ptr, nbytes)
    return out if len(shape) == 2 else out.view(*shape[:-1], n)


def moe_w4(x: torch.Tensor, router: torch.Tensor, q13: torch.Tensor, s13: torch.Tensor, q2: torch.Tensor,
           s2: torch.Tensor, top_k: int, group: int = 128, renormalize: bool = True,
           act: int = L.QI8_ACT_SILU) -> torch.Tensor:
    """A mixture-of-experts layer on ``x`` [..., H] with 4-bit experts: ``router`` [E, H], ``q13``/``s13`` of
    [E, 2 I, H] (gate rows above up rows), ``q2``/``s2`` of [E, H, I]."""
    out = _fast("moe_w4", x, router, q13, s13, q2, s2, top_k, group, bool(renormalize), act)
    if out is not None:
        return out
    dev = _one_device(x, router, q13, s13, q2, s2)
    _no_grad(x, router, s13, s2)
    h = x.shape[-1]
    _check_i4(q13, s13, h, group, 3)
    e, i2 = q13.shape[:2]
    assert i2 % 2 == 0, f"gate and up weights of {i2} rows: expected as many of each"
    i = i2 // 2
    _check_i4(q2, s2, i, group, 3)
    assert tuple(q2.shape[:2]) == (e, h), f"down weights of shape {tuple(q2.shape)}: expected [{e}, {h}, ...]"
    assert tuple(router.shape) == (e, h), f"router of shape {tuple(router.shape)}: expected [{e}, {h}]"
    assert router.is_contiguous(), "router must be contiguous"
    # before they become C integers, which would take their lowest bits
    assert 0 < top_k <= e, f"top_k {top_k}: 1 to the {e} experts"
    assert act in (L.QI8_ACT_SILU, L.QI8_ACT_GELU), f"activation must be SiLU or GELU, got code {act}"
    x2 = x if x.dim() == 2 else x.reshape(-1, h)
    if x2.stride(1) != 1 or x2.stride(0) < h:
        x2 = x2.contiguous()
    t = x2.shape[0]
    lib = L.load()
    nbytes = lib.qi8_moe_w4_workspace_bytes(t, h, e, i, top_k)
    if nbytes == 0:
        L.check(L.QI8_ESHAPE, "qi8_moe_w4")
    out = torch.empty(t, h, dtype=x.dtype, device=dev)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(dev, "qi8_moe_w4", lib.qi8_moe_w4, x2.data_ptr(), L.dtype_code(x.dtype), t, h, max(x2.stride(0), h),
            router.data_ptr(), L.dtype_code(router.dtype), e, q13.data_ptr(), s13.data_ptr(), i, q2.data_ptr(),
            s2.data_ptr(), group, top_k, int(bool(renormalize)), act, out.data_ptr(), h, ws.data_ptr(), nbytes)
    return out if x.dim() == 2 else out.view(x.shape)


# ---------------------------------------------------------------------------
# fp8 with block scales, and the producers of quantized activations (formats:
# include/qi8.h)
# ---------------------------------------------------------------------------

_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_FLOATS = (L.QI8_BF16, L.QI8_F16, L.QI8_F32)


def _f8_blocks(n: int) -> int:
    """Blocks of 128 columns (or rows) that ``n`` of them make."""
    return -(-n // 128)


def _refuse_grad(*tensors: Optional[torch.Tensor]) -> None:
    _no_grad(*tensors, what="fp8 and fused quantization operators")


def _float_code(dt: torch.dtype, what: str) -> int:
    code = L._DTYPE.get(dt)
    if code not in _FLOATS:
        raise TypeError(f"{what} must be bfloat16, float16 or float32, got {dt}")
    return code


def _strided_rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """``x`` as rows with unit column stride, and their stride."""
    n = x.shape[-1]
    x = x.resolve_neg()
    x2 = x if x.dim() == 2 else x.reshape(-1, n)
    if x2.shape[0] == 1 and (n <= 1 or x2.stride(1) == 1):
        return x2, max(n, 1)
    if (x2.stride(1) != 1 and n > 1) or x2.stride(0) < n:
        x2 = x2.contiguous()
    return x2, max(x2.stride(0), n, 1)


def _new_codes(shape: tuple, dtype: torch.dtype, device) -> torch.Tensor:
    """Room for codes of one byte whose rows start on 16-byte boundaries: the last dimension's rows are padded in
    memory where they are no multiple of 16 long (a view, then)."""
    n = shape[-1]
    pitch = -(-n // 16) * 16
    if pitch == n:
        return torch.empty(shape, dtype=dtype, device=device)
    return torch.empty((*shape[:-1], pitch), dtype=dtype, device=device)[..., :n]


def _code_rows(q: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """Codes as rows [-1, n] and their stride; a layout that has no single row stride is copied."""
    if q.dim() != 2:
        q = q.reshape(-1, q.shape[-1])
    return _strided_rows(q)


def aligned_codes(q: torch.Tensor) -> torch.Tensor:
    """``q`` [..., K] with rows that start on 16-byte boundaries, as the quantizers return them: itself, or a copy."""
    steps = (step for size, step in zip(q.shape[:-1], q.stride()) if size != 1)
    if q.numel() == 0 or ((q.shape[-1] == 1 or q.stride(-1) == 1) and q.storage_offset() % 16 == 0
                          and all(step % 16 == 0 for step in steps)):
        return q
    return _new_codes(q.shape, q.dtype, q.device).copy_(q)


def _check_f8(q: torch.Tensor, scale: torch.Tensor, tile: int) -> None:
    """``q`` e4m3 [..., n] with a scale per row and 128 columns, or [N, K] with 128 x 128 tiles."""
    if q.dtype != _F8 or scale.dtype != _E8:
        raise TypeError(f"fp8 operands are float8_e4m3fn codes and float8_e8m0fnu scales, got {q.dtype} and {scale.dtype}")
    assert q.dim() >= 1 and (tile == 1 or q.dim() == 2), f"fp8 codes of shape {tuple(q.shape)}"
    lead = q.shape[:-1] if tile == 1 else (_f8_blocks(q.shape[0]),)
    want = (*lead, _f8_blocks(q.shape[-1]))
    assert tuple(scale.shape) == want, f"scales of shape {tuple(scale.shape)} for codes of shape {tuple(q.shape)}: " \
                                       f"expected {want}"
    assert scale.is_contiguous(), "fp8 scales must be contiguous"


def quant_rows_f8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp8 codes ``[..., n]`` of ``x`` and one scale for each row and 128 columns ``[..., ceil(n / 128)]``."""
    pair = _fast("quant_rows_f8", x)
    if pair is not None:
        return pair
    dev = _one_device(x)
    dt = _float_code(x.dtype, "activations")
    _refuse_grad(x)
    assert x.dim() >= 1, "activations need a last dimension"
    n = x.shape[-1]
    q = _new_codes(x.shape, _F8, dev)
    s = torch.empty(*x.shape[:-1], _f8_blocks(n), dtype=_E8, device=dev)
    if q.numel():
        x2, ld = _strided_rows(x)
        _launch(dev, "qi8_quant_rows_f8", L.load().qi8_quant_rows_f8, x2.data_ptr(), dt, x2.shape[0], n, ld,
                q.data_ptr(), -(-n // 16) * 16, s.data_ptr())
    return q, s


def quant_weight_f8(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp8 codes of ``w`` [N, K] (a parameter is read as it is) and one scale for each 128 x 128 tile."""
    pair = _fast("quant_weight_f8", w)
    if pair is not None:
        return pair
    dev = _one_device(w)
    with torch.no_grad():  # a parameter's gradient may be lost, a tangent not
        _refuse_grad(w)
    dt = _float_code(w.dtype, "weights")
    assert w.dim() == 2, f"weight of shape {tuple(w.shape)}: expected [N, K]"
    n, k = w.shape
    q = _new_codes(w.shape, _F8, dev)
    s = torch.empty(_f8_blocks(n), _f8_blocks(k), dtype=_E8, device=dev)
    if q.numel():
        w2, ld = _strided_rows(w.detach())
        _launch(dev, "qi8_quant_weight_f8", L.load().qi8_quant_weight_f8, w2.data_ptr(), dt, n, k, ld, q.data_ptr(),
                -(-k // 16) * 16, s.data_ptr())
    return q, s


def dequant_f8(q: torch.Tensor, scale: torch.Tensor, tile: int, out_dtype: torch.dtype) -> torch.Tensor:
    """The values that fp8 codes stand for: ``tile`` 1 for activations' scales, 128 for a weight's."""
    dev = _one_device(q, scale)
    _refuse_grad(q, scale)
    _check_f8(q, scale, tile)
    dt = _float_code(out_dtype, "output dtype")
    out = torch.empty(q.shape, dtype=out_dtype, device=dev)
    if out.numel():
        q2, ld = _code_rows(q)
        n = q.shape[-1]
        _launch(dev, "qi8_dequant_f8", L.load().qi8_dequant_f8, q2.data_ptr(), q2.shape[0], n, ld, scale.data_ptr(), tile,
                out.data_ptr(), dt, n)
    return out


def _f8_bias(bias: Optional[torch.Tensor], n: int) -> Tuple[Optional[torch.Tensor], Optional[int], int]:
    if bias is None:
        return None, None, 0
    assert bias.dim() == 1 and bias.shape[0] == n, f"Bias must be 1D with length {n}, got shape {tuple(bias.shape)}"
    bias = bias.resolve_neg().contiguous()
    return bias, bias.data_ptr(), _float_code(bias.dtype, "bias")


def _no_columns(shape: tuple, n: int, bias: Optional[torch.Tensor], dtype: torch.dtype, dev) -> torch.Tensor:
    """The product over no columns at all: the bias."""
    out = torch.zeros(*shape, n, dtype=dtype, device=dev)
    return out if bias is None else out.copy_(bias)


def gemm_f8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
            bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a [..., K] b [N, K]^T + bias`` of fp8 operands."""
    out = _fast("gemm_f8", a, a_scale, b, b_scale, bias, out_dtype)
    if out is not None:
        return out
    dev = _one_device(a, a_scale, b, b_scale, bias)
    _refuse_grad(a, a_scale, b, b_scale, bias)
    _check_f8(a, a_scale, 1)
    _check_f8(b, b_scale, 128)
    n, k = b.shape
    assert a.shape[-1] == k, f"Shape mismatch: b.shape={tuple(b.shape)}, expected [N, {a.shape[-1]}]"
    dt = _float_code(out_dtype, "output dtype")
    bias, bias_ptr, bias_dt = _f8_bias(bias, n)
    if k == 0:
        return _no_columns(a.shape[:-1], n, bias, out_dtype, dev)
    out = torch.empty(*a.shape[:-1], n, dtype=out_dtype, device=dev)
    if out.numel() == 0:
        return out
    a2, ld_a = _code_rows(a)
    b2, ld_b = _strided_rows(b)
    m = a2.shape[0]
    lib = L.load()
    nbytes = lib.qi8_gemm_f8_workspace_bytes(a2.data_ptr(), m, k, ld_a, b2.data_ptr(), n, ld_b)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch(dev, "qi8_gemm_f8", lib.qi8_gemm_f8, a2.data_ptr(), a_scale.data_ptr(), m, k, ld_a, b2.data_ptr(),
            b_scale.data_ptr(), n, ld_b, bias_ptr, bias_dt, out.data_ptr(), dt, n, ws.data_ptr() if nbytes else None, nbytes)
    return out


def linear_f8(x: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
              bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``quantized(x) b^T + bias`` in x's dtype: ``quant_rows_f8`` and ``gemm_f8``."""
    out = _fast("linear_f8", x, b, b_scale, bias)
    if out is not None:
        return out
    dev = _one_device(x, b, b_scale, bias)
    _refuse_grad(x, b, b_scale, bias)
    _check_f8(b, b_scale, 128)
    n, k = b.shape
    dt = _float_code(x.dtype, "activations")
    assert x.dim() >= 1 and x.shape[-1] == k, f"input of shape {tuple(x.shape)}, weight expects {k} features"
    bias, bias_ptr, bias_dt = _f8_bias(bias, n)
    if k == 0:
        return _no_columns(x.shape[:-1], n, bias, x.dtype, dev)
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=dev)
    if out.numel() == 0:
        return out
    x2, ld = _strided_rows(x)
    b2, ld_b = _strided_rows(b)
    m = x2.shape[0]
    lib = L.load()
    nbytes = lib.qi8_linear_f8_workspace_bytes(m, k, b2.data_ptr(), n, ld_b)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch(dev, "qi8_linear_f8", lib.qi8_linear_f8, x2.data_ptr(), dt, m, k, ld, b2.data_ptr(), b_scale.data_ptr(), n,
            ld_b, bias_ptr, bias_dt, out.data_ptr(), dt, n, ws.data_ptr() if nbytes else None, nbytes)
    return out


def _quantized_out(shape: tuple, mode: int, dev) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales that a producer fills."""
    n = shape[-1]
    if mode == L.QI8_Q_FP8:
        return _new_codes(shape, _F8, dev), torch.empty(*shape[:-1], _f8_blocks(n), dtype=_E8, device=dev)
    # int8 rows are contiguous: the int8 products take them so
    assert mode == L.QI8_Q_TOKEN or n % 128 == 0, \
        f"Last dimension size must be divisible by block_size (block_size=128), got {n}"
    s = torch.empty(*shape[:-1], 1 if mode == L.QI8_Q_TOKEN else n // 128, dtype=torch.float32, device=dev)
    if n == 0:
        s.fill_(1e-30)  # rows of no columns: the least scale, and no kernel to write it
    return torch.empty(shape, dtype=torch.int8, device=dev), s


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   residual: Optional[torch.Tensor] = None, mode: int = L.QI8_Q_FP8):
    """The root-mean-square norm of ``h = x + residual`` over the last dimension, times ``weight``, quantized:
    ``(q, scale)``, and ``h`` in x's dtype as a third result where there is a residual."""
    got = _fast("rms_norm_quant", x, weight, eps, residual, mode)
    if got is not None:
        return got
    dev = _one_device(x, weight, residual)
    _refuse_grad(x, weight, residual)
    dt = _float_code(x.dtype, "activations")
    assert x.dim() >= 1, "activations need a last dimension"
    n = x.shape[-1]
    w_ptr, w_dt = None, 0
    if weight is not None:
        assert weight.dim() == 1 and weight.shape[0] == n, f"weight of shape {tuple(weight.shape)}: expected [{n}]"
        weight = weight.resolve_neg().contiguous()
        w_ptr, w_dt = weight.data_ptr(), _float_code(weight.dtype, "weight")
    if residual is not None:
        assert residual.shape == x.shape, f"residual of shape {tuple(residual.shape)} for {tuple(x.shape)}"
        if residual.dtype != x.dtype:
            raise TypeError(f"residual of {residual.dtype} for activations of {x.dtype}")
    assert eps == 0.0 or 1e-37 <= eps < 1e30, f"eps {eps}: 0, or from 1e-37 to 1e30"
    q, s = _quantized_out(x.shape, mode, dev)
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if residual is not None else None
    if q.numel():
        x2, ld = _strided_rows(x)
        r_ptr, ld_r, h_ptr = None, 0, None
        if residual is not None:
            r2, ld_r = _strided_rows(residual)
            r_ptr, h_ptr = r2.data_ptr(), h.data_ptr()
        _launch(dev, "qi8_rms_norm_quant", L.load().qi8_rms_norm_quant, x2.data_ptr(), dt, x2.shape[0], n, ld, r_ptr,
                ld_r, w_ptr, w_dt, eps, mode, q.data_ptr(), -(-n // 16) * 16 if mode == L.QI8_Q_FP8 else n, s.data_ptr(),
                h_ptr, n)
    return (q, s) if residual is None else (q, s, h)


def gated_quant(gate: torch.Tensor, up: torch.Tensor, act: int = L.QI8_ACT_SILU,
                mode: int = L.QI8_Q_FP8) -> Tuple[torch.Tensor, torch.Tensor]:
    """``act(gate) * up``, quantized: ``(q, scale)``."""
    pair = _fast("gated_quant", gate, up, act, mode)
    if pair is not None:
        return pair
    dev = _one_device(gate, up)
    _refuse_grad(gate, up)
    dt = _float_code(gate.dtype, "activations")
    if up.dtype != gate.dtype:
        raise TypeError(f"gate of {gate.dtype} and up of {up.dtype}")
    assert gate.dim() >= 1 and gate.shape == up.shape, f"gate of shape {tuple(gate.shape)}, up of {tuple(up.shape)}"
    n = gate.shape[-1]
    q, s = _quantized_out(gate.shape, mode, dev)
    if q.numel():
        g2, ld_g = _strided_rows(gate)
        u2, ld_u = _strided_rows(up)
        _launch(dev, "qi8_gated_quant", L.load().qi8_gated_quant, g2.data_ptr(), ld_g, u2.data_ptr(), ld_u, dt,
                g2.shape[0], n, act, mode, q.data_ptr(), -(-n // 16) * 16 if mode == L.QI8_Q_FP8 else n, s.data_ptr())
    return q, s


def device_status(reset: bool = True) -> None:
    """Raise if a kernel's bounded wait expired since the last check."""
    L.check(L.load().qi8_device_status(int(reset)), "device status")
