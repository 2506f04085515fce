"""Torch-tensor wrappers over the C ABI (device memory, streams and shapes only).

Every function here launches kernels from libtesm_b200.so on the current torch
stream; none computes anything with torch ops.  Tensors must live on the CUDA
device; ownership stays with torch.
"""
from __future__ import annotations

import ctypes
import os
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Sequence

import torch

from . import _lib

F32, BF16 = 0, 1
LAYOUT_ROWMAJOR, LAYOUT_GEMV = 0, 1
GEMV_MAX_M = 64

_DT = {torch.float32: F32, torch.bfloat16: BF16}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DT[dt]
    except KeyError:
        raise _lib.TesmError(f"tesm_b200: unsupported dtype {dt} (float32 or bfloat16)") from None


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def round_up(x: int, m: int) -> int:
    return (x + m - 1) // m * m


@dataclass
class PackedWeight:
    """Device-resident ternary weight of one BitLinear.

    packed: (N, Kp/4) uint8 in the reference INT2 byte format, Kp = K rounded up to 256
    tern:   (N, Kp) int8 ternary values for the tensor-core path (None until needed)
    scale:  (1,) or (N,) float32 quantisation scale 1/mean|W|
    deq:    (1,) or (N,) float32 dequantisation factor fl(1/scale)
    """
    packed: torch.Tensor
    tern: Optional[torch.Tensor]
    scale: torch.Tensor
    deq: torch.Tensor
    N: int
    K: int
    per_row: bool


def weight_scale(w: torch.Tensor, eps: float, per_row: bool = False, scale_out=None, deq_out=None):
    N, K = w.shape
    n = N if per_row else 1
    scale = scale_out if scale_out is not None else torch.empty(n, device=w.device, dtype=torch.float32)
    deq = deq_out if deq_out is not None else torch.empty(n, device=w.device, dtype=torch.float32)
    work = torch.empty(N, device=w.device, dtype=torch.float64)
    _lib.call("tesm_b200_weight_scale", w.data_ptr(), dtype_code(w.dtype), N, K, w.stride(0), int(per_row),
              float(eps), scale.data_ptr(), deq.data_ptr(), work.data_ptr(), _stream())
    return scale, deq


def pack_weight(w: torch.Tensor, eps: float = 1e-5, per_row: bool = False, with_tern: bool = True,
                scale: Optional[torch.Tensor] = None) -> PackedWeight:
    """Ternarise and pack a (N, K) weight; ``scale`` overrides the computed 1/mean|W|."""
    assert w.is_cuda and w.dim() == 2 and w.stride(1) == 1
    N, K = w.shape
    Kp = round_up(K, 256)
    if scale is None:
        scale, deq = weight_scale(w, eps, per_row)
    else:
        scale = scale.to(device=w.device, dtype=torch.float32).reshape(-1).contiguous()
        deq = torch.reciprocal(scale)  # not used on the parity path
    packed = torch.empty(N, Kp // 4, device=w.device, dtype=torch.uint8)
    tern = torch.empty(N, Kp, device=w.device, dtype=torch.int8) if with_tern else None
    _lib.call("tesm_b200_pack_ternary", w.data_ptr(), dtype_code(w.dtype), N, K, w.stride(0), int(per_row),
              scale.data_ptr(), packed.data_ptr(), packed.stride(0), _ptr(tern), Kp if tern is not None else 0,
              _stream())
    return PackedWeight(packed, tern, scale, deq, N, K, per_row)


def packed_from_int2(packed: torch.Tensor, weight_scale, K: int, device) -> PackedWeight:
    """PackedWeight from an exported INT2 weight (pack_int2_to_uint8 bytes, (N, ceil(K/4)) uint8,
    and its weight_scale = 1 / mean|W|; int2_quantization.py:21-60): the bytes are kept as they
    are (rows padded with code 1 up to K rounded to 256) and the int8 ternary operand of the
    tensor-core GEMM is unpacked from them on the device."""
    N, kb = packed.shape
    if packed.dtype != torch.uint8 or kb != (K + 3) // 4:
        raise ValueError(f"packed INT2 weight must be uint8 (N, ceil(K/4)) = (N, {(K + 3) // 4}), got "
                         f"{tuple(packed.shape)} {packed.dtype}")
    Kp = round_up(K, 256)
    dev = torch.device(device)
    buf = torch.full((N, Kp // 4), 0x55, device=dev, dtype=torch.uint8)
    buf[:, :kb] = packed.to(dev)
    scale = torch.as_tensor(weight_scale, dtype=torch.float32).reshape(1).to(dev)
    deq = torch.reciprocal(scale)
    tern = torch.empty(N, Kp, device=dev, dtype=torch.int8)
    _lib.call("tesm_b200_unpack_ternary", buf.data_ptr(), buf.stride(0), N, Kp, tern.data_ptr(), tern.stride(0),
              _stream())
    return PackedWeight(buf, tern, scale, deq, N, K, False)


def ensure_tern(pw: PackedWeight, w: torch.Tensor):
    if pw.tern is None:
        Kp = round_up(pw.K, 256)
        tern = torch.empty(pw.N, Kp, device=w.device, dtype=torch.int8)
        scratch = torch.empty_like(pw.packed)
        _lib.call("tesm_b200_pack_ternary", w.data_ptr(), dtype_code(w.dtype), pw.N, pw.K, w.stride(0),
                  int(pw.per_row), pw.scale.data_ptr(), scratch.data_ptr(), scratch.stride(0), tern.data_ptr(), Kp,
                  _stream())
        pw.tern = tern
    return pw.tern


def quant_act(x2d: torch.Tensor, eps: float, layout: int):
    """Per-row int8 codes of a (M, K) activation (row stride may exceed K)."""
    assert x2d.is_cuda and x2d.dim() == 2 and x2d.stride(1) == 1
    M, K = x2d.shape
    ld = round_up(K, 256) if layout == LAYOUT_GEMV else round_up(K, 16)
    codes = torch.empty(M, ld, device=x2d.device, dtype=torch.int8)
    inv = torch.empty(M, device=x2d.device, dtype=torch.float32)
    rowsum = torch.empty(M, device=x2d.device, dtype=torch.int32) if layout == LAYOUT_GEMV else None
    _lib.call("tesm_b200_quant_act", x2d.data_ptr(), dtype_code(x2d.dtype), M, K, x2d.stride(0), float(eps),
              codes.data_ptr(), ld, layout, inv.data_ptr(), _ptr(rowsum), _stream())
    return codes, inv, rowsum


def quant_act_into(x2d: torch.Tensor, eps: float, codes: torch.Tensor, col0: int, inv: torch.Tensor):
    """Row-major int8 codes of x written into columns [col0, col0 + K) of ``codes`` (16-byte
    aligned rows and col0), 1/s into ``inv``."""
    assert x2d.is_cuda and x2d.dim() == 2 and x2d.stride(1) == 1 and col0 % 16 == 0
    M, K = x2d.shape
    _lib.call("tesm_b200_quant_act", x2d.data_ptr(), dtype_code(x2d.dtype), M, K, x2d.stride(0), float(eps),
              codes.data_ptr() + col0, codes.stride(0), LAYOUT_ROWMAJOR, inv.data_ptr(), None, _stream())


def gemv(codes, inv, rowsum, pw: PackedWeight, M: int, out_dtype: torch.dtype, out=None, acc=False):
    dev = codes.device
    out = out if out is not None else torch.empty(M, pw.N, device=dev, dtype=out_dtype)
    accb = torch.empty(M, pw.N, device=dev, dtype=torch.int32) if acc else None
    _lib.call("tesm_b200_gemv_int2", codes.data_ptr(), codes.stride(0), inv.data_ptr(), rowsum.data_ptr(),
              pw.packed.data_ptr(), pw.packed.stride(0), pw.deq.data_ptr(), int(pw.per_row), M, pw.N, pw.K,
              out.data_ptr(), dtype_code(out.dtype), out.stride(0), _ptr(accb), pw.N, _stream())
    return (out, accb) if acc else out


_SPLITK = {}
SPLITK_MAX_M = 1024


SPLITK_COUNTERS = 4096  # int32 tile counters at the start of the scratch (zero between calls)


def splitk_workspace(M: int, N: int, device):
    """int32 split-K scratch shared by the small-M tensor-core GEMMs of a device: tile counters
    (zero-initialised here; every GEMM call leaves them zero again) followed by room for 8
    partial M x N slices.  None for large M, where split-K is never chosen."""
    if M > SPLITK_MAX_M:
        return None
    need = SPLITK_COUNTERS + 8 * round_up(M, 256) * round_up(N, 32)  # slices cover whole tiles
    key = torch.device(device).index
    buf = _SPLITK.get(key)
    if buf is None or buf.numel() < need:
        if buf is not None:
            torch.cuda.current_stream(device).synchronize()  # the old buffer may still be in use
        buf = torch.zeros(max(need, 1 << 20), device=device, dtype=torch.int32)
        _SPLITK[key] = buf
    return buf


def gemm(codes, inv, pw: PackedWeight, M: int, out_dtype: torch.dtype, out=None, acc=False):
    dev = codes.device
    out = out if out is not None else torch.empty(M, pw.N, device=dev, dtype=out_dtype)
    accb = torch.empty(M, pw.N, device=dev, dtype=torch.int32) if acc else None
    ws = splitk_workspace(M, pw.N, dev)
    _lib.call("tesm_b200_gemm_i8", codes.data_ptr(), codes.stride(0), inv.data_ptr(), pw.tern.data_ptr(),
              pw.tern.stride(0), pw.deq.data_ptr(), int(pw.per_row), M, pw.N, pw.K, out.data_ptr(),
              dtype_code(out.dtype), out.stride(0), _ptr(accb), pw.N, _ptr(ws), ws.numel() * 4 if ws is not None else 0,
              _stream())
    return (out, accb) if acc else out


def gemm_bf16(a: torch.Tensor, b: torch.Tensor, out_dtype=torch.bfloat16, out=None):
    """a (M, K) @ b (N, K)^T on the tensor cores (bf16 in, fp32 accumulate)."""
    M, K = a.shape
    N = b.shape[0]
    out = out if out is not None else torch.empty(M, N, device=a.device, dtype=out_dtype)
    _lib.call("tesm_b200_gemm_bf16", a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), M, N, K, out.data_ptr(),
              dtype_code(out.dtype), out.stride(0), _stream())
    return out


def gemm_acc(codes, inv, pw: PackedWeight, M: int, acc: torch.Tensor):
    """int32 accumulators only (no scaled output): the partial product of a row-parallel shard."""
    ws = splitk_workspace(M, pw.N, codes.device)
    _lib.call("tesm_b200_gemm_i8", codes.data_ptr(), codes.stride(0), inv.data_ptr(), pw.tern.data_ptr(),
              pw.tern.stride(0), pw.deq.data_ptr(), int(pw.per_row), M, pw.N, pw.K, None, dtype_code(torch.float32),
              pw.N, acc.data_ptr(), acc.stride(0), _ptr(ws), ws.numel() * 4 if ws is not None else 0, _stream())
    return acc


def acc_scale(acc, inv, pw: PackedWeight, out_dtype, out=None):
    """out = acc * inv_scale[row] * deq (the GEMM epilogue's float operations, bit for bit)."""
    M, N = acc.shape
    out = out if out is not None else torch.empty(M, N, device=acc.device, dtype=out_dtype)
    _lib.call("tesm_b200_acc_scale", acc.data_ptr(), M, N, inv.data_ptr(), pw.deq.data_ptr(), int(pw.per_row),
              out.data_ptr(), dtype_code(out.dtype), out.stride(0), _stream())
    return out


def combine_acc(acc1, acc2, inv1, inv2, deq1, deq2, proj, c_local, c_gate, out):
    """The dual-accumulator combine epilogue on summed int32 accumulators (bit for bit)."""
    M, N = out.shape
    _lib.call("tesm_b200_combine_acc", acc1.data_ptr(), acc2.data_ptr(), acc1.stride(0), M, N, inv1.data_ptr(),
              inv2.data_ptr(), deq1.data_ptr(), deq2.data_ptr(), proj.data_ptr(), dtype_code(proj.dtype),
              proj.stride(0), c_local, c_gate, out.data_ptr(), dtype_code(out.dtype), out.stride(0), _stream())
    return out


def row_absmax(x2d: torch.Tensor, out=None):
    M, K = x2d.shape
    out = out if out is not None else torch.empty(M, device=x2d.device, dtype=torch.float32)
    _lib.call("tesm_b200_row_absmax", x2d.data_ptr(), dtype_code(x2d.dtype), M, K, x2d.stride(0), out.data_ptr(),
              _stream())
    return out


def quant_act_amax(x2d: torch.Tensor, eps: float, amax: torch.Tensor) -> "QuantAct":
    """Row-major int8 codes of x with the row maxima given (global across tensor-parallel shards)."""
    M, K = x2d.shape
    ld = round_up(K, 16)
    codes = torch.empty(M, ld, device=x2d.device, dtype=torch.int8)
    inv = torch.empty(M, device=x2d.device, dtype=torch.float32)
    _lib.call("tesm_b200_quant_act_amax", x2d.data_ptr(), dtype_code(x2d.dtype), M, K, x2d.stride(0), float(eps),
              amax.data_ptr(), codes.data_ptr(), ld, LAYOUT_ROWMAJOR, inv.data_ptr(), None, _stream())
    return QuantAct(codes, inv, None, LAYOUT_ROWMAJOR, M)


def pack_shard(w_full: torch.Tensor, eps: float, rows=None, cols=None, per_row: bool = False) -> PackedWeight:
    """Ternary pack of a row or column slice of a weight with the scale of the FULL weight (the
    reference quantises each BitLinear as a whole, tesm.py:211-215)."""
    scale, deq = weight_scale(w_full, eps, per_row)
    w = w_full
    if rows is not None:
        w = w[rows[0]:rows[1]]
        if per_row:
            scale, deq = scale[rows[0]:rows[1]].contiguous(), deq[rows[0]:rows[1]].contiguous()
    if cols is not None:
        w = w[:, cols[0]:cols[1]]
    pw = pack_weight(w, eps, per_row, with_tern=True, scale=scale)
    pw.deq = deq
    return pw


def bitlinear_2d(x2d: torch.Tensor, pw: PackedWeight, eps: float, out_dtype=None, out=None, acc=False,
                 force: Optional[str] = None):
    """Quantise a (M, K) activation and multiply by a packed ternary weight."""
    M = x2d.shape[0]
    out_dtype = out_dtype or x2d.dtype
    path = force or ("gemv" if M <= GEMV_MAX_M else "gemm")
    if path == "gemv":
        codes, inv, rowsum = quant_act(x2d, eps, LAYOUT_GEMV)
        return gemv(codes, inv, rowsum, pw, M, out_dtype, out, acc)
    codes, inv, _ = quant_act(x2d, eps, LAYOUT_ROWMAJOR)
    return gemm(codes, inv, pw, M, out_dtype, out, acc)


# ------------------------------------------------------------------ pre-quantised activations
@dataclass
class QuantAct:
    """int8 activation codes of M rows ready for a BitLinear (layout GEMV or ROWMAJOR)."""
    codes: torch.Tensor
    inv: torch.Tensor
    rowsum: Optional[torch.Tensor]
    layout: int
    M: int


def layout_for(M: int) -> int:
    return LAYOUT_GEMV if M <= GEMV_MAX_M else LAYOUT_ROWMAJOR


def alloc_quant(M: int, K: int, device, layout: Optional[int] = None) -> QuantAct:
    layout = layout_for(M) if layout is None else layout
    ld = round_up(K, 256) if layout == LAYOUT_GEMV else round_up(K, 16)
    codes = torch.empty(M, ld, device=device, dtype=torch.int8)
    inv = torch.empty(M, device=device, dtype=torch.float32)
    rowsum = torch.empty(M, device=device, dtype=torch.int32) if layout == LAYOUT_GEMV else None
    return QuantAct(codes, inv, rowsum, layout, M)


def quantize(x2d: torch.Tensor, eps: float) -> QuantAct:
    M = x2d.shape[0]
    layout = layout_for(M)
    codes, inv, rowsum = quant_act(x2d, eps, layout)
    return QuantAct(codes, inv, rowsum, layout, M)


def matmul_q(q: QuantAct, pw: PackedWeight, out_dtype: torch.dtype, out=None):
    if q.layout == LAYOUT_GEMV:
        return gemv(q.codes, q.inv, q.rowsum, pw, q.M, out_dtype, out)
    return gemm(q.codes, q.inv, pw, q.M, out_dtype, out)


def pack_into(w: torch.Tensor, eps: float, packed: torch.Tensor, tern: Optional[torch.Tensor],
              scale: torch.Tensor, deq: torch.Tensor):
    """Pack one weight into caller-provided row slices (used to fuse gate/up weights)."""
    N, K = w.shape
    work = torch.empty(N, device=w.device, dtype=torch.float64)
    _lib.call("tesm_b200_weight_scale", w.data_ptr(), dtype_code(w.dtype), N, K, w.stride(0), 0, float(eps),
              scale.data_ptr(), deq.data_ptr(), work.data_ptr(), _stream())
    _lib.call("tesm_b200_pack_ternary", w.data_ptr(), dtype_code(w.dtype), N, K, w.stride(0), 0, scale.data_ptr(),
              packed.data_ptr(), packed.stride(0), _ptr(tern), tern.stride(0) if tern is not None else 0, _stream())


# ------------------------------------------------------------------ layer kernels
def scan_workspace(B: int, L: int, C: int, RM: int, device) -> torch.Tensor:
    n = ctypes.c_int64(0)
    _lib.call("tesm_b200_scan_workspace", B, L, C, RM, ctypes.addressof(n))
    return torch.empty(n.value, device=device, dtype=torch.uint8)


def siso_scan(proj, B, L, Dm, D, R, decay_bias, h0, states, f32, f64, scan_chunk=16):
    """SISO scan; ``scan_chunk`` is the module's state_scan_chunk_size (the reference's chunked
    fp64 formula clamps the in-chunk decay product at 1e-12, which the kernel reproduces)."""
    ws = scan_workspace(B, L, D, 1, proj.device)
    _lib.call("tesm_b200_siso_scan", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, D, R,
              int(scan_chunk), decay_bias.data_ptr(), _ptr(h0), states.data_ptr(), f32.data_ptr(), f64.data_ptr(), ws.data_ptr(),
              ws.numel(), _stream())


def mimo_scan(proj, B, L, Dm, H, D, R, RM, decay_bias, mimo_x, states, f32, f64):
    ws = scan_workspace(B, L, H * D, RM, proj.device)
    _lib.call("tesm_b200_mimo_scan", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, H, D, R, RM,
              decay_bias.data_ptr(), mimo_x.data_ptr(), states.data_ptr(), f32.data_ptr(), f64.data_ptr(),
              ws.data_ptr(), ws.numel(), _stream())


def siso_local_ent(proj, B, L, Dm, D, R, W, cross, bias, states, thr, es, base, out_tanh, out_chg):
    _lib.call("tesm_b200_siso_local_ent", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, D, R, W,
              _ptr(cross), bias.data_ptr(), states.data_ptr(), float(thr), float(es), float(base),
              out_tanh.data_ptr(), out_chg.data_ptr(), dtype_code(out_tanh.dtype), _stream())


def global_relbias(embed, scale, bias0, L):
    out = torch.empty(2 * L - 1, device=embed.device, dtype=torch.float32)
    _lib.call("tesm_b200_global_relbias", embed.data_ptr(), embed.numel(), float(scale), float(bias0), L,
              out.data_ptr(), _stream())
    return out


def global_ent_tc_ok(D, R):
    return R <= 64 and R % 2 == 0 and D <= 256


def siso_global_ent(proj, B, L, Dm, D, R, cross, relb, states, thr, es, base, out_tanh, out_chg, force=None):
    """Causal global entanglement: tensor-core kernel when ent_rank <= 64 and d_state <= 256
    (force="tc" / "simt" picks one for tests), else the fp32 SIMT kernel."""
    path = force or ("tc" if global_ent_tc_ok(D, R) else "simt")
    if path == "tc":
        n = ctypes.c_int64(0)
        _lib.call("tesm_b200_global_ent_tc_workspace", B, L, D, R, ctypes.addressof(n))
        raw = torch.empty(n.value + 1024, device=proj.device, dtype=torch.uint8)
        off = (-raw.data_ptr()) % 1024  # 1024-byte aligned start
        _lib.call("tesm_b200_siso_global_ent_tc", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm,
                  D, R, _ptr(cross), relb.data_ptr(), states.data_ptr(), float(thr), float(es), float(base),
                  out_tanh.data_ptr(), out_chg.data_ptr(), dtype_code(out_tanh.dtype), raw.data_ptr() + off,
                  n.value, _stream())
        return
    _lib.call("tesm_b200_siso_global_ent", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, D, R,
              _ptr(cross), relb.data_ptr(), states.data_ptr(), float(thr), float(es), float(base),
              out_tanh.data_ptr(), out_chg.data_ptr(), dtype_code(out_tanh.dtype), _stream())


def mimo_local_ent(proj, B, L, Dm, H, D, R, RM, W, bias, mimo_o, states, thr, es, base, quirk, out_tanh, out_chg):
    _lib.call("tesm_b200_mimo_local_ent", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, H, D, R,
              RM, W, bias.data_ptr(), mimo_o.data_ptr(), states.data_ptr(), float(thr), float(es), float(base),
              int(quirk), out_tanh.data_ptr(), out_chg.data_ptr(), dtype_code(out_tanh.dtype), _stream())


def combine(proj, M, Dm, C, Rc, sp, ep, y):
    _lib.call("tesm_b200_combine", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), M, Dm, C, Rc,
              sp.data_ptr(), ep.data_ptr(), dtype_code(sp.dtype), y.data_ptr(), dtype_code(y.dtype), _stream())


def cache_fill(proj, states, RM, B, L, Dm, H, D, R, W, base, final64, state, kc, vc, ctl):
    _lib.call("tesm_b200_cache_fill", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), states.data_ptr(), RM,
              B, L, Dm, H, D, R, W, float(base), final64.data_ptr(), state.data_ptr(), kc.data_ptr(), vc.data_ptr(),
              ctl.data_ptr(), _stream())


def decode_step(proj, B, Dm, H, D, R, W, decay_bias, bias, cross, state, kc, vc, ctl, thr, es, base, out_tanh,
                out_chg, new_state):
    _lib.call("tesm_b200_decode_step", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, Dm, H, D, R, W,
              decay_bias.data_ptr(), bias.data_ptr(), _ptr(cross), state.data_ptr(), kc.data_ptr(), vc.data_ptr(),
              ctl.data_ptr(), float(thr), float(es), float(base), out_tanh.data_ptr(), out_chg.data_ptr(),
              dtype_code(out_tanh.dtype), _ptr(new_state), _stream())


def siso_decode_step_codes(proj, B, Dm, D, R, W, decay_bias, bias, cross, state, kc, vc, ctl, thr, es, base,
                           act_dtype, eps1, eps2, new_state, xstate=None, xq: Optional[PackedWeight] = None,
                           xq_eps=0.0):
    """One-token SISO step emitting the int8 codes of tanh(ent) | ent - s for the combine GEMM.
    With ``xstate`` (the previous layer's fp32 state, (B, D)) and ``xq`` (cross_layer_q_proj's
    packed weight) the step computes the cross-layer query bias itself."""
    Dp = round_up(D, 128)
    codes = torch.empty(B, 2 * Dp, device=proj.device, dtype=torch.int8)
    inv1 = torch.empty(B, device=proj.device, dtype=torch.float32)
    inv2 = torch.empty(B, device=proj.device, dtype=torch.float32)
    _lib.call("tesm_b200_siso_decode_step_codes", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, Dm, D,
              R, W, decay_bias.data_ptr(), bias.data_ptr(), _ptr(cross), state.data_ptr(), kc.data_ptr(),
              vc.data_ptr(), ctl.data_ptr(), float(thr), float(es), float(base), dtype_code(act_dtype), float(eps1),
              float(eps2), codes.data_ptr(), codes.stride(0), Dp, inv1.data_ptr(), inv2.data_ptr(), _ptr(new_state),
              _ptr(xstate), _ptr(xq.tern) if xq is not None else None, xq.tern.stride(0) if xq is not None else 0,
              _ptr(xq.deq) if xq is not None else None, float(xq_eps), _stream())
    return codes, inv1, inv2, Dp


def embed(ids, emb, pos_emb, pos_dev, pos_host, out):
    B, L = ids.shape
    _lib.call("tesm_b200_embed", ids.data_ptr(), B, L, emb.data_ptr(), pos_emb.data_ptr(), dtype_code(emb.dtype),
              emb.shape[1], _ptr(pos_dev), int(pos_host), out.data_ptr(), dtype_code(out.dtype), _stream())


def add_rmsnorm_quant(x, residual, residual_out, weight, eps, qeps, q: Optional[QuantAct], y_out=None):
    M, K = x.shape
    _lib.call("tesm_b200_add_rmsnorm_quant", x.data_ptr(), dtype_code(x.dtype), _ptr(residual), _ptr(residual_out),
              weight.data_ptr(), float(eps), M, K, float(qeps), _ptr(q.codes) if q else None,
              q.codes.stride(0) if q else 0, q.layout if q else 0, _ptr(q.inv) if q else None,
              _ptr(q.rowsum) if q else None, _ptr(y_out), dtype_code(y_out.dtype) if y_out is not None else 0,
              _stream())


def silu_mul(gu, F, out, blk=0):
    _lib.call("tesm_b200_silu_mul", gu.data_ptr(), dtype_code(gu.dtype), gu.shape[0], F, blk, out.data_ptr(),
              dtype_code(out.dtype), _stream())


_SWIGLU_WIDE = os.environ.get("TESM_SKINNY_WIDE", "1") != "0"


def gemm_swiglu(q: QuantAct, pw: PackedWeight, out_dtype, out=None):
    """Interleaved gate/up weight (blocks of 128 rows) -> silu(gate) * up, width pw.N // 2."""
    F = pw.N // 2
    out = out if out is not None else torch.empty(q.M, F, device=q.codes.device, dtype=out_dtype)
    if q.M <= 128 or (q.M <= 256 and not _SWIGLU_WIDE):
        # small batches: skinny-tile GEMM, then the gate on the interleaved output
        gu = gemm(q.codes, q.inv, pw, q.M, out_dtype)
        silu_mul(gu, F, out, 128)
        return out
    ws = splitk_workspace(q.M, pw.N, q.codes.device)
    _lib.call("tesm_b200_gemm_i8_swiglu", q.codes.data_ptr(), q.codes.stride(0), q.inv.data_ptr(), pw.tern.data_ptr(),
              pw.tern.stride(0), pw.deq.data_ptr(), q.M, F, pw.K, out.data_ptr(), dtype_code(out.dtype),
              out.stride(0), _ptr(ws), ws.numel() * 4 if ws is not None else 0, _stream())
    return out


def device_status() -> int:
    v = ctypes.c_int(0)
    _lib.call("tesm_b200_device_status", ctypes.addressof(v))
    return v.value



def siso_local_ent_codes(proj, B, L, Dm, D, R, W, cross, bias, states, thr, es, base, act_dtype, eps1, eps2):
    """Local entanglement emitting the int8 codes of tanh(ent) | ent - s (see the C header)."""
    Dp = round_up(D, 128)
    M = B * L
    codes = torch.empty(M, 2 * Dp, device=proj.device, dtype=torch.int8)
    inv1 = torch.empty(M, device=proj.device, dtype=torch.float32)
    inv2 = torch.empty(M, device=proj.device, dtype=torch.float32)
    _lib.call("tesm_b200_siso_local_ent_codes", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, D,
              R, W, _ptr(cross), bias.data_ptr(), states.data_ptr(), float(thr), float(es), float(base),
              dtype_code(act_dtype), float(eps1), float(eps2), codes.data_ptr(), codes.stride(0), Dp,
              inv1.data_ptr(), inv2.data_ptr(), _stream())
    return codes, inv1, inv2, Dp


def gemm_combine(codes, Kh, inv1, inv2, tern, deq1, deq2, proj, c_local, c_gate, M, N, out):
    _lib.call("tesm_b200_gemm_i8_combine", codes.data_ptr(), codes.stride(0), Kh, inv1.data_ptr(), inv2.data_ptr(),
              tern.data_ptr(), tern.stride(0), deq1.data_ptr(), deq2.data_ptr(), proj.data_ptr(),
              dtype_code(proj.dtype), proj.stride(0), c_local, c_gate, M, N, out.data_ptr(), dtype_code(out.dtype),
              out.stride(0), _stream())
    return out


def mimo_global_ent(proj, B, L, Dm, H, D, R, RM, relb, mimo_o, states, thr, base, out_tanh, out_chg):
    acc_e = acc_c = None
    if RM > 1:
        acc_e = torch.empty(B * L, H * D, device=proj.device, dtype=torch.float32)
        acc_c = torch.empty_like(acc_e)
    _lib.call("tesm_b200_mimo_global_ent", proj.data_ptr(), dtype_code(proj.dtype), proj.stride(0), B, L, Dm, H, D,
              R, RM, relb.data_ptr(), mimo_o.data_ptr(), states.data_ptr(), float(thr), float(base), _ptr(acc_e),
              _ptr(acc_c), out_tanh.data_ptr(), out_chg.data_ptr(), dtype_code(out_tanh.dtype), _stream())


# ------------------------------------------------------------------ beam search
MAX_BEAMS = 32


def _need(ok, what: str):
    if not ok:
        raise ValueError("tesm_b200 " + what)


def _no_grad(what: str, *tensors):
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"tesm_b200 {what} has no autograd path (use torch.no_grad())")


def _call_on(index: int, name: str, *args):
    """Launch on the current stream of device ``index``, whichever device is current."""
    if index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _check(what: str, name: str, t: Optional[torch.Tensor], shape, dtype: torch.dtype, index: int):
    """A dense tensor of this shape and type on device ``index`` (or None)."""
    if t is not None and (t.shape != shape or t.dtype != dtype or t.get_device() != index or not t.is_contiguous()):
        raise ValueError(f"tesm_b200 {what}: {name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on "
                         f"cuda:{index}, got {t.dtype} {tuple(t.shape)} {t.stride()} on {t.device}")


@dataclass
class BeamStep:
    """One selection step: (prompts, beams) tensors of the chosen continuations."""
    tokens: torch.Tensor    # int64
    parents: torch.Tensor   # int32, the beam each one continues
    scores: torch.Tensor    # float32 summed log-probabilities
    finished: torch.Tensor  # bool
    lengths: torch.Tensor   # int32


@lru_cache(maxsize=256)
def _beam_workspace(dtype: int, G: int, W: int, V: int, K: int) -> int:
    n = ctypes.c_int64(0)
    _lib.call("tesm_b200_beam_select_workspace", dtype, G, W, V, K, ctypes.addressof(n))
    return n.value


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                eos_token_id: Optional[int] = None, pad_token_id: int = 0,
                length_penalty: float = 0.0) -> BeamStep:
    """The best ``beams`` continuations of every prompt's beams (tesm_b200_beam_select).

    logits (prompts, W, vocab) float32 or bfloat16 with unit vocabulary stride, scores (prompts, W)
    float32.  A live beam offers ``scores + log_softmax(logits)`` for every token, a ``finished`` one
    (bool) only itself with ``pad_token_id``; they are ranked by score / length ** length_penalty with
    ``lengths`` (int32) counting the new token, ties to the lower beam, then the lower token (beams
    whose keys differ by less than about 1e-6 may change places: fp32 exponentials).  Beams
    start as ``scores = [0, -inf, ...]``: candidates of score -inf never win, and slots that
    nothing is left for come back finished with score -inf.  ``beams`` defaults to W; both at most 32."""
    what = "beam_select"
    if logits.dim() != 3 or not logits.is_cuda:
        raise ValueError(f"tesm_b200 {what}: logits must be a (prompts, beams, vocab) CUDA tensor, got "
                         f"{tuple(logits.shape)} on {logits.device}")
    G, W, V = logits.shape
    K = W if beams is None else int(beams)
    code, dev = dtype_code(logits.dtype), logits.get_device()
    if not (1 <= W <= MAX_BEAMS and 1 <= K <= MAX_BEAMS):
        raise ValueError(f"tesm_b200 {what}: 1 to {MAX_BEAMS} beams, got {W} in and {K} out")
    ldg, ldw, ldv = logits.stride()
    if V < 1 or (ldv != 1 and V > 1):
        raise ValueError(f"tesm_b200 {what}: the logits need unit stride over a vocabulary, got {logits.stride()}")
    if not 0 <= pad_token_id < V:
        raise ValueError(f"tesm_b200 {what}: pad_token_id {pad_token_id} is outside the vocabulary of {V}")
    if length_penalty != 0.0 and lengths is None:
        raise ValueError(f"tesm_b200 {what}: a length penalty needs lengths")
    _check(what, "scores", scores, (G, W), torch.float32, dev)
    _check(what, "finished", finished, (G, W), torch.bool, dev)
    _check(what, "lengths", lengths, (G, W), torch.int32, dev)
    _no_grad(what, logits, scores)
    out = (G, K)
    tokens = scores.new_empty(out, dtype=torch.int64)
    parents = scores.new_empty(out, dtype=torch.int32)
    out_scores = scores.new_empty(out)
    out_finished = scores.new_empty(out, dtype=torch.bool)
    out_lengths = scores.new_empty(out, dtype=torch.int32)
    ws_bytes = _beam_workspace(code, G, W, V, K)
    ws = scores.new_empty(ws_bytes, dtype=torch.uint8)
    _call_on(dev, "tesm_b200_beam_select", logits.data_ptr(), code, ldg if G > 1 else 0, ldw if W > 1 else 0, G, W, V,
             K, scores.data_ptr(), _ptr(finished), _ptr(lengths), -1 if eos_token_id is None else eos_token_id,
             pad_token_id, length_penalty, tokens.data_ptr(), parents.data_ptr(), out_scores.data_ptr(),
             out_finished.data_ptr(), out_lengths.data_ptr(), ws.data_ptr(), ws_bytes)
    return BeamStep(tokens, parents, out_scores, out_finished, out_lengths)


def _row_layout(what: str, t: torch.Tensor, rows: int):
    """(data pointer, row bytes, row stride in bytes) of a tensor whose rows are dense."""
    if t.dim() < 1 or t.shape[0] != rows:
        raise ValueError(f"tesm_b200 {what}: a state of shape {tuple(t.shape)} has not {rows} rows")
    n = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != n:
            raise ValueError(f"tesm_b200 {what}: the rows of a state must be dense (shape {tuple(t.shape)}, strides "
                             f"{t.stride()})")
        n *= size
    es = t.element_size()
    stride = t.stride(0) if rows > 1 else n
    _need(stride >= n, f"{what}: the rows of a state overlap")
    return t.data_ptr(), n * es, stride * es


def _rows_disjoint(a, b) -> bool:
    """Whether two (pointer, row bytes, stride, rows) sets of rows share no byte."""
    (pa, na, sa, ra), (pb, nb, sb, rb) = sorted((a, b))
    if not na or not nb or not ra or not rb or pa + (ra - 1) * sa + na <= pb:
        return True
    off = (pb - pa) % sa
    return sa == sb and off >= na and off + nb <= sa  # interleaved columns of one buffer


class StateReorder:
    """Moves the rows of a fixed set of state tensors along with their beams, in place.

    ``states``: tensors of prompts * beams rows (any type and row shape; rows dense, any row
    stride), e.g. the caches of all layers.  ``plan(parents)`` with parents (prompts, beams) int32
    makes row g * beams + k of every state the row g * beams + parents[g, k], all in one launch per 128
    tensors; each column of rows is read into registers before it is stored, so no copy is kept.
    With ``out`` (tensors of prompts * beams rows) the rows come from ``states`` of prompts * ``beams_in``
    rows instead: beams_in = 1 and parents of zeros spreads one row per prompt over its beams.
    A parent out of range leaves its row as it is and sets :func:`device_status` to 1.  The plan holds
    the tensors and their addresses: they stay where they are for its life.  Making one costs about 0.25 ms of
    host time for 96 tensors (2 ms if all are slices of one buffer), a call 7 us."""

    def __init__(self, states: Sequence[torch.Tensor], beams: int, out: Optional[Sequence[torch.Tensor]] = None,
                 beams_in: Optional[int] = None):
        what = "reorder_states"
        states = list(states)
        dst = states if out is None else list(out)
        beams_in = beams if beams_in is None else int(beams_in)
        _need(len(states) > 0, f"{what}: no states")
        _need(1 <= beams <= MAX_BEAMS, f"{what}: 1 to {MAX_BEAMS} beams, got {beams}")
        _need(beams_in >= 1 and (out is not None or beams_in == beams), f"{what}: in place, beams_in equals beams")
        _need(len(dst) == len(states), f"{what}: {len(states)} states but {len(dst)} outputs")
        self.device = states[0].get_device()
        _need(all(t.is_cuda and t.get_device() == self.device for t in states + dst),
              f"{what}: all states must be on one CUDA device")
        rows_in = states[0].shape[0] if states[0].dim() else 0
        _need(rows_in % beams_in == 0, f"{what}: {rows_in} rows are no multiple of {beams_in} beams")
        self.prompts, self.beams, self.beams_in = rows_in // beams_in, int(beams), beams_in
        rows_out = self.prompts * self.beams
        self._table = (_lib.StateRows * len(states))()
        src_rows, dst_rows = [], []
        for e, s, d in zip(self._table, states, dst):
            e.src, e.row_bytes, e.src_stride = _row_layout(what, s, rows_in)
            src_rows.append((e.src or 0, e.row_bytes, e.src_stride, rows_in))
            if d is s:
                e.dst, e.dst_stride = e.src, e.src_stride
                dst_rows.append(src_rows[-1])
            else:
                _need(s.dtype == d.dtype and s.shape[1:] == d.shape[1:], f"{what}: a state and its output differ in type "
                                                                         f"or row shape")
                e.dst, _, e.dst_stride = _row_layout(what, d, rows_out)
                dst_rows.append((e.dst or 0, e.row_bytes, e.dst_stride, rows_out))
        _no_grad(what, *states, *dst)
        # what is written is written once, and nothing that another entry reads; sorted by address, a
        # set of rows can only meet those that begin before its end
        every = sorted([(r, True) for r in dst_rows] + ([(r, False) for r in src_rows] if out is not None else []))
        for i, (r, written) in enumerate(every):
            end = r[0] + (r[3] - 1) * r[2] + r[1]
            for other, also in every[i + 1:]:
                if other[0] >= end:
                    break
                _need(not (written or also) or _rows_disjoint(r, other), f"{what}: states share memory")
        self._keep = (states, dst)
        self._args = (ctypes.addressof(self._table), len(states), self.prompts, self.beams_in, self.beams)

    def __call__(self, parents: torch.Tensor):
        _check("reorder_states", "parents", parents, (self.prompts, self.beams), torch.int32, self.device)
        _call_on(self.device, "tesm_b200_reorder_states", *self._args, parents.data_ptr())
        return self._keep[1]


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, out: Optional[Sequence[torch.Tensor]] = None):
    """One :class:`StateReorder` call; a loop keeps the plan.  Returns the reordered tensors."""
    _need(parents.dim() == 2 and parents.shape[0] > 0, "reorder_states: parents must be (prompts, beams)")
    states = list(states)
    _need(len(states) > 0 and states[0].dim() > 0 and states[0].shape[0] % parents.shape[0] == 0,
          f"reorder_states: the states' rows are no multiple of {parents.shape[0]} prompts")
    return StateReorder(states, parents.shape[1], out, None if out is None else
                        states[0].shape[0] // parents.shape[0])(parents)


# ------------------------------------------------------------------ selective state space scan
def _rows3(what: str, name: str, t: torch.Tensor, shape, dtype, index: int):
    """(batch, token) element strides of a (B, L, n) tensor with unit innermost stride."""
    if t.shape != shape or t.dtype != dtype or t.get_device() != index:
        raise ValueError(f"tesm_b200 {what}: {name} must be a {dtype} tensor of shape {tuple(shape)} on cuda:{index}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    b, l, n = t.stride()
    if n != 1 and shape[2] > 1:
        raise ValueError(f"tesm_b200 {what}: {name} needs unit stride along its last dimension, got {t.stride()}")
    return b if shape[0] > 1 else 0, l if shape[1] > 1 else 0


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, silu: bool = True,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Short causal depthwise convolution of a prompt, or of one token (L = 1), with SiLU.

    x (B, L, D) float32 or bfloat16 with unit channel stride; weight (D, K) float32, K = 2 .. 8, the last
    tap on the current token; bias (D,) float32.  ``state`` (B, K - 1, D) of x's type holds the inputs
    before the first token (zeros if not given) and is replaced by the last K - 1 inputs.
    ``lengths`` (B,) int32: tokens of each sequence (right-padded); outputs behind them are zeros."""
    what = "causal_conv"
    if x.dim() != 3 or not x.is_cuda:
        raise ValueError(f"tesm_b200 {what}: x must be a (batch, tokens, channels) CUDA tensor")
    shape, xdt, dev = x.shape, x.dtype, x.get_device()
    B, L, D = shape
    code = dtype_code(xdt)
    xb, xl = _rows3(what, "x", x, shape, xdt, dev)
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        raise ValueError(f"tesm_b200 {what}: weight must be (channels, 2 to 8 taps), got {tuple(weight.shape)}")
    K = weight.shape[1]
    _check(what, "weight", weight, (D, K), torch.float32, dev)
    _check(what, "bias", bias, (D,), torch.float32, dev)
    _check(what, "state", state, (B, K - 1, D), xdt, dev)
    _check(what, "lengths", lengths, (B,), torch.int32, dev)
    _no_grad(what, x, weight, bias)
    if out is None:
        out = x.new_empty(shape)
    ob, ol = _rows3(what, "out", out, shape, xdt, dev)
    _call_on(dev, "tesm_b200_causal_conv", x.data_ptr(), code, xb, xl, B, L, D, K, weight.data_ptr(), _ptr(bias),
             _ptr(state), _ptr(lengths), silu, out.data_ptr(), ob, ol)
    return out


@lru_cache(maxsize=256)
def _scan_workspace(B: int, L: int, D: int, N: int) -> int:
    n = ctypes.c_int64(0)
    _lib.call("tesm_b200_ssm_scan_workspace", B, L, D, N, ctypes.addressof(n))
    return n.value


def ssm_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, Bm: torch.Tensor, Cm: torch.Tensor, *,
             D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
             dt_bias: Optional[torch.Tensor] = None, softplus: bool = True, state: Optional[torch.Tensor] = None,
             lengths: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Selective state space scan of a prompt, or of one token (L = 1):

        dt = softplus(dt + dt_bias);  h = exp(dt A) h + (dt x) Bm;  y = Cm . h + D x;  out = y silu(z)

    x, dt, z (B, L, channels) and Bm, Cm (B, L, N) of one type (float32 or bfloat16) with unit
    innermost stride, so slices of a projection are taken as they are; A (channels, N), D and dt_bias
    (channels,) float32; N = 1 .. 128.  ``state`` (B, channels, N) float32 holds h before the first token
    (zeros if not given) and is replaced by h after the last.  ``lengths`` (B,) int32: tokens of each
    sequence (right-padded); outputs behind them are zeros and do not touch the state.  A step or an x
    that is infinite or NaN makes its channel's outputs and states from there on infinite or NaN; other
    channels do not see it."""
    what = "ssm_scan"
    if x.dim() != 3 or not x.is_cuda:
        raise ValueError(f"tesm_b200 {what}: x must be a (batch, tokens, channels) CUDA tensor")
    shape, xdt, dev = x.shape, x.dtype, x.get_device()
    B, L, C = shape
    code = dtype_code(xdt)
    if A.dim() != 2 or not 1 <= A.shape[1] <= 128:
        raise ValueError(f"tesm_b200 {what}: A must be (channels, 1 to 128 states), got {tuple(A.shape)}")
    N = A.shape[1]
    if out is None:
        out = x.new_empty(shape)
    bc = (B, L, N)
    strides = (ctypes.c_int64 * 12)(*_rows3(what, "x", x, shape, xdt, dev), *_rows3(what, "dt", dt, shape, xdt, dev),
                                    *_rows3(what, "Bm", Bm, bc, xdt, dev), *_rows3(what, "Cm", Cm, bc, xdt, dev),
                                    *((0, 0) if z is None else _rows3(what, "z", z, shape, xdt, dev)),
                                    *_rows3(what, "out", out, shape, xdt, dev))
    _check(what, "A", A, (C, N), torch.float32, dev)
    _check(what, "D", D, (C,), torch.float32, dev)
    _check(what, "dt_bias", dt_bias, (C,), torch.float32, dev)
    _check(what, "state", state, (B, C, N), torch.float32, dev)
    _check(what, "lengths", lengths, (B,), torch.int32, dev)
    _no_grad(what, x, dt, A, Bm, Cm, D, z, dt_bias, state)
    ws_bytes = _scan_workspace(B, L, C, N) if L > 1 else 0
    ws = A.new_empty(ws_bytes // 4) if ws_bytes else None
    _call_on(dev, "tesm_b200_ssm_scan", x.data_ptr(), dt.data_ptr(), Bm.data_ptr(), Cm.data_ptr(), _ptr(z),
             out.data_ptr(), strides, code, B, L, C, N, A.data_ptr(), _ptr(D), _ptr(dt_bias), softplus, _ptr(state),
             _ptr(lengths), _ptr(ws), ws_bytes)
    return out
