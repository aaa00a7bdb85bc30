"""Python entry points over the C ABI, taking torch device tensors.

Each function fills one descriptor of ``include/th_hip.h`` and launches on the
current torch stream. No function here computes anything on the host: if the
library is missing or the device is not gfx950 they raise
:class:`~torch_helion.hip.abi.HipBackendError`.
"""

from __future__ import annotations

import contextlib
import ctypes as C
import functools
import math
import struct
from dataclasses import dataclass, field
from typing import Sequence

import torch

from . import abi

_DT = {torch.float32: abi.TH_F32, torch.bfloat16: abi.TH_BF16, torch.float16: abi.TH_F16,
       torch.float8_e4m3fn: abi.TH_F8E4M3, torch.int32: abi.TH_I32, torch.int64: abi.TH_I64}


def th_dtype(t: torch.Tensor | torch.dtype) -> int:
    dt = t if isinstance(t, torch.dtype) else t.dtype
    if dt not in _DT:
        raise abi.HipBackendError("dtype", abi.TH_ERR_UNSUPPORTED, f"{dt} has no kernel")
    return _DT[dt]


def _lib(t: torch.Tensor) -> C.CDLL:
    if t.device.type != "cuda":
        raise abi.HipBackendError("device", abi.TH_ERR_INVALID, f"tensor on {t.device}, expected a HIP device")
    return abi.init_device(t.device.index or 0)


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _row_major(t: torch.Tensor, name: str) -> int:
    """Row stride of a 2-D tensor whose last dim is contiguous."""
    if t.dim() != 2 or t.stride(1) != 1:
        raise abi.HipBackendError(name, abi.TH_ERR_INVALID, f"expected a 2-D row-major tensor, got {tuple(t.shape)} strides {t.stride()}")
    return t.stride(0)


# ------------------------------------------------------------------ gemm
def acc_tile(n: int, n_acc: int, dtype: torch.dtype) -> int:
    return int(abi.load().th_gemm_acc_tile(n, n_acc, th_dtype(dtype)))


def pack_rhs(ws: Sequence[torch.Tensor], dtype: torch.dtype, out: torch.Tensor | None = None) -> torch.Tensor:
    """Pack [K, N] operands into th_gemm's K-contiguous interleaved layout."""
    lib = _lib(ws[0])
    k, n = ws[0].shape
    for w in ws:
        if tuple(w.shape) != (k, n) or w.dtype != ws[0].dtype:
            raise abi.HipBackendError("th_gemm_pack_rhs", abi.TH_ERR_INVALID, "operands differ in shape/dtype")
    nbytes = lib.th_gemm_packed_bytes(n, k, len(ws), th_dtype(dtype))
    if nbytes <= 0:
        raise abi.HipBackendError("th_gemm_packed_bytes", abi.TH_ERR_INVALID, f"N={n} K={k} n_acc={len(ws)}")
    if out is None:
        out = torch.empty(nbytes, dtype=torch.uint8, device=ws[0].device)
    elif out.numel() * out.element_size() < nbytes:
        raise abi.HipBackendError("th_gemm_pack_rhs", abi.TH_ERR_INVALID, "packed buffer too small")
    ptrs = (C.c_void_p * len(ws))(*[w.data_ptr() for w in ws])
    lds = (C.c_int64 * len(ws))(*[_row_major(w, "pack_rhs") for w in ws])
    abi.check(lib.th_gemm_pack_rhs(ptrs, lds, th_dtype(ws[0]), n, k, len(ws), th_dtype(dtype), out.data_ptr(),
                                   _stream(ws[0])), "th_gemm_pack_rhs")
    return out


@dataclass
class EpiSpec:
    """One fused output of th_gemm (see th_epi_op in include/th_hip.h). ``cols``: the
    accumulator column window [begin, end) the output holds (None: all N columns)."""

    op: int
    out: torch.Tensor
    a: int = 0
    b: int = -1
    e: int = -1
    cols: tuple[int, int] | None = None


@dataclass
class GemmCall:
    M: int
    N: int
    K: int
    n_acc: int
    lhs: torch.Tensor
    packed: torch.Tensor
    outs: list[EpiSpec]
    sumsq: bool = False
    rscale_mask: int = 0
    inv_k: float = 0.0
    eps: float = 0.0
    extras: list[torch.Tensor] = field(default_factory=list)
    rope_cos: torch.Tensor | None = None
    rope_sin: torch.Tensor | None = None
    rope_head_dim: int = 0
    rope_period: int = 0
    sumsq_out: torch.Tensor | None = None
    in_dtype: torch.dtype | None = None        # torch.float8_e4m3fn: bf16 lhs x e4m3 packed rhs
    rhs_scale: torch.Tensor | None = None      # fp8: [n_acc, N] fp32 per-column scales
    workspace: torch.Tensor | None = None      # gemm_workspace_bytes(...) bytes (fp8: required; fp32: optional)
    lhs_gain: torch.Tensor | None = None       # fp8: [K] fp32, products use lhs * gain (RMSNorm gain)
    rs_parts: torch.Tensor | None = None       # bf16 (fp8 without lhs_gain), with sumsq: [M, parts] fp32, the
                                               # rows' sums of squares as partial sums (the lhs producer's),
                                               # used instead of sum lhs^2
    gain_out: tuple[int, torch.Tensor, torch.Tensor] | None = None
    # fp8: (output index, gain [N] fp32, ss_parts_out [M, N/256] fp32): that bf16 output is stored as
    # bf16(bf16(v) * gain) and its rows' sums of bf16(v)^2 go to ss_parts_out, 256 columns per part
    # (the next GEMM's lhs with its RMSNorm gain applied, and that GEMM's rs_parts)

    def descriptor(self) -> abi.GemmDesc:
        d = abi.GemmDesc()
        d.M, d.N, d.K, d.n_acc = self.M, self.N, self.K, self.n_acc
        d.in_dtype = th_dtype(self.in_dtype if self.in_dtype is not None else self.lhs)
        if self.rhs_scale is not None:
            if self.rhs_scale.dtype != torch.float32 or not self.rhs_scale.is_contiguous() \
                    or self.rhs_scale.numel() != self.n_acc * self.N:
                raise abi.HipBackendError("th_gemm", abi.TH_ERR_INVALID, "rhs_scale must be contiguous fp32 [n_acc, N]")
            d.rhs_scale = self.rhs_scale.data_ptr()
        if self.workspace is not None:
            d.workspace = self.workspace.data_ptr()
            d.workspace_bytes = self.workspace.numel() * self.workspace.element_size()
        d.lhs = self.lhs.data_ptr()
        d.ld_lhs = _row_major(self.lhs, "th_gemm lhs")
        d.rhs_packed = self.packed.data_ptr()
        d.sumsq = 1 if self.sumsq else 0
        d.rscale_mask = self.rscale_mask
        d.inv_k, d.eps = self.inv_k, self.eps
        d.n_extra = len(self.extras)
        for i, x in enumerate(self.extras):
            d.extra[i] = x.data_ptr()
            d.ld_extra[i] = _row_major(x, "th_gemm extra")
            d.extra_dtype[i] = th_dtype(x)
        if self.rope_cos is not None:
            d.rope_cos, d.rope_sin = self.rope_cos.data_ptr(), self.rope_sin.data_ptr()
            d.rope_head_dim, d.rope_period = self.rope_head_dim, self.rope_period
        d.n_out = len(self.outs)
        for i, o in enumerate(self.outs):
            e = d.out[i]
            e.op, e.a, e.b, e.e = o.op, o.a, o.b, o.e
            e.ptr = o.out.data_ptr()
            e.ld = _row_major(o.out, "th_gemm out")
            e.dtype = th_dtype(o.out)
            if o.cols is not None:
                e.col_begin, e.col_end = o.cols
        if self.sumsq_out is not None:
            d.sumsq_out = self.sumsq_out.data_ptr()
        if self.lhs_gain is not None:
            if self.lhs_gain.dtype != torch.float32 or not self.lhs_gain.is_contiguous() or self.lhs_gain.numel() != self.K:
                raise abi.HipBackendError("th_gemm", abi.TH_ERR_INVALID, "lhs_gain must be contiguous fp32 [K]")
            d.lhs_gain = self.lhs_gain.data_ptr()
        if self.rs_parts is not None:
            if self.rs_parts.dtype != torch.float32 or self.rs_parts.dim() != 2 or self.rs_parts.shape[0] != self.M:
                raise abi.HipBackendError("th_gemm", abi.TH_ERR_INVALID, "rs_parts must be fp32 [M, parts]")
            d.rs_parts, d.ld_rs_parts = self.rs_parts.data_ptr(), _row_major(self.rs_parts, "th_gemm rs_parts")
            d.n_rs_parts = self.rs_parts.shape[1]
        if self.gain_out is not None:
            idx, g, parts = self.gain_out
            if g.dtype != torch.float32 or not g.is_contiguous() or g.numel() != self.N:
                raise abi.HipBackendError("th_gemm", abi.TH_ERR_INVALID, "gain_out gain must be contiguous fp32 [N]")
            if parts.dtype != torch.float32 or parts.dim() != 2 or parts.shape[0] != self.M \
                    or parts.shape[1] < self.N // 256:
                raise abi.HipBackendError("th_gemm", abi.TH_ERR_INVALID, "ss_parts_out must be fp32 [M, N/256]")
            d.gain_out, d.gain_out_index = g.data_ptr(), idx
            d.ss_parts_out, d.ld_ss_parts_out = parts.data_ptr(), _row_major(parts, "th_gemm ss_parts_out")
        return d


def gemm_workspace_bytes(M: int, N: int, K: int, n_acc: int, in_dtype: torch.dtype) -> int:
    n = abi.load().th_gemm_workspace_bytes(M, N, K, n_acc, th_dtype(in_dtype))
    if n < 0:
        raise abi.HipBackendError("th_gemm_workspace_bytes", abi.TH_ERR_INVALID, f"M={M} N={N} K={K} n_acc={n_acc}")
    return int(n)


def gemm(call: GemmCall, kernel: str | None = None) -> None:
    lib = _lib(call.lhs)
    d = call.descriptor()
    abi.check(lib.th_gemm(C.byref(d), _stream(call.lhs)), "th_gemm", kernel)


def gemm_route(call: GemmCall) -> tuple[int, int, int, float]:
    """(abi.LOOP_*, tile rows, packed tile columns) that th_gemm runs for this call, and the
    time a bf16 loop is estimated to take (us on the device, 0.0 for the other types)."""
    route, us = (C.c_int32 * 3)(), C.c_double()
    d = call.descriptor()
    abi.check(abi.load().th_gemm_route(C.byref(d), route, C.byref(us)), "th_gemm_route")
    return route[0], route[1], route[2], us.value


def gemm_noalloc(call: GemmCall, kernel: str | None = None) -> None:
    """th_gemm_noalloc: the same GEMM with the library's fixed per-GPU scratch in place of a
    workspace (``call.workspace`` is ignored); allocates nothing."""
    lib = _lib(call.lhs)
    d = call.descriptor()
    abi.check(lib.th_gemm_noalloc(C.byref(d), _stream(call.lhs)), "th_gemm_noalloc", kernel)


# --------------------------------------------------------------- RMSNorm
def rmsnorm(x: torch.Tensor, gain: torch.Tensor, eps: float, out: torch.Tensor, inv_k: float | None = None,
            kernel: str | None = None, out32: torch.Tensor | None = None) -> torch.Tensor:
    lib = _lib(x)
    d = abi.RmsNormDesc()
    d.M, d.K = x.shape
    d.x, d.ld_x, d.x_dtype = x.data_ptr(), _row_major(x, "th_rmsnorm x"), th_dtype(x)
    d.out, d.ld_out, d.out_dtype = out.data_ptr(), _row_major(out, "th_rmsnorm out"), th_dtype(out)
    if gain.dtype != torch.float32 or not gain.is_contiguous() or gain.numel() != x.shape[1]:
        raise abi.HipBackendError("th_rmsnorm", abi.TH_ERR_INVALID, "gain must be a contiguous fp32 [K] tensor")
    d.gain = gain.data_ptr()
    d.inv_k = 1.0 / x.shape[1] if inv_k is None else inv_k
    d.eps = eps
    if out32 is not None:
        d.out32, d.ld_out32 = out32.data_ptr(), _row_major(out32, "th_rmsnorm out32")
    abi.check(lib.th_rmsnorm(C.byref(d), _stream(x)), "th_rmsnorm", kernel)
    return out


# ------------------------------------------------------------- attention
def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, *, batch: int,
                      seq_q: int, seq_kv: int, heads_q: int, heads_kv: int, head_dim: int, scale: float,
                      causal: bool, kernel: str | None = None) -> torch.Tensor:
    lib = _lib(q)
    d = abi.AttnDesc()
    d.batch, d.seq_q, d.seq_kv, d.heads_q, d.heads_kv, d.head_dim = batch, seq_q, seq_kv, heads_q, heads_kv, head_dim
    d.scale, d.causal, d.dtype = scale, 1 if causal else 0, th_dtype(q)
    for t in (k, v, out):
        if t.dtype != q.dtype:
            raise abi.HipBackendError("th_attention_prefill", abi.TH_ERR_INVALID, "q/k/v/o dtypes differ")
    d.q, d.ld_q = q.data_ptr(), _row_major(q, "attention q")
    d.k, d.ld_k = k.data_ptr(), _row_major(k, "attention k")
    d.v, d.ld_v = v.data_ptr(), _row_major(v, "attention v")
    d.o, d.ld_o = out.data_ptr(), _row_major(out, "attention o")
    abi.check(lib.th_attention_prefill(C.byref(d), _stream(q)), "th_attention_prefill", kernel)
    return out


def attention_decode_workspace_bytes(batch: int, heads_q: int, heads_kv: int, head_dim: int, max_len: int,
                                     n_split: int = 0) -> int:
    n = abi.load().th_attention_decode_workspace_bytes(batch, heads_q, heads_kv, head_dim, max_len, n_split)
    if n < 0:
        raise abi.HipBackendError("th_attention_decode_workspace_bytes", abi.TH_ERR_INVALID, "bad sizes")
    return int(n)


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, out: torch.Tensor, *,
                     scale: float, lengths: torch.Tensor | None = None, fixed_len: int = 0, n_split: int = 0,
                     workspace: torch.Tensor | None = None, kernel: str | None = None) -> torch.Tensor:
    """One query token per sequence against a [batch, max_len, heads_kv, head_dim] KV cache.

    ``q``/``out``: [batch, heads_q*head_dim]; ``lengths``: optional int32 [batch] on the device."""
    lib = _lib(q)
    B, max_len, hkv, hd = k_cache.shape
    if v_cache.shape != k_cache.shape:
        raise abi.HipBackendError("th_attention_decode", abi.TH_ERR_INVALID, "k and v caches differ in shape")
    for t in (k_cache, v_cache):
        if t.stride(3) != 1 or t.stride(2) != hd:
            raise abi.HipBackendError("th_attention_decode", abi.TH_ERR_INVALID, "cache rows must be [heads_kv][head_dim] contiguous")
    d = abi.DecodeDesc()
    d.batch, d.heads_q, d.heads_kv, d.head_dim = B, q.shape[1] // hd, hkv, hd
    d.max_len, d.n_split, d.fixed_len, d.dtype, d.scale = max_len, n_split, fixed_len, th_dtype(q), scale
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.device != q.device:
            raise abi.HipBackendError("th_attention_decode", abi.TH_ERR_INVALID, "lengths must be int32 on the device")
        d.lengths = lengths.data_ptr()
    d.q, d.ld_q = q.data_ptr(), _row_major(q, "decode q")
    d.k_cache, d.k_stride_b, d.k_stride_t = k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1)
    d.v_cache, d.v_stride_b, d.v_stride_t = v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1)
    d.o, d.ld_o = out.data_ptr(), _row_major(out, "decode o")
    if workspace is not None:
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    abi.check(lib.th_attention_decode(C.byref(d), _stream(q)), "th_attention_decode", kernel)
    return out


# --------------------------------------------------- rotary positions, paged cache
# One token's calls are shorter on the device than a Python call's bookkeeping, so these test all
# their tensors in one expression, ask the checks below for the fault only when it fails, and fill
# a descriptor in one go.
def _refuse(entry: str, message: str) -> None:
    raise abi.HipBackendError(entry, abi.TH_ERR_INVALID, message)


_ROPE, _APPEND, _ATTEND, _COPY = (abi.packer(d) for d in (abi.RopeDesc, abi.PagedAppendDesc, abi.PagedAttnDesc, abi.PageCopyDesc))


def _pack(entry: str, packer: struct.Struct, *values) -> bytes:
    try:
        return packer.pack(*values)
    except (struct.error, OverflowError) as e:   # a size past its 32 or 64 bits, a float past its range
        raise abi.HipBackendError(entry, abi.TH_ERR_INVALID, f"argument out of range: {e}") from None


def _launch(entry: str, desc: bytes, dev: int, kernel: str | None) -> None:
    """One library call on the current stream of device ``dev`` (a tensor's get_device()), whichever
    device is current."""
    if dev < 0:
        _refuse("device", "tensors on the CPU, expected a HIP device")
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return _launch(entry, desc, dev, kernel)
    lib = abi.init_device(dev)
    status = getattr(lib, entry)(desc, torch._C._cuda_getCurrentRawStream(dev))
    if status != abi.TH_OK:
        abi.check(status, entry, kernel)


def _place(dev: int) -> str:
    return "the CPU" if dev < 0 else f"device {dev}"


def _vector(t: torch.Tensor, n: int, dtype: torch.dtype, dev: int, entry: str, name: str) -> int:
    """Pointer of n contiguous values on device ``dev``."""
    if t.dtype is not dtype or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(entry, f"{name} must be {n} contiguous {dtype} values on {_place(dev)}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _rows_of(t: torch.Tensor, n: int, width: int, dtype: torch.dtype, dev: int, entry: str, name: str) -> tuple[int, int]:
    """(pointer, row stride) of a row-major [n, width] tensor on device ``dev``."""
    strides = t.stride()
    if t.dtype is not dtype or t.shape != (n, width) or (strides[1] != 1 and width != 1) or t.get_device() != dev:
        _refuse(entry, f"{name} must be a row-major [{n}, {width}] {dtype} tensor on {_place(dev)}, got {tuple(t.shape)} strides "
                       f"{strides} {t.dtype} on {t.device}")
    return t.data_ptr(), strides[0] if n > 1 else width


def _ld(strides: tuple, shape: tuple) -> int:
    """Row stride of a row-major tensor (a single row's is free, so its width)."""
    return strides[0] if shape[0] > 1 else shape[1]


def _heads(t: torch.Tensor, head_dim: int, entry: str, name: str) -> tuple[int, int]:
    """(tokens, width) of a [tokens, heads * head_dim] tensor."""
    shape = t.shape
    if len(shape) != 2 or head_dim <= 0 or shape[1] % head_dim:
        _refuse(entry, f"{name} {tuple(shape)} is no [tokens, heads * {head_dim}] tensor")
    return shape


def rope_frequencies(rot_dim: int, theta: float, *, scaling: str | None = None, factor: float = 1.0,
                     original_len: int = 0, low: float = 1.0, high: float = 32.0,
                     device: torch.device | str | int | None = None) -> torch.Tensor:
    """Radians per position of the rot_dim / 2 rotary pairs, ``theta^(-2 i / rot_dim)``, as the
    float64 tensor that :func:`rope` and :func:`paged_append` take.

    ``scaling`` stretches a context by ``factor``: "linear" divides every frequency by it; "ntk"
    raises theta to ``theta factor^(rot_dim / (rot_dim - 2))``, which keeps the fastest pair and
    divides the slowest by ``factor``; "by_parts" keeps the pairs that turn more than ``high`` times
    in ``original_len`` positions, divides those that turn less than ``low`` times and blends the
    ones between linearly in their turns (Peng et al. 2023, YaRN; its temperature is
    ``scale = 1 + 0.1 ln(factor)`` of the rotation)."""
    entry = "rope_frequencies"
    if rot_dim <= 0 or rot_dim % 2:
        _refuse(entry, f"rot_dim {rot_dim} must be even and positive")
    if not (factor > 0.0 and theta > 0.0):
        _refuse(entry, f"theta {theta} and factor {factor} must be positive")
    if scaling not in (None, "linear", "ntk", "by_parts"):
        _refuse(entry, f"unknown scaling {scaling!r}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        if rot_dim == 2:
            _refuse(entry, "ntk scaling needs at least two pairs")
        theta = theta * factor ** (rot_dim / (rot_dim - 2))
    f = theta ** (-i / rot_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        if original_len <= 0 or high <= low:
            _refuse(entry, "by_parts needs original_len and low < high")
        keep = ((f * (original_len / (2 * math.pi)) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f if device is None else f.to(torch.device("cuda", device) if isinstance(device, int) else device)


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, out: torch.Tensor, *, head_dim: int,
         interleaved: bool = False, scale: float = 1.0, inverse: bool = False, kernel: str | None = None) -> torch.Tensor:
    """Rotary positions: every head of x [tokens, heads * head_dim] (bf16 or fp32) has its first
    ``2 * len(freqs)`` dims turned by the token's own position (int32 or int64 [tokens]; angles are reduced in 64 bits).

    Pairs are dims (i, i + len(freqs)), or (2 i, 2 i + 1) with ``interleaved``; ``scale`` multiplies
    the rotated dims, the others are copied. ``inverse`` turns back: called on the gradient of the
    output with the same scale it gives the gradient of x. Like every call here it writes into
    ``out`` and records nothing for autograd: the gradient is the caller's to ask for. ``out`` may be
    x; otherwise the two must not overlap."""
    entry = "th_rope"
    shape = n, width = _heads(x, head_dim, entry, "x")
    dev, dt, pt, half = x.get_device(), x.dtype, positions.dtype, freqs.numel()
    sx, so = x.stride(), out.stride()
    if pt is not torch.int32 and pt is not torch.int64:
        _refuse(entry, f"positions are int32 or int64, got {pt}")
    if not (sx[1] == 1 and out.shape == shape and out.dtype is dt and so[1] == 1 and out.get_device() == dev
            and positions.numel() == n and positions.get_device() == dev and positions.is_contiguous()
            and freqs.dtype is torch.float64 and freqs.get_device() == dev and freqs.is_contiguous()):
        _rows_of(x, n, width, dt, dev, entry, "x")
        _rows_of(out, n, width, dt, dev, entry, "out")
        _vector(positions, n, pt, dev, entry, "positions")
        _vector(freqs, half, torch.float64, dev, entry, "freqs")
    d = _pack(entry, _ROPE, n, width // head_dim, head_dim, 2 * half, interleaved, inverse, th_dtype(dt), _DT[pt], scale,
              x.data_ptr(), _ld(sx, shape), positions.data_ptr(), freqs.data_ptr(), out.data_ptr(), _ld(so, shape))
    _launch(entry, d, dev, kernel)
    return out


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dev: int, entry: str) -> tuple:
    """(shape, strides of k, strides of v) of one layer's caches on device ``dev``."""
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not k_cache.dtype:
        _refuse(entry, "k and v caches must be [pages, page_size, heads_kv, head_dim] of one shape and dtype")
    if ks[3] != 1 or vs[3] != 1:
        _refuse(entry, "the head_dim axis of the caches must be contiguous")
    if k_cache.get_device() != dev or v_cache.get_device() != dev:
        _refuse(entry, f"the caches must be on {_place(dev)}")
    return shape, ks, vs


def _places(page_table: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor | None, n: int, dev: int, entry: str) -> tuple:
    """(rows of the table, pages per row, pointer of positions, of rows, of the table, its row stride)."""
    shape, strides = page_table.shape, page_table.stride()
    if not (len(shape) == 2 and page_table.dtype is torch.int32 and strides[1] == 1 and page_table.get_device() == dev
            and positions.dtype is torch.int32 and positions.numel() == n and positions.get_device() == dev
            and positions.is_contiguous()):
        if len(shape) != 2 or page_table.dtype is not torch.int32:
            _refuse(entry, "page_table must be int32 [rows, pages per row]")
        _rows_of(page_table, shape[0], shape[1], torch.int32, dev, entry, "page_table")
        _vector(positions, n, torch.int32, dev, entry, "positions")
    return (shape[0], shape[1], positions.data_ptr(), 0 if rows is None else _vector(rows, n, torch.int32, dev, entry, "rows"),
            page_table.data_ptr(), _ld(strides, shape))


def paged_append(k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, *, rows: torch.Tensor | None = None, freqs: torch.Tensor | None = None,
                 interleaved: bool = False, rope_scale: float = 1.0, q: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, n_invalid: torch.Tensor | None = None,
                 kernel: str | None = None) -> None:
    """Store new tokens' keys (rotated by ``freqs`` as :func:`rope` does, if given) and values in
    their cache pages, and rotate their queries ``q`` into the bf16 ``q_out``, in one launch.

    k, v: [tokens, heads_kv * head_dim] bf16 or fp32; the caches ``[pages, page_size, heads_kv,
    head_dim]`` bf16 or e4m3 (stored as ``x / scale`` of the kv head, saturated at +-448). Token t
    stands at ``positions[t]`` (int32) of row ``rows[t]`` of ``page_table`` (of row t without
    ``rows``); a negative position marks a padded token, of which nothing is written. A token
    outside the table or the cache is left out and counted in ``n_invalid`` (an int32 device
    scalar that the caller zeroes). Two tokens of a call must not share a slot."""
    entry = "th_paged_append"
    dev, dt = k.get_device(), k.dtype
    (pages, page_size, hk, hd), ks, vs = _cache(k_cache, v_cache, dev, entry)
    shape = n, width = k.shape[0], hk * hd
    n_rows, row_pages, pos, rp, tp, ldt = _places(page_table, positions, rows, n, dev, entry)
    sk, sv = k.stride(), v.stride()
    if not (k.shape == shape and v.shape == shape and v.dtype is dt and sk[1] == 1 and sv[1] == 1 and v.get_device() == dev):
        _rows_of(k, n, width, dt, dev, entry, "k")
        _rows_of(v, n, width, dt, dev, entry, "v")
    half = fp = 0
    if freqs is not None:
        half = freqs.numel()
        fp = _vector(freqs, half, torch.float64, dev, entry, "freqs")
    hq = qp = ldq = op = ldo = 0
    if q is not None:
        if q_out is None:
            _refuse(entry, "q needs a q_out")
        sq, so, shape_q = q.stride(), q_out.stride(), _heads(q, hd, entry, "q")
        if not (shape_q[0] == n and q.dtype is dt and sq[1] == 1 and q.get_device() == dev and q_out.shape == shape_q
                and q_out.dtype is torch.bfloat16 and so[1] == 1 and q_out.get_device() == dev):
            _rows_of(q, n, shape_q[1], dt, dev, entry, "q")
            _rows_of(q_out, n, shape_q[1], torch.bfloat16, dev, entry, "q_out")
        hq, qp, ldq, op, ldo = shape_q[1] // hd, q.data_ptr(), _ld(sq, shape_q), q_out.data_ptr(), _ld(so, shape_q)
    d = _pack(
        entry, _APPEND, n, hq, hk, hd, 2 * half, interleaved, th_dtype(dt), th_dtype(k_cache.dtype), page_size, n_rows, row_pages,
        pages, rope_scale, 0, pos, rp, tp, ldt, fp, qp, ldq, op, ldo, k.data_ptr(), _ld(sk, shape), v.data_ptr(), _ld(sv, shape),
        k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
        0 if k_scale is None else _vector(k_scale, hk, torch.float32, dev, entry, "k_scale"),
        0 if v_scale is None else _vector(v_scale, hk, torch.float32, dev, entry, "v_scale"),
        0 if n_invalid is None else _vector(n_invalid, 1, torch.int32, dev, entry, "n_invalid"))
    _launch(entry, d, dev, kernel)


@functools.lru_cache(maxsize=1024)
def _paged_workspace(dev: int, tokens: int, heads_q: int, heads_kv: int, head_dim: int, max_keys: int, window: int,
                     dtype: torch.dtype) -> int:
    # by the compute units of the current device: of dev, which th_init makes current, until here
    with torch.cuda.device(dev) if dev >= 0 else contextlib.nullcontext():
        lib = abi.init_device(dev) if dev >= 0 else abi.load()
        n = lib.th_paged_attention_workspace_bytes(tokens, heads_q, heads_kv, head_dim, th_dtype(dtype), max_keys, window)
    if n < 0:
        _refuse("th_paged_attention_workspace_bytes", f"tokens={tokens} heads_q={heads_q} heads_kv={heads_kv} "
                                                      f"head_dim={head_dim} max_keys={max_keys} window={window} {dtype}")
    return int(n)


def paged_attention_workspace_bytes(tokens: int, heads_q: int, heads_kv: int, head_dim: int, max_keys: int, *, window: int = 0,
                                    dtype: torch.dtype = torch.bfloat16, device: torch.device | str | int | None = None) -> int:
    """Workspace of :func:`paged_attention` over a cache of ``dtype`` whose page table has room for
    ``max_keys`` keys a row (pages per row * page_size), on ``device`` (the current one by default;
    without any, that of an MI355X). 0 where it needs none."""
    if device is None:
        dev = torch.cuda.current_device() if torch.cuda.is_available() else -1
    else:
        at = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if at.type != "cuda":
            _refuse("th_paged_attention_workspace_bytes", f"device {device} is not a HIP device")
        dev = torch.cuda.current_device() if at.index is None else at.index
    return _paged_workspace(dev, tokens, heads_q, heads_kv, head_dim, max_keys, window, dtype)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    positions: torch.Tensor, out: torch.Tensor, *, scale: float, rows: torch.Tensor | None = None,
                    window: int = 0, softcap: float = 0.0, slopes: torch.Tensor | None = None,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None, kernel: str | None = None) -> torch.Tensor:
    """One query per token against the pages of its row (see :func:`paged_append` for the caches,
    ``positions`` and ``rows``). ``q``/``out``: [tokens, heads_q * head_dim] bf16, at most 65535
    tokens; ``out`` may be ``q``. head_dim is 64 or 128, the pages hold 16 tokens or more.

    The token at position p sees the keys 0 .. p of its row, the last ``window`` of them if given.
    Scores are ``scale q . k``, capped as ``softcap tanh(s / softcap)`` if given (2^-20 to
    1024), then biased by ``-slopes[h] (p - j)`` (fp32 [heads_q]) if given. A token without keys gets zeros.
    ``workspace``: :func:`paged_attention_workspace_bytes` bytes that no concurrent call uses;
    without one the call takes it from torch's allocator. A table cut to the pages in use
    (``page_table[:, :n]``) lets short rows take a faster form."""
    entry = "th_paged_attention"
    dev = q.get_device()
    (pages, page_size, hk, hd), ks, vs = _cache(k_cache, v_cache, dev, entry)
    shape = n, width = _heads(q, hd, entry, "q")
    hq = width // hd
    if not 0 <= window < 1 << 31:
        _refuse(entry, f"window {window} out of range")
    n_rows, row_pages, pos, rp, tp, ldt = _places(page_table, positions, rows, n, dev, entry)
    sq, so = q.stride(), out.stride()
    if not (q.dtype is torch.bfloat16 and sq[1] == 1 and out.shape == shape and out.dtype is torch.bfloat16 and so[1] == 1
            and out.get_device() == dev):
        _rows_of(q, n, width, torch.bfloat16, dev, entry, "q")
        _rows_of(out, n, width, torch.bfloat16, dev, entry, "out")
    wp = wn = 0
    if workspace is not None:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            _refuse(entry, f"workspace must be a contiguous tensor on {_place(dev)}")
        wp, wn = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    elif dev >= 0:
        wn = _paged_workspace(dev, n, hq, hk, hd, row_pages * page_size, window, k_cache.dtype)
        if wn:
            workspace = torch.empty(wn, dtype=torch.uint8, device=q.device)
            wp = workspace.data_ptr()
    d = _pack(
        entry, _ATTEND, n, hq, hk, hd, th_dtype(k_cache.dtype), page_size, n_rows, row_pages, pages, window, scale, softcap, 0, pos,
        rp, tp, ldt, q.data_ptr(), _ld(sq, shape), k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2],
        0 if slopes is None else _vector(slopes, hq, torch.float32, dev, entry, "slopes"),
        0 if k_scale is None else _vector(k_scale, hk, torch.float32, dev, entry, "k_scale"),
        0 if v_scale is None else _vector(v_scale, hk, torch.float32, dev, entry, "v_scale"), out.data_ptr(), _ld(so, shape), wp, wn)
    _launch(entry, d, dev, kernel)
    return out


def copy_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, *,
               page_table: torch.Tensor | None = None, page_map: torch.Tensor | None = None,
               kernel: str | None = None) -> None:
    """Copy page ``src[i]`` onto page ``dst[i]`` (int32 device tensors) of both caches, ``[layers,
    pages, page_size, heads_kv, head_dim]`` or one layer's four axes, in every layer.

    With ``page_table`` (int32) and ``page_map`` (int32 [pages]) the table's entries p are renamed
    to ``page_map[p]`` in the same launch: a move. Pairs and entries outside the cache are left
    alone. No page may be both a source and a destination, or twice a destination."""
    entry = "th_page_copy"
    shape, dev = k_cache.shape, k_cache.get_device()
    if len(shape) not in (4, 5) or v_cache.shape != shape or v_cache.dtype is not k_cache.dtype or v_cache.get_device() != dev:
        _refuse(entry, "k and v caches must be [layers, pages, page_size, heads_kv, head_dim] of one shape, dtype and device")
    size, n = k_cache.element_size(), src.numel()
    layered, pages = len(shape) == 5, shape[-4]
    page = shape[-3] * shape[-2] * shape[-1] * size
    operands = []
    for t, name in ((k_cache, "k"), (v_cache, "v")):
        strides = t.stride()
        if strides[-3:] != (shape[-2] * shape[-1], shape[-1], 1):   # else some other order of one dense block
            run = 1
            for stride, extent in sorted(zip(strides[-3:], shape[-3:])):
                if extent != 1 and stride != run:
                    _refuse(entry, f"a page of the {name} cache must be one dense block, got strides {strides}")
                run *= extent
        operands += [t.data_ptr(), strides[0] * size if layered else 0, strides[-4] * size]
    table = (0, 0, 0, 0, 0)
    if page_table is not None:
        if page_map is None:
            _refuse(entry, "renaming a page_table needs a page_map")
        if page_table.dtype is not torch.int32 or page_table.dim() != 2:
            _refuse(entry, "page_table must be int32 [rows, pages per row]")
        rows, width = page_table.shape
        tp, ldt = _rows_of(page_table, rows, width, torch.int32, dev, entry, "page_table")
        table = (tp, ldt, rows, width, _vector(page_map, pages, torch.int32, dev, entry, "page_map"))
    d = _pack(entry, _COPY, shape[0] if layered else 1, n, pages, page, *operands,
              _vector(src, n, torch.int32, dev, entry, "src"), _vector(dst, n, torch.int32, dev, entry, "dst"), *table)
    _launch(entry, d, dev, kernel)


# ------------------------------------------------- microscaled linear layers
# Tensors in blocks of 32 columns that share a power of two (OCP microscaling): ``codes``, uint8
# [rows, 16 ceil(cols / 32)] of e2m1 pairs or float8_e4m3fn [rows, 32 ceil(cols / 32)], and ``scales``,
# uint8 or float8_e8m0fnu [rows, ceil(cols / 32)]. Rows may be strided (codes: by whole 16 bytes).
_MXQ, _MXD, _MXN, _MXG = (abi.packer(d) for d in (abi.MxQuantizeDesc, abi.MxDequantizeDesc, abi.MxRmsNormDesc, abi.MxGemmDesc))
_E4M3, _BYTE, _E8M0 = torch.float8_e4m3fn, torch.uint8, torch.float8_e8m0fnu


def mx_empty(rows: int, cols: int, *, bits: int, device: torch.device | str | int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (``bits`` 8: e4m3, 4: e2m1 pairs) and scales of a [rows, cols] tensor, not written yet."""
    if bits not in (4, 8) or rows < 0 or cols <= 0:
        _refuse("mx_empty", f"no blocks of {bits} bits for [{rows}, {cols}]")
    n, dev = -(-cols // 32), torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    return (torch.empty(rows, n * 4 * bits, dtype=_E4M3 if bits == 8 else _BYTE, device=dev),
            torch.empty(rows, n, dtype=_BYTE, device=dev))


def _mx(codes: torch.Tensor, scales: torch.Tensor, rows: int, blocks: int, dev: int, entry: str, name: str) -> tuple:
    """(th_dtype of the codes, their pointer and row stride, the scales' pointer and row stride)."""
    dt, width = codes.dtype, 32 * blocks if codes.dtype is _E4M3 else 16 * blocks
    if ((dt is _E4M3 or dt is _BYTE) and (scales.dtype is _BYTE or scales.dtype is _E8M0) and codes.get_device() == dev
            and scales.get_device() == dev and codes.shape == (rows, width) and scales.shape == (rows, blocks)):
        form = abi.TH_F8E4M3 if dt is _E4M3 else abi.TH_F4E2M1
        if codes.is_contiguous() and scales.is_contiguous():
            return form, codes.data_ptr(), width, scales.data_ptr(), blocks
        sc, ss = codes.stride(), scales.stride()
        if sc[1] == 1 and (ss[1] == 1 or blocks == 1):
            return form, codes.data_ptr(), sc[0] if rows > 1 else width, scales.data_ptr(), ss[0] if rows > 1 else blocks
    _refuse(entry, f"{name}: codes {tuple(codes.shape)} {dt} strides {codes.stride()} on {codes.device} with scales {tuple(scales.shape)} "
                   f"{scales.dtype} strides {scales.stride()} on {scales.device} are no {rows} rows of {blocks} blocks on {_place(dev)}")


def _matrix(t: torch.Tensor, entry: str, name: str) -> tuple:
    """(rows, cols, th_dtype, pointer, row stride) of a row-major bf16 or fp32 matrix."""
    shape, dt = t.shape, t.dtype
    if len(shape) == 2 and (dt is torch.bfloat16 or dt is torch.float32):
        rows, cols = shape
        if t.is_contiguous():
            return rows, cols, abi.TH_BF16 if dt is torch.bfloat16 else abi.TH_F32, t.data_ptr(), cols
        strides = t.stride()
        if strides[1] == 1 or cols == 1:
            return rows, cols, abi.TH_BF16 if dt is torch.bfloat16 else abi.TH_F32, t.data_ptr(), strides[0] if rows > 1 else cols
    _refuse(entry, f"{name} must be a row-major bf16 or fp32 matrix, got {tuple(shape)} strides {t.stride()} {dt}")


def mx_quantize(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, *, kernel: str | None = None) -> None:
    """Quantise x [rows, cols] (bf16 or fp32) to blocks of 32 columns: scale 2^(s - 127) with s =
    floor(log2(max |x|)) - emax + 127 held to 0 .. 254 (emax 8 for e4m3 codes, 2 for e2m1), elements
    x over the scale, rounded to nearest even and held to the largest (448, 6). A block with an
    infinity or a NaN becomes NaN (s = 255). The last block is filled up with zeros."""
    entry = "th_mx_quantize"
    rows, cols, xt, xp, ldx = _matrix(x, entry, "x")
    dev = x.get_device()
    mt, cp, ldc, sp, lds = _mx(codes, scales, rows, -(-cols // 32), dev, entry, "x's blocks")
    _launch(entry, _pack(entry, _MXQ, rows, cols, xt, mt, 0, xp, ldx, cp, ldc, sp, lds), dev, kernel)


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor, *, kernel: str | None = None) -> torch.Tensor:
    """The values that codes and scales stand for, into out [rows, cols] (bf16 or fp32, rounded once)."""
    entry = "th_mx_dequantize"
    rows, cols, ot, op, ldo = _matrix(out, entry, "out")
    dev = out.get_device()
    mt, cp, ldc, sp, lds = _mx(codes, scales, rows, -(-cols // 32), dev, entry, "out's blocks")
    _launch(entry, _pack(entry, _MXD, rows, cols, mt, ot, 0, cp, ldc, sp, lds, op, ldo), dev, kernel)
    return out


def mx_rmsnorm(x: torch.Tensor, gain: torch.Tensor, eps: float, codes: torch.Tensor, scales: torch.Tensor, *,
               residual: torch.Tensor | None = None, sum_out: torch.Tensor | None = None, kernel: str | None = None) -> None:
    """h = x + residual (rounded to their type), y = h / sqrt(mean(h^2) + eps) * gain per row, y
    quantised as :func:`mx_quantize` does. x, residual and sum_out: [rows, cols] of one type (bf16 or
    fp32), cols at most 65536; gain fp32 [cols]. ``sum_out`` gets h; it may be x or residual."""
    entry = "th_mx_rmsnorm"
    rows, cols, xt, xp, ldx = _matrix(x, entry, "x")
    dev, dt = x.get_device(), x.dtype
    mt, cp, ldc, sp, lds = _mx(codes, scales, rows, -(-cols // 32), dev, entry, "the blocks")
    rp = ldr = hp = ldh = 0
    if residual is not None:
        rp, ldr = _rows_of(residual, rows, cols, dt, dev, entry, "residual")
    if sum_out is not None:
        hp, ldh = _rows_of(sum_out, rows, cols, dt, dev, entry, "sum_out")
    d = _pack(entry, _MXN, rows, cols, xt, mt, eps, xp, ldx, rp, ldr, hp, ldh,
              _vector(gain, cols, torch.float32, dev, entry, "gain"), cp, ldc, sp, lds)
    _launch(entry, d, dev, kernel)


def _mx_gemm_desc(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: torch.Tensor,
                  residual: torch.Tensor | None) -> tuple[bytes, int]:
    entry = "th_mx_gemm"
    rows, outs, ot, op, ldo = _matrix(out, entry, "out")
    if len(a_scales.shape) != 2:
        _refuse(entry, "scales are [rows, blocks]")
    dev, blocks = out.get_device(), a_scales.shape[1]
    at, ap, lda, asp, ldas = _mx(a, a_scales, rows, blocks, dev, entry, "a")
    wt, wp, ldw, wsp, ldws = _mx(w, w_scales, outs, blocks, dev, entry, "w")
    if wt != abi.TH_F4E2M1:
        _refuse(entry, "w must be uint8 codes of e2m1 pairs")
    rp = ldr = 0
    if residual is not None:
        rp, ldr = _rows_of(residual, rows, outs, out.dtype, dev, entry, "residual")
    return _pack(entry, _MXG, rows, outs, blocks, at, ot, 0, 0, ap, lda, asp, ldas, wp, ldw, wsp, ldws, rp, ldr, op, ldo,
                 0, 0), dev


def _mx_swiglu_desc(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, codes: torch.Tensor,
                    scales: torch.Tensor) -> tuple[bytes, int]:
    entry = "th_mx_gemm"
    if len(scales.shape) != 2 or len(a_scales.shape) != 2:
        _refuse(entry, "scales are [rows, blocks]")
    (rows, out_blocks), blocks, dev = scales.shape, a_scales.shape[1], codes.get_device()
    at, ap, lda, asp, ldas = _mx(a, a_scales, rows, blocks, dev, entry, "a")
    wt, wp, ldw, wsp, ldws = _mx(w, w_scales, 64 * out_blocks, blocks, dev, entry, "w")
    ct, cp, ldc, sp, lds = _mx(codes, scales, rows, out_blocks, dev, entry, "the result's blocks")
    if wt != abi.TH_F4E2M1:
        _refuse(entry, "w must be uint8 codes of e2m1 pairs")
    return _pack(entry, _MXG, rows, 32 * out_blocks, blocks, at, ct, 1, 0, ap, lda, asp, ldas, wp, ldw, wsp, ldws, 0, 0, cp, ldc,
                 sp, lds), dev


def mx_gemm(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: torch.Tensor, *,
            residual: torch.Tensor | None = None, kernel: str | None = None) -> torch.Tensor:
    """out[m, n] = sum_k a[m, k] w[n, k] (+ residual[m, n]): activations in e4m3 or e2m1 blocks,
    weights in e2m1 blocks ([outs, k], one row an output column), fp32 sums, out and residual bf16 or
    fp32 of one type. ``residual`` may be ``out``. k is whole blocks: what :func:`mx_quantize` filled up with zeros adds
    nothing."""
    _launch("th_mx_gemm", *_mx_gemm_desc(a, a_scales, w, w_scales, out, residual), kernel)
    return out


def mx_swiglu(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, codes: torch.Tensor,
              scales: torch.Tensor, *, kernel: str | None = None) -> None:
    """silu(a wg^T) * (a wu^T), quantised as :func:`mx_quantize` does: the input of a down projection.
    w holds the gate's rows and then the up projection's, [2 outs, k] in e2m1 blocks; codes and scales
    are of [rows, outs], outs a multiple of 32. The products are not rounded before."""
    _launch("th_mx_gemm", *_mx_swiglu_desc(a, a_scales, w, w_scales, codes, scales), kernel)


def _mx_form(desc: bytes, dev: int) -> tuple[int, bool]:
    form = (C.c_int32 * 2)()
    with torch.cuda.device(dev) if dev >= 0 else contextlib.nullcontext():
        abi.check(abi.load().th_mx_gemm_form(desc, form), "th_mx_gemm_form")
    return form[0], bool(form[1])


def mx_gemm_form(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: torch.Tensor, *,
                 residual: torch.Tensor | None = None) -> tuple[int, bool]:
    """(abi.MX_*, whether the scales are loaded byte by byte): what :func:`mx_gemm` runs for these tensors, which may
    also be on the CPU (then for 256 compute units)."""
    return _mx_form(*_mx_gemm_desc(a, a_scales, w, w_scales, out, residual))


def mx_swiglu_form(a: torch.Tensor, a_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, codes: torch.Tensor,
                   scales: torch.Tensor) -> tuple[int, bool]:
    """The same of :func:`mx_swiglu`."""
    return _mx_form(*_mx_swiglu_desc(a, a_scales, w, w_scales, codes, scales))


# ----------------------------------------------------------- epilogue VM
def epilogue_vm(M: int, N: int, operands: list[tuple[torch.Tensor, bool]], ops: list[tuple], outs: list[tuple[torch.Tensor, int]],
                n_slots: int, workspace: torch.Tensor, kernel: str | None = None) -> None:
    """``operands``: (tensor, is_column); ``ops``: (code, dst, a, b, scalar, mode);
    ``outs``: (tensor, slot)."""
    ref = workspace
    lib = _lib(ref)
    if len(operands) > abi.VM_MAX_IN or len(ops) > abi.VM_MAX_OPS or len(outs) > abi.VM_MAX_OUT:
        raise abi.HipBackendError("th_epilogue_vm", abi.TH_ERR_UNSUPPORTED, "epilogue program too large")
    if workspace.dtype != torch.float32 or workspace.numel() < n_slots * M * N:
        raise abi.HipBackendError("th_epilogue_vm", abi.TH_ERR_INVALID, "workspace too small")
    d = abi.VmDesc()
    d.M, d.N = M, N
    d.n_in, d.n_ops, d.n_out, d.n_slots = len(operands), len(ops), len(outs), n_slots
    for i, (t, col) in enumerate(operands):
        d.in_[i].ptr, d.in_[i].ld, d.in_[i].dtype, d.in_[i].column = t.data_ptr(), t.stride(0), th_dtype(t), 1 if col else 0
    for i, (code, dst, a, b, scalar, mode) in enumerate(ops):
        o = d.ops[i]
        o.code, o.dst, o.a, o.b, o.scalar, o.mode = code, dst, a, b, scalar, mode
    for i, (t, slot) in enumerate(outs):
        d.out[i].ptr, d.out[i].ld, d.out[i].dtype, d.out[i].slot = t.data_ptr(), _row_major(t, "vm out"), th_dtype(t), slot
    d.workspace = workspace.data_ptr()
    abi.check(lib.th_epilogue_vm(C.byref(d), _stream(ref)), "th_epilogue_vm", kernel)


# ------------------------------------------------------------------- SSD
def ssd_workspace_bytes(batch: int, seq: int, heads: int, head_dim: int, state_dim: int, chunk: int,
                        ngroups: int | None = None) -> int:
    """Workspace of th_ssd_chunked: the minimum, or with ``ngroups`` the size that also holds
    the chunks' shared G^T tiles (formed once per B/C group instead of once per head)."""
    if ngroups is None:
        return int(abi.load().th_ssd_workspace_bytes(batch, seq, heads, head_dim, state_dim, chunk))
    return int(abi.load().th_ssd_gtile_workspace_bytes(batch, seq, heads, head_dim, state_dim, chunk, ngroups))


def ssd_chunked(*, x, b, c, dt, out, workspace, batch, seq, heads, head_dim, state_dim, ngroups, chunk, A=None, D=None,
                cum=None, dt_stride=1, dskip=None, gate=None, out32=None, y_gain=None, rs_parts=None,
                kernel: str | None = None) -> None:
    """One th_ssd_chunked launch. ``y_gain`` (fp32 [heads * head_dim]) stores y times that
    per-column gain and writes, into ``rs_parts`` (fp32 [batch * seq, heads * head_dim / 32]),
    the sums of squares of y before it per token and 32 columns: an RMSNorm whose row scale
    the consuming th_gemm applies (its ``rs_parts``)."""
    lib = _lib(x)
    d = abi.SsdDesc()
    d.batch, d.seq, d.heads, d.head_dim, d.state_dim, d.ngroups, d.chunk = batch, seq, heads, head_dim, state_dim, ngroups, chunk
    d.dtype = th_dtype(x)
    for t in (b, c, dt) + ((cum,) if cum is not None else ()) + ((dskip,) if dskip is not None else ()):
        if t.dtype != x.dtype:
            raise abi.HipBackendError("th_ssd_chunked", abi.TH_ERR_INVALID, "scan operands must share one dtype", kernel)
    d.x, d.ld_x = x.data_ptr(), _row_major(x, "ssd x")
    d.b, d.ld_b = b.data_ptr(), _row_major(b, "ssd b")
    d.c, d.ld_c = c.data_ptr(), _row_major(c, "ssd c")
    d.dt, d.ld_dt, d.dt_stride = dt.data_ptr(), _row_major(dt, "ssd dt"), dt_stride
    if cum is not None:
        d.cum, d.ld_cum = cum.data_ptr(), _row_major(cum, "ssd cum")
    if A is not None:
        d.A = A.data_ptr()
    if D is not None:
        d.D = D.data_ptr()
    if dskip is not None:
        d.dskip, d.ld_dskip = dskip.data_ptr(), _row_major(dskip, "ssd dskip")
    if gate is not None:
        d.gate, d.ld_gate, d.gate_dtype = gate.data_ptr(), _row_major(gate, "ssd gate"), th_dtype(gate)
    d.y, d.ld_y, d.y_dtype = out.data_ptr(), _row_major(out, "ssd y"), th_dtype(out)
    if out32 is not None:
        d.y32, d.ld_y32 = out32.data_ptr(), _row_major(out32, "ssd y32")
    if y_gain is not None:
        if y_gain.dtype != torch.float32 or not y_gain.is_contiguous() or y_gain.numel() != heads * head_dim:
            raise abi.HipBackendError("th_ssd_chunked", abi.TH_ERR_INVALID, "y_gain must be contiguous fp32 [H*P]", kernel)
        if rs_parts is None or rs_parts.dtype != torch.float32:
            raise abi.HipBackendError("th_ssd_chunked", abi.TH_ERR_INVALID, "y_gain needs fp32 rs_parts", kernel)
        d.y_gain = y_gain.data_ptr()
        d.rs_parts, d.ld_rs_parts = rs_parts.data_ptr(), _row_major(rs_parts, "ssd rs_parts")
    d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    abi.check(lib.th_ssd_chunked(C.byref(d), _stream(x)), "th_ssd_chunked", kernel)


def conv1d_causal(x, w, out, *, batch: int, seq: int, activation: str | None, out32=None, kernel: str | None = None) -> None:
    lib = _lib(x)
    if w.dtype != torch.float32 or not w.is_contiguous():
        raise abi.HipBackendError("th_conv1d_causal", abi.TH_ERR_INVALID, "weights must be contiguous fp32 [C, K]", kernel)
    d = abi.ConvDesc()
    d.batch, d.seq, d.width, d.kernel = batch, seq, w.shape[0], w.shape[1]
    d.activation = 1 if activation == "silu" else 0
    d.x_dtype, d.y_dtype = th_dtype(x), th_dtype(out)
    d.x, d.ld_x = x.data_ptr(), _row_major(x, "conv x")
    d.w = w.data_ptr()
    d.y, d.ld_y = out.data_ptr(), _row_major(out, "conv y")
    if out32 is not None:
        d.y32, d.ld_y32 = out32.data_ptr(), _row_major(out32, "conv y32")
    abi.check(lib.th_conv1d_causal(C.byref(d), _stream(x)), "th_conv1d_causal", kernel)


def embedding(table: torch.Tensor, ids: torch.Tensor, out: torch.Tensor, *, out32: torch.Tensor | None = None,
              n_invalid: torch.Tensor | None = None, kernel: str | None = None) -> None:
    """out[t] = table[ids[t]] (th_embedding). Rows of ids outside [0, vocab) are
    written as zeros and counted in ``n_invalid`` (an int32 device scalar) if given."""
    lib = _lib(table)
    if ids.dtype not in (torch.int64, torch.int32) or not ids.is_contiguous():
        raise abi.HipBackendError("th_embedding", abi.TH_ERR_INVALID, "ids must be contiguous int64 or int32", kernel)
    if out.dtype != table.dtype or out.shape[-1] != table.shape[1] or out.numel() != ids.numel() * table.shape[1]:
        raise abi.HipBackendError("th_embedding", abi.TH_ERR_INVALID,
                                  f"out {tuple(out.shape)} {out.dtype} does not match ids {tuple(ids.shape)} "
                                  f"x table {tuple(table.shape)} {table.dtype}", kernel)
    if n_invalid is not None and (n_invalid.dtype != torch.int32 or n_invalid.device != table.device):
        raise abi.HipBackendError("th_embedding", abi.TH_ERR_INVALID, "n_invalid must be an int32 device tensor", kernel)
    out2 = out.reshape(-1, table.shape[1]) if out.dim() != 2 else out
    d = abi.EmbeddingDesc()
    d.tokens, d.dim, d.vocab = ids.numel(), table.shape[1], table.shape[0]
    d.dtype, d.ids_dtype = th_dtype(table), th_dtype(ids)
    d.table, d.ld_table = table.data_ptr(), _row_major(table, "embedding table")
    d.ids = ids.data_ptr()
    d.out, d.ld_out = out2.data_ptr(), _row_major(out2, "embedding out")
    if out32 is not None:
        o32 = out32.reshape(-1, table.shape[1]) if out32.dim() != 2 else out32
        d.out32, d.ld_out32 = o32.data_ptr(), _row_major(o32, "embedding out32")
    if n_invalid is not None:
        d.n_invalid = n_invalid.data_ptr()
    abi.check(lib.th_embedding(C.byref(d), _stream(table)), "th_embedding", kernel)
