"""Host-side mirror of Mference's Swift operator surface over the C ABI.

Class and method names follow Sources/Mference/Kernels/** (Swift camelCase
turned into snake_case); a command buffer becomes a HIP stream, an
(MTLBuffer, offset) pair becomes a torch tensor (device memory only: torch is
the allocator and stream provider, every computation is libmfmoe's).
Argument errors raise MfError carrying the mf_status the C ABI returned.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from struct import Struct
from typing import Optional, Sequence
from weakref import ref as _ref

import numpy as np
import torch

from . import _capi
from ._capi import (ACT_GELU, ACT_GELU_TANH, ACT_NONE, ACT_SILU, BF16_EXPERTS_ROWS, BITS_2, BITS_4, BITS_8, BITS_TERNARY,
                    GATE_CHANNEL, GATE_ELEMENT, GATE_NONE, GATE_ROW, GROUP_SIZE, MAX_ADAPTER_RANK, MAX_ADAPTER_TARGETS, MAX_ADAPTERS, MAX_EXPERTS,
                    MAX_ROWS, MAX_TOKENS, MAX_TOPK, ROUTER_FULL_SOFTMAX, ROUTER_TOPK_SOFTMAX, SAME_POSITIONS, ExpertOffsets, MfError, check)

__all__ = [
    "MetalContext", "QuantizedTensor", "Quantization", "DequantInt4GEMV", "DequantInt4GEMVMultiX",
    "Elementwise", "FamilyRouters", "SharedExpertInt4", "MPPPrefillInt4QMM", "MoEExpertOffsets", "MoE", "MoELayerWeights",
    "PrefillMoEGrouping", "PrefillTokenExpertPair", "MfError", "BITS_2", "BITS_4", "BITS_TERNARY",
    "ROUTER_TOPK_SOFTMAX", "ROUTER_FULL_SOFTMAX", "bf16_tensor", "bf16_bits",
    "AdapterGrouping", "AdapterPlan", "LowRankAdapters", "BlockNorm", "GATE_NONE", "GATE_ROW", "GATE_ELEMENT", "GATE_CHANNEL",
    "Projection", "HeadNorms", "Bf16Experts", "ACT_NONE", "ACT_SILU", "ACT_GELU_TANH", "ACT_GELU",
]

MoEExpertOffsets = ExpertOffsets


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("libmfmoe operates on device memory; got a CPU tensor")
    return t.data_ptr()


# the current stream's handle without a torch.cuda.Stream object around it (3.1 -> 0.2 us per call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_this_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream(stream) -> int:
    if stream is None:
        if _raw_stream is None or _this_device is None:
            return torch.cuda.current_stream().cuda_stream
        return _raw_stream(_this_device())
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


def bf16_tensor(bits: np.ndarray, device="cuda") -> torch.Tensor:
    """uint16 bf16 bit patterns (host) -> torch.bfloat16 tensor on `device`."""
    a = np.ascontiguousarray(bits, dtype=np.uint16)
    return torch.from_numpy(a.view(np.int16)).to(device).view(torch.bfloat16)


def bf16_bits(t: torch.Tensor) -> np.ndarray:
    """torch.bfloat16 tensor -> uint16 bit patterns on the host."""
    return t.detach().contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


class MetalContext:
    """Device + kernel state every operator is built from
    (Infrastructure/Metal/MetalContext.swift:45-65)."""

    def __init__(self, device: int = 0):
        self._h = C.c_void_p()
        check(_capi.lib().mf_ctx_create(device, C.byref(self._h)))
        self.device = torch.device("cuda", device)

    @property
    def handle(self):
        return self._h

    def close(self):
        if self._h:
            _capi.lib().mf_ctx_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


@dataclass
class QuantizedTensor:
    """rows x n group-quantized tensor in device memory
    (Quantization.Int4AffineRow for every row, Quantization.swift:34-46)."""
    packed: torch.Tensor            # uint8 [rows, n*bits/8]
    scales: torch.Tensor            # bf16 [rows, n/64]
    biases: Optional[torch.Tensor]  # bf16 [rows, n/64]; None for ternary
    bits: int
    rows: int
    n: int

    def c(self) -> _capi.QTensor:
        return _capi.QTensor(_ptr(self.packed), _ptr(self.scales), _ptr(self.biases))

    @classmethod
    def from_host(cls, packed: np.ndarray, scales: np.ndarray, biases: Optional[np.ndarray],
                  bits: int, rows: int, n: int, device="cuda") -> "QuantizedTensor":
        return cls(torch.from_numpy(np.ascontiguousarray(packed)).to(device),
                   bf16_tensor(scales, device),
                   None if biases is None else bf16_tensor(biases, device), bits, rows, n)


class Quantization:
    """Infrastructure/ModelIO/Quantization.swift:3 on device."""
    group_size = GROUP_SIZE

    def __init__(self, context: MetalContext):
        self.context = context

    def quantize_affine(self, w: torch.Tensor, bits: int = BITS_4, stream=None) -> QuantizedTensor:
        """quantizeInt4Affine (Quantization.swift:50-102) for every row of w (fp32)."""
        if w.dtype != torch.float32 or w.dim() != 2:
            raise ValueError("w must be a 2-D float32 tensor")
        w = w.contiguous()
        rows, n = w.shape
        store = {BITS_8: 8, BITS_4: 4}.get(bits, 2)   # 8-bit: quantizeInt8Affine (Quantization.swift:135-176)
        packed = torch.empty((rows, n * store // 8), dtype=torch.uint8, device=w.device)
        scales = torch.empty((rows, n // GROUP_SIZE), dtype=torch.bfloat16, device=w.device)
        biases = torch.empty_like(scales)
        check(_capi.lib().mf_quantize_affine(self.context.handle, _stream(stream), _ptr(w), rows, n,
                                             bits, _ptr(packed), _ptr(scales), _ptr(biases)),
              self.context.handle)
        return QuantizedTensor(packed, scales, biases, bits, rows, n)

    def dequantize(self, q: QuantizedTensor, stream=None) -> torch.Tensor:
        """dequantizeInt4Affine (Quantization.swift:104-119): fp32 [rows, n]."""
        out = torch.empty((q.rows, q.n), dtype=torch.float32, device=q.packed.device)
        check(_capi.lib().mf_dequantize(self.context.handle, _stream(stream), q.c(), q.rows, q.n,
                                        q.bits, _ptr(out)), self.context.handle)
        return out


class DequantInt4GEMV:
    """Kernels/Quant/DequantInt4GEMV.swift:57-103 (any supported bit width)."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode(self, weights: QuantizedTensor, x: torch.Tensor, y: torch.Tensor, m: int, n: int,
               output_float32: bool = False, stream=None, t: int = 1) -> None:
        check(_capi.lib().mf_gemv(self.context.handle, _stream(stream), weights.c(), weights.bits,
                                  _ptr(x), _ptr(y), m, n, t, 1 if output_float32 else 0),
              self.context.handle)


class DequantInt4GEMVMultiX(DequantInt4GEMV):
    """Kernels/Quant/DequantInt4GEMVMultiX.swift:48-82: x [t, n], y [t, m], t <= 8."""
    max_tokens = MAX_TOKENS

    def encode(self, weights: QuantizedTensor, x: torch.Tensor, y: torch.Tensor, m: int, n: int,
               t: int, output_float32: bool = False, stream=None) -> None:
        super().encode(weights, x, y, m, n, output_float32, stream, t)


class MPPPrefillInt4QMM:
    """Kernels/TensorCore/MPPPrefillInt4QMM.swift:34-78: y[m, n] = x[m, k] . deq(W[n, k])^T for many
    rows.  `encode` returns the path taken, like the reference's `Path`."""
    tile_m, tile_n, tile_k = 64, 32, GROUP_SIZE

    def __init__(self, context: MetalContext):
        self.context = context
        self._ws = None

    def workspace_bytes(self, m: int, n: int, k: int) -> int:
        return int(_capi.lib().mf_qmm_workspace_bytes(m, n, k))

    def encode(self, weights: QuantizedTensor, x: torch.Tensor, y: torch.Tensor, m: int, n: int, k: int,
               workspace: Optional[torch.Tensor] = None, stream=None) -> str:
        if workspace is None:
            need = self.workspace_bytes(m, n, k)
            if self._ws is None or self._ws.numel() < need:
                self._ws = torch.empty(max(need, 256), dtype=torch.uint8, device=x.device)
            workspace = self._ws
        ws_bytes = workspace.numel() * workspace.element_size()
        # the reference's guard conditions (MPPPrefillInt4QMM.swift:43-55) give "unavailable"; a path that
        # ran is named for the kernel that ran it
        path = _capi.lib().mf_qmm_path(weights.c(), weights.bits, _ptr(x), _ptr(y), m, n, k, _ptr(workspace), ws_bytes)
        if path < 0:
            return "unavailable"
        check(_capi.lib().mf_qmm(self.context.handle, _stream(stream), weights.c(), weights.bits, _ptr(x), _ptr(y),
                                 m, n, k, 1 if y.dtype == torch.float32 else 0, _ptr(workspace), ws_bytes),
              self.context.handle)
        return self.PATHS[path]

    PATHS = {1: "affine-matrix-core-bf16", 2: "affine-rows-gemv"}


class Elementwise:
    """Kernels/Primitives/Elementwise.swift:60-87."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode_silu_mul(self, gate, up, out, count: int, stream=None):
        check(_capi.lib().mf_silu_mul(self.context.handle, _stream(stream), _ptr(gate), _ptr(up),
                                      _ptr(out), count), self.context.handle)

    def encode_sigmoid_scalar_mul(self, y, gate, count: int, rows: int = 1, stream=None):
        check(_capi.lib().mf_sigmoid_scalar_mul(self.context.handle, _stream(stream), _ptr(y),
                                                _ptr(gate), count, rows), self.context.handle)

    def encode_residual_add(self, hidden, delta, count: int, stream=None):
        check(_capi.lib().mf_residual_add(self.context.handle, _stream(stream), _ptr(hidden),
                                          _ptr(delta), count), self.context.handle)


class RMSNorm:
    """Kernels/Primitives/RMSNorm.swift:52-64 (`encodeBF16W`), with the residual add that
    precedes it in the runner folded into the same launch when `delta` is given."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode_bf16w(self, x, weight, out, d: int, eps: float, t: int = 1, delta=None, stream=None):
        """x [t, d] bf16 is the hidden state: updated in place by `delta` when given"""
        check(_capi.lib().mf_residual_rmsnorm(self.context.handle, _stream(stream), _ptr(x), _ptr(delta),
                                              _ptr(weight), _ptr(out), d, t, C.c_float(eps)),
              self.context.handle)


def _on(context: MetalContext, stream) -> int:
    """the stream's handle; the current stream of the context's device (not of the current device) when none is given"""
    if stream is None:
        if _raw_stream is None:
            return torch.cuda.current_stream(context.device).cuda_stream
        return _raw_stream(context.device.index)
    return stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else int(stream)


def _stream_object(context: MetalContext, stream) -> torch.cuda.Stream:
    """torch's object for a stream that a call was given (an ExternalStream of handle 0 would be one of torch's own streams)"""
    if isinstance(stream, torch.cuda.Stream):
        return stream
    handle = int(stream)
    return torch.cuda.ExternalStream(handle, context.device) if handle else torch.cuda.default_stream(context.device)


def _taken_on(context: MetalContext, stream, take):
    """take(), a buffer from torch's allocator, as memory of the stream that a call was given: a block that was freed on the current
    stream may still be in use there"""
    if stream is None or _on(context, stream) == _on(context, None):
        return take()
    with torch.cuda.stream(_stream_object(context, stream)):
        return take()


def _address(t: torch.Tensor, what: str, dtype, device: int) -> int:
    """the address of a tensor that lies on the context's device and has the type asked for"""
    if t.dtype is not dtype or t.get_device() != device:
        if not t.is_cuda:
            raise ValueError(f"libmfmoe operates on device memory; {what} is a CPU tensor")
        if t.dtype is not dtype:
            raise ValueError(f"{what} must be {dtype}, not {t.dtype}")
        raise ValueError(f"{what} lies on another device than the context")
    return t.data_ptr()


_U32 = (1 << 32) - 1  # the largest number the library's arguments hold


def _row_stride(t: torch.Tensor, what: str, shape) -> int:
    """elements from row to row of a tensor of this shape [rows, width] whose rows are contiguous"""
    if t.shape != shape:
        raise MfError(-2, f"{what} is {tuple(t.shape)}, not {tuple(shape)}")
    rows, width = shape
    if t.is_contiguous() or rows == 1 and (width == 1 or t.stride(1) == 1):
        return width
    if width > 1 and t.stride(1) != 1:
        raise MfError(-1, f"the rows of {what} must be contiguous")
    stride = t.stride(0)
    if stride < width:
        raise MfError(-2, f"the rows of {what} overlap")
    if stride > _U32:
        raise MfError(-2, f"the rows of {what} are {stride} elements apart")
    return stride


def _rows(t: torch.Tensor, what: str, dtype, device: int, shape):
    """the address and the row stride of a tensor of this type and shape [rows, width] on the context's device"""
    if t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous():  # nothing more to ask: 0.3 us less a tensor
        return t.data_ptr(), shape[1]
    return _address(t, what, dtype, device), _row_stride(t, what, shape)


def _vector(t: torch.Tensor, what: str, dtype, device: int, shape) -> int:
    """the address of a contiguous vector of this type and shape [size] on the context's device"""
    if t.shape != shape or not t.is_contiguous():
        raise MfError(-2, f"{what} must be a contiguous vector of {shape[0]}")
    return _address(t, what, dtype, device)


class AdapterPlan:
    """What AdapterGrouping.encode fills: the rows of a batch in the order of their adapters (mf_adapter_group)."""

    def __init__(self, t: int, num_adapters: int, words: torch.Tensor):
        need = int(_capi.lib().mf_adapter_plan_bytes(t, num_adapters)) if 0 <= t <= MAX_ROWS and 0 < num_adapters <= MAX_ADAPTERS else 0
        if need == 0 or words.dtype is not torch.int32 or words.dim() != 1 or not words.is_contiguous() or words.numel() * 4 < need:
            raise MfError(-1, f"t={t}, num_adapters={num_adapters}: {need // 4} contiguous int32 words")
        self.t, self.num_adapters, self.words = t, num_adapters, words
        self.rows = words[:t]                               # int32 [t]: row numbers, stably sorted, rows without an adapter last
        self.offsets = words[t:t + num_adapters + 1]        # int32: where every adapter's rows start; then the rows without one

    def _address_for(self, t: int, num_adapters: int, device: int) -> int:
        """the address of its words, for a call of t rows and a pool of num_adapters on this device"""
        if self.t != t or self.num_adapters != num_adapters:
            raise MfError(-2, f"the plan is one of {self.t} rows and {self.num_adapters} adapters")
        return _address(self.words, "the plan", torch.int32, device)


class AdapterGrouping:
    """mf_adapter_group: the rows of a batch by adapter, on the device, once for all projections of a step (what
    MoE.encode_group is for routes).  A row whose adapter is not in [0, num_adapters) has none."""

    def __init__(self, context: MetalContext, num_adapters: int):
        if not 1 <= num_adapters <= MAX_ADAPTERS:
            raise MfError(-1, f"num_adapters={num_adapters}")
        self.context, self.num_adapters = context, num_adapters

    def plan(self, t: int) -> AdapterPlan:
        """room for the plan of t rows"""
        need = int(_capi.lib().mf_adapter_plan_bytes(t, self.num_adapters)) if 0 <= t <= MAX_ROWS else 0
        return AdapterPlan(t, self.num_adapters, torch.empty(need // 4, dtype=torch.int32, device=self.context.device if need else "cpu"))

    def encode(self, adapter_of_row: torch.Tensor, plan: Optional[AdapterPlan] = None, stream=None) -> AdapterPlan:
        """adapter_of_row int32 [t]"""
        ctx = self.context
        device, t = ctx.device.index, adapter_of_row.numel()
        ids = _vector(adapter_of_row, "adapter_of_row", torch.int32, device, (t,))
        if plan is None:
            plan = _taken_on(ctx, stream, lambda: self.plan(t))
            if stream is not None:  # the caller may go on with it on the current stream
                plan.words.record_stream(torch.cuda.current_stream(ctx.device))
        words = plan._address_for(t, self.num_adapters, device)
        check(_capi.lib().mf_adapter_group(ctx.handle, _on(ctx, stream), ids, t, self.num_adapters, words, plan.words.numel() * 4), ctx.handle)
        return plan


class LowRankAdapters:
    """mf_adapter_apply: the low-rank corrections of many requests, added to the results of projections that read the same x
    (DequantInt4GEMV, MPPPrefillInt4QMM, SharedExpertInt4 leave them).  a[s] bf16 [num_adapters, rank, n] and
    b[s] bf16 [num_adapters, m_s, rank] for every projection s; scales float32 and ranks int32 [num_adapters]
    (below 0: 0; past rank: rank)."""

    def __init__(self, context: MetalContext, a: Sequence[torch.Tensor], b: Sequence[torch.Tensor],
                 scales: Optional[torch.Tensor] = None, ranks: Optional[torch.Tensor] = None):
        a, b = ([a] if isinstance(a, torch.Tensor) else list(a)), ([b] if isinstance(b, torch.Tensor) else list(b))
        if not 1 <= len(a) <= MAX_ADAPTER_TARGETS or len(a) != len(b):
            raise MfError(-1, f"{len(a)} tensors a, {len(b)} tensors b")
        if a[0].dim() != 3:
            raise MfError(-2, "a must be [num_adapters, rank, n]")
        self.context = context
        self.num_adapters, self.rank, self.n = a[0].shape
        self.a, self.b, self.scales, self.ranks = a, b, scales, ranks  # kept: the pool's addresses stay valid
        device = context.device.index
        self._fixed = []  # a, b and m of every projection
        for wa, wb in zip(a, b):
            if wa.shape != a[0].shape or wb.dim() != 3 or wb.shape[0] != self.num_adapters or wb.shape[2] != self.rank:
                raise MfError(-2, f"a {tuple(wa.shape)}, b {tuple(wb.shape)}")
            if not (wa.is_contiguous() and wb.is_contiguous()):
                raise MfError(-1, "the adapter pool must be contiguous")
            self._fixed.append((_address(wa, "a", torch.bfloat16, device), _address(wb, "b", torch.bfloat16, device), wb.shape[1]))
        self.ms = [wb.shape[1] for wb in b]
        self._pack = Struct("@" + "PPPII" * len(a)).pack  # mf_adapter_target [len(a)]
        self.pool = _capi.AdapterPool(self.num_adapters, self.rank, self.n, None, None)
        for name, v, dtype in (("ranks", ranks, torch.int32), ("scales", scales, torch.float32)):
            if v is not None:
                setattr(self.pool, name, _vector(v, name, dtype, device, (self.num_adapters,)))
        if max(self.num_adapters, self.rank, self.n) > _U32 or max(self.ms) > 1 << 28 or self.workspace_bytes(1) == 0:
            raise MfError(-2, f"num_adapters={self.num_adapters} rank={self.rank} n={self.n} m={self.ms}")

    def workspace_bytes(self, t: int) -> int:
        """bytes that a call of t rows, or fewer, asks for"""
        return int(_capi.lib().mf_adapter_workspace_bytes(C.byref(self.pool), len(self._fixed), t)) if 0 <= t <= MAX_ROWS else 0

    def encode(self, x: torch.Tensor, adapter_of_row: torch.Tensor, ys, plan: Optional[AdapterPlan] = None,
               workspace: Optional[torch.Tensor] = None, stream=None) -> None:
        """ys[s][i] += scales[a] * b[s][a] @ (a[s][a] @ x[i]), a = adapter_of_row[i]; rows without an adapter stay as they
        are.  x bf16 [t, n]; ys[s] bf16 or float32 [t, m_s], all of one type.  plan: AdapterGrouping's of the same rows, for
        batches that mix many adapters.  Without a workspace the call takes one of its own from torch's allocator."""
        ctx = self.context
        device = ctx.device.index
        if isinstance(ys, torch.Tensor):
            ys = (ys,)
        if len(ys) != len(self._fixed):
            raise MfError(-2, f"{len(ys)} results for {len(self._fixed)} projections")
        t = adapter_of_row.numel()
        ids = _vector(adapter_of_row, "adapter_of_row", torch.int32, device, (t,))
        x_ptr, x_stride = _rows(x, "x", torch.bfloat16, device, (t, self.n))
        dtype = ys[0].dtype
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            raise ValueError(f"the results must be bfloat16 or float32, not {dtype}")
        targets = []
        for (a, b, m), y in zip(self._fixed, ys):
            y_ptr, y_stride = _rows(y, "y", dtype, device, (t, m))
            targets += (a, b, y_ptr, m, y_stride)
        words = None if plan is None else plan._address_for(t, self.num_adapters, device)
        if t == 0:
            return
        if t > MAX_ROWS:
            raise MfError(-1, f"t={t} rows are more than one call takes")
        if workspace is None:
            workspace = _taken_on(ctx, stream, lambda: torch.empty(self.workspace_bytes(t), dtype=torch.uint8, device=ctx.device))
        elif not workspace.is_contiguous():
            raise MfError(-1, "the workspace must be contiguous")
        elif workspace.get_device() != device:
            raise ValueError("the workspace lies on another device than the context")
        check(_capi.lib().mf_adapter_apply(ctx.handle, _on(ctx, stream), C.byref(self.pool), self._pack(*targets), len(ys), x_ptr, x_stride, ids, t,
                                           1 if dtype is torch.float32 else 0, words, workspace.data_ptr(), workspace.nbytes), ctx.handle)


class BlockNorm:
    """mf_block_norm: what stands between two blocks of a layer, in one launch -- the norm behind the block, its gate and scale,
    the residual add, the norm in front of the next block (RMSNorm and Elementwise.encode_residual_add are its two halves)."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode(self, hidden: torch.Tensor, delta: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               pre_weight: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, gate_kind: int = GATE_NONE, eps: float = 1e-6,
               post_eps: Optional[float] = None, residual_scale: float = 1.0, branch_scale: float = 1.0,
               weight_bias: float = 0.0, stream=None) -> None:
        """hidden bf16 [t, d] is updated in place: residual_scale * hidden + branch_scale * gate * norm(delta); out gets its norm.
        gate: GATE_ROW [t] or [t, 1] and GATE_ELEMENT [t, d] go through a sigmoid, GATE_CHANNEL [d] is taken as it is."""
        ctx, bf16 = self.context, torch.bfloat16
        device, shape = ctx.device.index, hidden.shape
        if len(shape) != 2:
            raise MfError(-2, "hidden must be [t, d]")
        t, d = shape
        if t > MAX_ROWS or d > _U32:
            raise MfError(-1 if t > MAX_ROWS else -2, f"t={t} rows of d={d} are more than one call takes")
        channels = (d,)
        h_ptr, h_stride = _rows(hidden, "hidden", bf16, device, shape)
        d_ptr = d_stride = f32 = o_ptr = o_stride = g_ptr = g_stride = pre = post = 0
        if delta is not None:
            f32 = 1 if delta.dtype is torch.float32 else 0
            d_ptr, d_stride = _rows(delta, "delta", torch.float32 if f32 else bf16, device, shape)
        elif residual_scale != 1.0:
            raise MfError(-1, f"residual_scale={residual_scale} without a block output: the stream is only read")
        if out is not None:
            o_ptr, o_stride = _rows(out, "out", bf16, device, shape)
        if pre_weight is not None:
            pre = _vector(pre_weight, "pre_weight", bf16, device, channels)
        if post_weight is not None:
            post = _vector(post_weight, "post_weight", bf16, device, channels)
        if gate is not None:
            g_ptr = _address(gate, "gate", bf16, device)
            if gate_kind == GATE_ROW:
                if gate.numel() != t or gate.dim() not in (1, 2) or gate.shape[0] != t:
                    raise MfError(-2, f"the gate must be one logit for each of {t} rows")
                g_stride = gate.stride(0) if t > 1 else 1
                if g_stride == 0 and t > 1:  # 0 means "not given" to the library
                    raise MfError(-2, "a gate of one logit a row cannot be an expanded one")
                if g_stride > _U32:
                    raise MfError(-2, f"the logits of the gate are {g_stride} elements apart")
            elif gate_kind == GATE_ELEMENT:
                g_stride = _row_stride(gate, "gate", shape)
            else:
                _vector(gate, "gate", bf16, device, channels)
        args = self._pack(h_ptr, d_ptr, g_ptr, post, pre, o_ptr, d, t, h_stride, d_stride, g_stride, o_stride, f32, gate_kind,
                          eps if post_eps is None else post_eps, eps, residual_scale, branch_scale, weight_bias)
        check(_capi.lib().mf_block_norm(ctx.handle, _on(ctx, stream), args), ctx.handle)

    _pack = Struct("@6P6I2i5f4x").pack  # mf_block_norm_args


def _workspace(context: MetalContext, workspace: Optional[torch.Tensor], need: int, stream) -> tuple:
    """address and size of a call's workspace: the caller's, or one of the call's stream from torch's allocator (kept by the tensor returned)"""
    if workspace is None:
        if need == 0:
            return None, 0, None
        workspace = _taken_on(context, stream, lambda: torch.empty(need, dtype=torch.uint8, device=context.device))
    elif not workspace.is_contiguous():
        raise MfError(-1, "the workspace must be contiguous")
    elif workspace.get_device() != context.device.index:
        raise ValueError("the workspace lies on another device than the context")
    return workspace.data_ptr(), workspace.nbytes, workspace


class Projection:
    """mf_project: y = residual + act(x W^T + bias) of a weight kept in 16 bits (what DequantInt4GEMV and MPPPrefillInt4QMM are for
    quantized ones), or with `gated` residual + act(x G^T + bias_g) * (x U^T + bias_u), the weight holding G's rows and then U's."""

    def __init__(self, context: MetalContext, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: int = ACT_NONE,
                 gated: bool = False):
        """weight bf16 [m, n], gated [2 m, n]; its rows are contiguous"""
        if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0 or gated and weight.shape[0] % 2:
            raise MfError(-2, f"weight {tuple(weight.shape)}")
        if not ACT_NONE <= activation <= ACT_GELU:
            raise MfError(-1, f"activation={activation}")
        rows, self.n = weight.shape
        self.m = rows // 2 if gated else rows
        if self.m > 1 << 24 or self.n > 1 << 22:
            raise MfError(-2, f"m={self.m} n={self.n}")
        self.context, self.gated, self.activation = context, bool(gated), activation
        self.weight, self.bias = weight, bias  # kept: the addresses stay valid
        device = context.device.index
        self._w, self._w_stride = _rows(weight, "weight", torch.bfloat16, device, weight.shape)
        self._bias = None if bias is None else _vector(bias, "bias", torch.bfloat16, device, (rows,))

    def workspace_bytes(self, t: int) -> int:
        """bytes that a call of t rows, or fewer, asks for"""
        return int(_capi.lib().mf_project_workspace_bytes(self.m, self.n, t, 1 if self.gated else 0)) if 0 <= t <= MAX_ROWS else 0

    def encode(self, x: torch.Tensor, y: torch.Tensor, residual: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
               stream=None) -> None:
        """x bf16 [t, n]; y bf16 or float32 [t, m]; residual of y's type, y itself for an update in place.  Without a workspace the call
        takes what it needs from torch's allocator."""
        ctx, m = self.context, self.m
        device, t = ctx.device.index, x.shape[0]
        dtype = y.dtype
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            raise ValueError(f"y must be bfloat16 or float32, not {dtype}")
        x_ptr, x_stride = _rows(x, "x", torch.bfloat16, device, (t, self.n))
        y_ptr, y_stride = _rows(y, "y", dtype, device, (t, m))
        r_ptr = r_stride = 0
        if residual is not None:
            r_ptr, r_stride = _rows(residual, "residual", dtype, device, (t, m))
        if t == 0:
            return
        if t > MAX_ROWS:
            raise MfError(-1, f"t={t} rows are more than one call takes")
        ws, size, _kept = _workspace(ctx, workspace, 0 if workspace is not None else self.workspace_bytes(t), stream)
        args = self._pack(x_ptr, self._w, self._bias or 0, r_ptr, y_ptr, t, m, self.n, x_stride, self._w_stride, r_stride, y_stride,
                          1 if dtype is torch.float32 else 0, 1 if self.gated else 0, self.activation)
        check(_capi.lib().mf_project(ctx.handle, _on(ctx, stream), args, ws, size), ctx.handle)

    _pack = Struct("@5P7I3i0P").pack  # mf_project_args


class HeadNorms:
    """mf_head_norms: the norms of query and key heads and their rotation by positions of one or several axes, in one launch (RMSNorm is
    the norm of whole rows)."""

    def __init__(self, context: MetalContext, head_dim: int, inv_freq: Optional[torch.Tensor] = None, axis_of_pair: Optional[torch.Tensor] = None,
                 interleaved: bool = False, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 weight_bias: float = 0.0, rotation_scale: float = 1.0):
        """inv_freq float32 [pairs]: the first 2 * pairs elements of a head are rotated (None: nothing is); axis_of_pair uint8 [pairs]:
        whose position turns a pair (None: the first axis; axes_of_sections makes one); interleaved: a pair is two neighbours,
        else one element of either half; weights bf16 [head_dim] (None: no norm)."""
        if not 1 <= head_dim <= 1024:
            raise MfError(-2, f"head_dim={head_dim}")
        self.context, self.head_dim, self.interleaved = context, head_dim, bool(interleaved)
        self.inv_freq, self.axis_of_pair, self.q_weight, self.k_weight = inv_freq, axis_of_pair, q_weight, k_weight  # kept: the addresses stay valid
        device, pairs = context.device.index, 0 if inv_freq is None else inv_freq.numel()
        if 2 * pairs > head_dim or inv_freq is not None and pairs == 0:
            raise MfError(-2, f"{pairs} pairs in heads of {head_dim}")
        if axis_of_pair is not None and inv_freq is None:
            raise MfError(-1, "axis_of_pair without inv_freq")
        self.rotary_dim = 2 * pairs
        self._tables = [0 if v is None else _vector(v, name, dtype, device, (n,)) for v, name, dtype, n in (
            (q_weight, "q_weight", torch.bfloat16, head_dim), (k_weight, "k_weight", torch.bfloat16, head_dim),
            (inv_freq, "inv_freq", torch.float32, pairs), (axis_of_pair, "axis_of_pair", torch.uint8, pairs))]
        self._numbers = (eps, weight_bias, rotation_scale)
        self._named = None if axis_of_pair is not None else 1

    def _axes_named(self) -> int:
        """how many axes the table names (numbers of 8 and more are none); read once, by the first call that gives the positions of one"""
        if self._named is None:
            if self.axis_of_pair.is_cuda and torch.cuda.is_current_stream_capturing():
                raise MfError(-1, "positions [t] beside a table of axes that no call has read yet, while a graph is captured: give [axes, t]")
            self._named = 1 + max((axis for axis in self.axis_of_pair.tolist() if axis < 8), default=0)
        return self._named

    @staticmethod
    def axes_of_sections(sections: Sequence[int], turns: bool = False, device="cuda") -> torch.Tensor:
        """axis_of_pair for axes that own so many pairs each: one section behind the other, or by turns while an axis has pairs left"""
        left, table = [int(n) for n in sections], []
        if not 1 <= len(left) <= 8 or min(left) < 0:
            raise MfError(-2, f"sections {left}")
        if not turns:
            table = [axis for axis, n in enumerate(left) for _ in range(n)]
        while turns and any(left):
            for axis, n in enumerate(left):
                if n:
                    table.append(axis)
                    left[axis] -= 1
        return torch.tensor(table, dtype=torch.uint8, device=device)

    def _heads(self, x: torch.Tensor, what: str, device: int, t: int, heads: int):
        """address, row stride and head stride (0: as the library takes it by itself) of a tensor [t, heads, head_dim]"""
        if x.shape != (t, heads, self.head_dim):
            raise MfError(-2, f"{what} is {tuple(x.shape)}, not {(t, heads, self.head_dim)}")
        row, head, element = x.stride()
        if self.head_dim > 1 and element != 1:
            raise MfError(-1, f"the heads of {what} must be contiguous")
        row, head = (row if t > 1 else 0), (head if heads > 1 else self.head_dim)
        if t > 1 and row < 1 or head < 1:
            raise MfError(-2, f"the rows of {what} overlap")
        if row > _U32 or head > _U32:
            raise MfError(-2, f"the rows of {what} are {max(row, head)} elements apart")
        return _address(x, what, torch.bfloat16, device), row, head

    def encode(self, q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None, stream=None) -> None:
        """q bf16 [t, heads, head_dim], k [t, kv heads, head_dim], views of a wider buffer or of any order of rows and heads among them;
        in place without q_out / k_out.  positions int32 [axes, t], one row expanded over the axes where they share it; or [t] where no more
        than one axis is named.  A pair whose axis is none of them is not turned."""
        ctx = self.context
        device = ctx.device.index
        if q.dim() != 3 or k is not None and k.dim() != 3:
            raise MfError(-2, "heads must be [t, heads, head_dim]")
        if k is None and k_out is not None:
            raise MfError(-1, "k_out without k")
        t = q.shape[0]
        if t > MAX_ROWS:
            raise MfError(-1, f"t={t} rows are more than one call takes")
        wq, wk, freq, axes_table = self._tables
        words = []
        for x, out, what, weight in ((q, q_out, "q", wq), (k, k_out, "k", wk)):
            if x is None:
                words += (0, 0, 0, 0, 0, 0, 0, 0)
                continue
            heads = x.shape[1]
            if heads > 65535:
                raise MfError(-2, f"{heads} heads")
            ptr, row, head = self._heads(x, what, device, t, heads)
            o_ptr, o_row, o_head = (ptr, row, head) if out is None else self._heads(out, what + "_out", device, t, heads)
            words += (ptr, o_ptr, weight, heads, row, head, o_row, o_head)
        if (positions is None) != (self.rotary_dim == 0):
            raise MfError(-1, "positions and inv_freq come together")
        at = axes = p_stride = 0
        if positions is not None:
            shape = positions.shape
            if len(shape) not in (1, 2) or shape[-1] != t:
                raise MfError(-2, f"positions {tuple(shape)} for {t} rows")
            axes, p_stride = 1, t
            if len(shape) == 2:
                axes = shape[0]
                if not 1 <= axes <= 8:
                    raise MfError(-2, f"{axes} axes")
                if axes > 1:
                    p_stride = positions.stride(0)
                    if p_stride == 0:
                        p_stride = SAME_POSITIONS
                    elif not t <= p_stride < SAME_POSITIONS:
                        raise MfError(-2, "the positions of the axes overlap, or are too far apart")
            elif self._axes_named() > 1:
                raise MfError(-2, f"positions of one axis for a table of {self._axes_named()}: give [axes, t] (a row expanded over the axes where they share it)")
            if t > 1 and positions.stride(-1) != 1:
                raise MfError(-1, "the positions of an axis must be contiguous")
            at = _address(positions, "positions", torch.int32, device)
        if t == 0:
            return
        args = self._pack(*words, at, freq, axes_table, t, self.head_dim, self.rotary_dim, axes, p_stride, 1 if self.interleaved else 0, *self._numbers)
        check(_capi.lib().mf_head_norms(ctx.handle, _on(ctx, stream), args), ctx.handle)

    _pack = Struct("@3P5I4x3P5I4x3P5Ii3f0P").pack  # mf_head_norms_args


class Bf16Experts:
    """mf_bf16_experts: a layer of experts kept in 16 bits for a few tokens, the routed ones and the shared one, in two launches, three beyond eight tokens (what
    MoE.encode_decode_layer is for quantized experts; the routing comes from MoE.encode_router or one of FamilyRouters)."""
    max_tokens = BF16_EXPERTS_ROWS

    def __init__(self, context: MetalContext, gate_up: torch.Tensor, down: torch.Tensor, top_k: int, gate_up_bias: Optional[torch.Tensor] = None,
                 down_bias: Optional[torch.Tensor] = None, shared_gate_up: Optional[torch.Tensor] = None, shared_down: Optional[torch.Tensor] = None,
                 shared_gate: Optional[torch.Tensor] = None, activation: int = ACT_SILU):
        """gate_up bf16 [experts, 2 f, d] (gate rows first), down [experts, d, f], biases [experts, 2 f] and [experts, d];
        shared_gate_up [2 shared_f, d], shared_down [d, shared_f], shared_gate [d] (its sigmoid scales the shared expert)"""
        if gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[1] % 2 or down.shape != (gate_up.shape[0], gate_up.shape[2], gate_up.shape[1] // 2):
            raise MfError(-2, f"gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)}")
        if (shared_gate_up is None) != (shared_down is None) or shared_gate is not None and shared_down is None:
            raise MfError(-1, "a shared expert has both of its matrices")
        experts, f2, d = gate_up.shape
        fs = 0 if shared_down is None else shared_down.shape[-1]
        if not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= MAX_TOPK or any(v % 8 or not 8 <= v <= 1 << 20 for v in (d, f2 // 2, fs or 8)):
            raise MfError(-2, f"experts={experts} top_k={top_k} d={d} f={f2 // 2} shared_f={fs}")
        self.context, self.num_experts, self.top_k, self.d, self.f, self.shared_f = context, experts, top_k, d, f2 // 2, fs
        device, bf16 = context.device.index, torch.bfloat16
        self.tensors = (gate_up, down, gate_up_bias, down_bias, shared_gate_up, shared_down, shared_gate)  # kept: the addresses stay valid
        shapes = ((experts, f2, d), (experts, d, f2 // 2), (experts, f2), (experts, d), (2 * fs, d), (d, fs), (d,))
        names = ("gate_up", "down", "gate_up_bias", "down_bias", "shared_gate_up", "shared_down", "shared_gate")
        self.pool = _capi.Bf16ExpertPool(num_experts=experts, top_k=top_k, d=d, f=f2 // 2, shared_f=fs, activation=activation)
        for name, v, shape in zip(names, self.tensors, shapes):
            if v is not None:
                if v.shape != shape or not v.is_contiguous():
                    raise MfError(-2, f"{name} must be contiguous {shape}")
                setattr(self.pool, name, _address(v, name, bf16, device))
        if not ACT_NONE <= activation <= ACT_GELU:
            raise MfError(-1, f"activation={activation}")
        self._pool = C.byref(self.pool)

    def workspace_bytes(self, t: int) -> int:
        """bytes that a call of t rows, or fewer, asks for"""
        return int(_capi.lib().mf_bf16_experts_workspace_bytes(self._pool, t)) if 0 <= t <= BF16_EXPERTS_ROWS else 0

    def encode(self, x: torch.Tensor, indices: torch.Tensor, routing_weights: torch.Tensor, y: torch.Tensor,
               residual: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None, stream=None) -> None:
        """x bf16 [t, d], t <= max_tokens; indices int32 and routing_weights float32 [t, top_k]; y bf16 [t, d]; residual bf16 [t, d], y
        itself for an update in place.  Without a workspace the call takes one from torch's allocator."""
        ctx = self.context
        device, t = ctx.device.index, x.shape[0]
        shape, routes = (t, self.d), (t, self.top_k)
        x_ptr, x_stride = _rows(x, "x", torch.bfloat16, device, shape)
        y_ptr, y_stride = _rows(y, "y", torch.bfloat16, device, shape)
        r_ptr = r_stride = 0
        if residual is not None:
            r_ptr, r_stride = _rows(residual, "residual", torch.bfloat16, device, shape)
        idx, w = _vector(indices, "indices", torch.int32, device, routes), _vector(routing_weights, "routing_weights", torch.float32, device, routes)
        if t == 0:
            return
        if t > BF16_EXPERTS_ROWS:
            raise MfError(-10, f"t={t}: at most {BF16_EXPERTS_ROWS} rows a call")
        ws, size, _kept = _workspace(ctx, workspace, 0 if workspace is not None else self.workspace_bytes(t), stream)
        check(_capi.lib().mf_bf16_experts(ctx.handle, _on(ctx, stream), self._pool, x_ptr, x_stride, idx, w, r_ptr, r_stride, t, y_ptr, y_stride, ws, size),
              ctx.handle)


class SharedExpertInt4:
    """Kernels/MoE/SharedExpertInt4.swift:70-165 (also the dense SwiGLU MLP)."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode(self, x: torch.Tensor, gate: QuantizedTensor, up: QuantizedTensor,
               down: QuantizedTensor, y: torch.Tensor, scratch_act: torch.Tensor, t: int = 1,
               stream=None) -> None:
        if not (gate.rows == up.rows and gate.n == up.n and down.rows == gate.n
                and down.n == gate.rows):
            raise MfError(-2, f"gate=({gate.rows},{gate.n}) up=({up.rows},{up.n}) "
                              f"down=({down.rows},{down.n})")
        check(_capi.lib().mf_shared_expert(
            self.context.handle, _stream(stream), _ptr(x), gate.c(), up.c(), down.c(), gate.bits,
            gate.n, gate.rows, t, _ptr(y), _ptr(scratch_act),
            scratch_act.numel() * scratch_act.element_size()), self.context.handle)

    def encode_adapted(self, x: torch.Tensor, gate: QuantizedTensor, up: QuantizedTensor, down: QuantizedTensor,
                       y: torch.Tensor, gate_up_adapters: LowRankAdapters, down_adapters: LowRankAdapters,
                       adapter_of_row: torch.Tensor, plan: Optional[AdapterPlan] = None, stream=None) -> None:
        """The MLP with an adapter beside each of its three projections (the same adapter of a row in all of them): the
        projections by themselves (mf_qmm), LowRankAdapters on their results, silu(gate) * up in between.  No counterpart in
        the reference.  x bf16 [t, d], y bf16 [t, d]; both pools hold the same number of adapters; buffers come from torch's
        allocator.  What does not fit together is refused in front of the first launch, y as it was."""
        if not (gate.rows == up.rows and gate.n == up.n and down.rows == gate.n and down.n == gate.rows):
            raise MfError(-2, f"gate=({gate.rows},{gate.n}) up=({up.rows},{up.n}) down=({down.rows},{down.n})")
        t, d, f = x.shape[0], gate.n, gate.rows
        if not (x.is_contiguous() and y.is_contiguous()) or x.shape != (t, d) or y.shape != (t, d):
            raise MfError(-2, f"x {tuple(x.shape)} and y {tuple(y.shape)} must be contiguous rows of {d}")
        for adapters, n, ms in ((gate_up_adapters, d, [f, f]), (down_adapters, f, [d])):  # in front of the first launch
            if adapters.n != n or adapters.ms != ms:
                raise MfError(-2, f"adapters of {adapters.n} to {adapters.ms} beside projections of {n} to {ms}")
            if adapters.context.device != self.context.device:
                raise ValueError("the adapters lie on another device than the context")
        if gate_up_adapters.num_adapters != down_adapters.num_adapters:  # a row's adapter is the same one in all three projections
            raise MfError(-2, f"{gate_up_adapters.num_adapters} adapters for gate and up, {down_adapters.num_adapters} for down")
        device = self.context.device.index
        _address(x, "x", torch.bfloat16, device), _address(y, "y", torch.bfloat16, device)
        _vector(adapter_of_row, "adapter_of_row", torch.int32, device, (t,))
        if plan is not None:
            plan._address_for(t, down_adapters.num_adapters, device)
        if t == 0:
            return
        if t * f >= 1 << 31:
            raise MfError(-1, f"t={t} rows of f={f} are more than one call takes")
        on = torch.cuda.current_stream(self.context.device) if stream is None else _stream_object(self.context, stream)
        with torch.cuda.stream(on):  # so that the allocator knows the stream of the buffers
            g, u, act = (torch.empty((t, f), dtype=torch.bfloat16, device=x.device) for _ in range(3))
            qmm, elementwise = MPPPrefillInt4QMM(self.context), Elementwise(self.context)
            need = max(qmm.workspace_bytes(t, f, d), qmm.workspace_bytes(t, d, f), 256)
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
            lib, handle, ws, s = _capi.lib(), self.context.handle, workspace.data_ptr(), on.cuda_stream
            projections = [(w.c(), w.bits, src.data_ptr(), out.data_ptr(), t, w.rows, w.n) for w, src, out in ((gate, x, g), (up, x, u), (down, act, y))]
            if any(lib.mf_qmm_path(*p, ws, need) < 0 for p in projections):
                raise MfError(-1, "a projection refuses its operands")
            for p in projections[:2]:
                check(lib.mf_qmm(handle, s, *p, 0, ws, need), handle)
            gate_up_adapters.encode(x, adapter_of_row, (g, u), plan=plan, stream=on)
            elementwise.encode_silu_mul(g, u, act, t * f, stream=on)
            check(lib.mf_qmm(handle, s, *projections[2], 0, ws, need), handle)
            down_adapters.encode(act, adapter_of_row, y, plan=plan, stream=on)

    @staticmethod
    def scratch_bytes(d: int, f: int, t: int) -> int:
        """bytes of scratch the call can use for t rows (the matrix-core path beyond 8 rows)"""
        return int(_capi.lib().mf_shared_expert_scratch_bytes(d, f, t))

    def encode_static(self, x: torch.Tensor, gate: QuantizedTensor, up: QuantizedTensor,
                      down: QuantizedTensor, y: torch.Tensor, t: int = 1, stream=None) -> None:
        """The same operator for callers that cannot allocate and bring no scratch: the
        activations go through the library's built-in device array (mf_shared_expert_static;
        t * f <= STATIC_ACT_ELEMS, calls on one GPU must not overlap)."""
        if not (gate.rows == up.rows and gate.n == up.n and down.rows == gate.n
                and down.n == gate.rows):
            raise MfError(-2, f"gate=({gate.rows},{gate.n}) up=({up.rows},{up.n}) "
                              f"down=({down.rows},{down.n})")
        check(_capi.lib().mf_shared_expert_static(
            self.context.handle, _stream(stream), _ptr(x), gate.c(), up.c(), down.c(), gate.bits,
            gate.n, gate.rows, t, _ptr(y)), self.context.handle)


class SharedExpertInt8:
    """Kernels/MoE/SharedExpertInt8.swift:78-181: the dense MLP on 8-bit affine tensors, GELU (tanh form) by
    default, SiLU with silu_activation (the reference's siluActivation)."""

    def __init__(self, context: MetalContext, silu_activation: bool = False):
        self.context = context
        self.silu_activation = silu_activation

    def encode(self, x: torch.Tensor, gate: QuantizedTensor, up: QuantizedTensor, down: QuantizedTensor,
               y: torch.Tensor, scratch_act: torch.Tensor, t: int = 1, stream=None) -> None:
        if not (gate.rows == up.rows and gate.n == up.n and down.rows == gate.n and down.n == gate.rows):
            raise MfError(-2, f"gate=({gate.rows},{gate.n}) up=({up.rows},{up.n}) down=({down.rows},{down.n})")
        check(_capi.lib().mf_shared_expert_int8(
            self.context.handle, _stream(stream), _ptr(x), gate.c(), up.c(), down.c(), gate.n, gate.rows, t,
            1 if self.silu_activation else 0, _ptr(y), _ptr(scratch_act),
            scratch_act.numel() * scratch_act.element_size()), self.context.handle)


class FamilyRouters:
    """The family-specific routers of the reference's operator classes, stand-alone: every call
    runs the router GEMV into the caller's fp32 `logits` buffer [t, rows] and then the selection.
    Routing weights are fp32 (the reference narrows them to fp16)."""

    def __init__(self, context: MetalContext):
        self.context = context

    def encode_router_top_k(self, weights, hidden, correction_bias, out_indices, out_weights,
                            num_experts: int, d: int, route_scale: float, logits, top_k: int = 6,
                            t: int = 1, x_stride: Optional[int] = None, stream=None):
        """MoEDeepseekV4.encodeRouterTopK (MoEDeepseekV4.swift:92-124): sqrtsoftplus selection."""
        check(_capi.lib().mf_router_sqrtsoftplus(
            self.context.handle, _stream(stream), _ptr(weights), _ptr(hidden), t,
            d if x_stride is None else x_stride, num_experts, d, top_k, _ptr(correction_bias),
            route_scale, _ptr(logits), _ptr(out_indices), _ptr(out_weights)), self.context.handle)

    def encode_router_hash_weights(self, weights, hidden, indices, out_weights, num_experts: int,
                                   d: int, route_scale: float, logits, top_k: int = 6, t: int = 1,
                                   x_stride: Optional[int] = None, stream=None):
        """MoEDeepseekV4.encodeRouterHashWeights (MoEDeepseekV4.swift:126-151)."""
        check(_capi.lib().mf_router_hash_weights(
            self.context.handle, _stream(stream), _ptr(weights), _ptr(hidden), t,
            d if x_stride is None else x_stride, num_experts, d, top_k, _ptr(indices), route_scale,
            _ptr(logits), _ptr(out_weights)), self.context.handle)

    def encode_router_inkling(self, weights, hidden, gate_bias, global_scale, out_indices,
                              out_weights, gammas_out, num_routed: int, num_shared: int, top_k: int,
                              route_scale: float, d: int, logits, t: int = 1,
                              x_stride: Optional[int] = None, stream=None):
        """InklingKernels.encodeRouter / encodeRouterPrefill (InklingKernels.swift:377-476)."""
        check(_capi.lib().mf_router_inkling(
            self.context.handle, _stream(stream), _ptr(weights), _ptr(hidden), t,
            d if x_stride is None else x_stride, num_routed, num_shared, d, top_k, _ptr(gate_bias),
            _ptr(global_scale), route_scale, _ptr(logits), _ptr(out_indices), _ptr(out_weights),
            _ptr(gammas_out)), self.context.handle)

    def encode_router_gemma4(self, weights, scales, biases, hidden, effective_scale,
                             per_expert_scale, out_indices, out_weights, num_experts: int, d: int,
                             top_k: int, logits, t: int = 1, x_stride: Optional[int] = None,
                             stream=None):
        """MoE.encodeRouterGemma4 (MoE.swift:153-202): 8-bit affine router rows."""
        check(_capi.lib().mf_router_gemma4(
            self.context.handle, _stream(stream), _ptr(weights), _ptr(scales), _ptr(biases),
            _ptr(hidden), t, d if x_stride is None else x_stride, _ptr(effective_scale),
            _ptr(per_expert_scale), num_experts, d, top_k, _ptr(logits), _ptr(out_indices),
            _ptr(out_weights)), self.context.handle)


def expert_blob_layout(d: int, f: int, bits: int = BITS_4, align: int = 256, repacked: bool = False):
    """(offsets, blob_bytes, stride) of one routed expert in the reference's blob order
    (RepackPlanner.swift:544-712, ModelExpertIO.swift:20-35): mf_expert_blob_layout, or with
    `repacked` mf_expert_blob_layout_repacked -- the byte layout of a packed_experts file, which for
    ternary experts also carries the negated-scale bias tables (RepackPlanner.swift:619-640)."""
    off = ExpertOffsets()
    blob, stride = C.c_size_t(0), C.c_size_t(0)
    fn = _capi.lib().mf_expert_blob_layout_repacked if repacked else _capi.lib().mf_expert_blob_layout
    check(fn(d, f, bits, align, C.byref(off), C.byref(blob), C.byref(stride)))
    return off, blob.value, stride.value


@dataclass
class MoELayerWeights:
    """Everything one MoE layer reads, resident in device memory."""
    router_w: torch.Tensor                 # bf16 [e, d]
    experts: torch.Tensor                  # uint8 [e, stride]
    offsets: ExpertOffsets
    shared: Optional[Sequence[QuantizedTensor]] = None  # gate, up, down
    w_sg: Optional[torch.Tensor] = None    # bf16 [d]
    w_sg_q8: Optional[QuantizedTensor] = None  # the scalar gate as an 8-bit affine row [1, d] (replaces w_sg)
    experts_tiled: Optional[torch.Tensor] = None  # uint8 [e, stride]: the pool in the prefill matmul's order (MoE.tile_experts)

    def _tensors(self):
        """every tensor the C struct points at, in a fixed order"""
        t = (self.router_w, self.experts, self.w_sg, self.experts_tiled)
        for q in self.shared or ():
            t += (q.packed, q.scales, q.biases)
        q = self.w_sg_q8
        return t if q is None else t + (q.packed, q.scales, q.biases)

    def c(self) -> _capi.LayerWeights:
        """The C struct of the layer.  It is kept between calls and is the same while every tensor named lies where it lay
        and the pools keep their shape (a field, or a tensor's storage, may be replaced at any time).  No tensor is held for
        it: one that the layer no longer names is the caller's to free, and an address is not trusted beyond its tensor."""
        now = self._tensors()
        key = [0 if t is None else t.data_ptr() for t in now]
        key += self.experts.stride()
        if self.experts_tiled is not None:
            key += (*self.experts.shape, *self.experts_tiled.shape, self.experts_tiled.stride(0))
        key.append(bytes(self.offsets))
        kept = self.__dict__.get("_kept")
        if kept is not None and kept[0] == key:
            return kept[1]
        struct = self._build()
        kept = [key, struct]
        kept.append([_ref(t, lambda _, k=kept: k.__setitem__(0, None)) for t in now if t is not None])
        self.__dict__["_kept"] = kept
        return struct

    def __getstate__(self):  # a copy makes its own C struct
        return {k: v for k, v in self.__dict__.items() if k != "_kept"}

    def _build(self) -> _capi.LayerWeights:
        if self.experts.ndim != 2 or self.experts.stride(1) != 1:
            # a 1-D pool would make stride(0) one byte: every expert would read expert 0's bytes
            raise MfError(-1, "experts must be a [num_experts, stride] byte tensor")
        L = _capi.LayerWeights()
        L.router_w = _ptr(self.router_w)
        L.expert_base = _ptr(self.experts)
        L.expert_stride = self.experts.stride(0)
        L.offsets = self.offsets
        if self.shared is not None:
            L.shared_gate, L.shared_up, L.shared_down = (q.c() for q in self.shared)
        L.w_sg = _ptr(self.w_sg)
        if self.w_sg_q8 is not None:
            L.w_sg_q8 = self.w_sg_q8.c()
        if self.experts_tiled is not None:
            if self.experts_tiled.shape != self.experts.shape or self.experts_tiled.stride(0) != self.experts.stride(0):
                raise MfError(-1, "experts_tiled must have the pool's shape and stride")
            L.expert_tiled = _ptr(self.experts_tiled)
        return L


class MoE:
    """Router + routed experts operator: MoE (Kernels/MoE/MoE.swift),
    MoEDeepseekV4 (2-bit, top-6) and MapleMoE (ternary) in one class, selected
    by `bits`, `top_k` and `router_mode`."""

    def __init__(self, context: MetalContext, d: int, f: int, num_experts: int, top_k: int,
                 bits: int = BITS_4, router_mode: int = ROUTER_TOPK_SOFTMAX,
                 swiglu_limit: float = 0.0, shared_f: int = 0, shared_bits: int = BITS_4,
                 maple_rounding: bool = False, gate_group_size: int = 0):
        """gate_group_size 32: MoEDeepseekV4.encodeRoutedPhase1(gateGroupSize:) -- the routed gate
        projection's tables hold an entry per 32 weights (2-bit experts only)."""
        self.context = context
        self.cfg = _capi.MoEConfig(d, f, num_experts, top_k, bits, router_mode, swiglu_limit,
                                   shared_f, shared_bits, 1 if maple_rounding else 0, gate_group_size)
        self._h = C.c_void_p()
        check(_capi.lib().mf_moe_create(context.handle, C.byref(self.cfg), C.byref(self._h)),
              context.handle)

    def close(self):
        if self._h:
            _capi.lib().mf_moe_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def encode_decode_layer_normed(self, weights: MoELayerWeights, hidden, norm_weight, y, t: int = 1, delta=None,
                                   eps: float = 1e-6, out_indices=None, out_weights=None, stream=None):
        """hidden += delta, x = RMSNorm(hidden) * norm_weight, y = layer(x), hidden += y: one launch where the
        fused launch takes the layer (RealForwardRunner.swift:2799-2808 and the layer behind it)."""
        lw = weights.c()
        check(_capi.lib().mf_moe_decode_layer_normed(self._h, _stream(stream), C.byref(lw), _ptr(hidden), _ptr(delta),
                                                     _ptr(norm_weight), eps, t, _ptr(y), _ptr(out_indices),
                                                     _ptr(out_weights)), self.context.handle)

    def set_fused(self, enabled) -> None:
        """single fused launch (True / 1, default) or the chain of separate launches (False / 0); 2: the fused
        launch through the instance that reads every dimension from its arguments"""
        check(_capi.lib().mf_moe_set_fused(self._h, int(enabled)), self.context.handle)

    def tile_experts(self, experts: torch.Tensor, offsets: ExpertOffsets, stream=None) -> torch.Tensor:
        """a copy of the expert pool [e, stride] in the prefill matmul's own order (mf_moe_tile_experts): pass it
        as MoELayerWeights.experts_tiled"""
        out = torch.empty_like(experts)
        check(_capi.lib().mf_moe_tile_experts(self._h, _stream(stream), _ptr(experts), experts.stride(0),
                                              C.byref(offsets), _ptr(out)), self.context.handle)
        return out

    def set_prefill_route_rounding(self, narrow: bool) -> None:
        """per-route down results of the prefill layer narrowed to bf16 before their routing weights (True: the
        reference's prefill rule, prefill.metal:817-819) or kept in fp32 as the decode step keeps them (False)"""
        check(_capi.lib().mf_moe_set_prefill_route_rounding(self._h, 1 if narrow else 0), self.context.handle)

    def set_phase_trace(self, buffer: Optional[torch.Tensor]) -> None:
        """int64 device tensor of num_cu*8 entries receiving per-workgroup stage
        timestamps of the fused launch (100 MHz clock); None switches it off"""
        check(_capi.lib().mf_moe_set_phase_trace(
            self._h, _ptr(buffer), 0 if buffer is None else buffer.numel() * 8),
            self.context.handle)

    def status(self, stream=None) -> None:
        """synchronises and raises if a fused launch gave up on a grid barrier"""
        check(_capi.lib().mf_moe_status(self._h, _stream(stream)), self.context.handle)

    def encode_router(self, router_w, x, out_indices, out_weights, t: int = 1,
                      x_stride: Optional[int] = None, out_logits=None, stream=None):
        """encodeRouterGemma4 (MoE.swift:153-203) / encodeRouterTopK / encodeRouterTop8."""
        check(_capi.lib().mf_moe_router(self._h, _stream(stream), _ptr(router_w), _ptr(x), t,
                                        self.cfg.d if x_stride is None else x_stride,
                                        _ptr(out_indices), _ptr(out_weights), _ptr(out_logits)),
              self.context.handle)

    def encode_routed_phase1(self, experts: torch.Tensor, offsets: ExpertOffsets, indices, x, acts,
                             t: int = 1, x_stride: Optional[int] = None, stream=None):
        """encodeRoutedPersistentPhase1U16Load (MoE.swift:220-253)."""
        check(_capi.lib().mf_moe_phase1(self._h, _stream(stream), _ptr(experts), experts.stride(0),
                                        C.byref(offsets), _ptr(indices), _ptr(x), t,
                                        self.cfg.d if x_stride is None else x_stride, _ptr(acts)),
              self.context.handle)

    def encode_routed_phase1_subset(self, experts: torch.Tensor, offsets: ExpertOffsets, indices, x, acts,
                                    active_slots, active_count: int, t: int = 1,
                                    x_stride: Optional[int] = None, stream=None):
        """encodeRoutedPersistentPhase1SubsetU16Load (MoE.swift:255-298): only the listed slots."""
        check(_capi.lib().mf_moe_phase1_subset(self._h, _stream(stream), _ptr(experts), experts.stride(0),
                                               C.byref(offsets), _ptr(indices), _ptr(x), t,
                                               self.cfg.d if x_stride is None else x_stride, _ptr(acts),
                                               _ptr(active_slots), active_count),
              self.context.handle)

    def encode_routed_phase2_reduce(self, experts: torch.Tensor, offsets: ExpertOffsets, indices,
                                    routing_weights, acts, residual, y, t: int = 1, stream=None):
        """encodeRoutedPersistentPhase2Reduce (MoE.swift:400-440)."""
        check(_capi.lib().mf_moe_phase2(self._h, _stream(stream), _ptr(experts), experts.stride(0),
                                        C.byref(offsets), _ptr(indices), _ptr(routing_weights),
                                        _ptr(acts), _ptr(residual), t, _ptr(y)),
              self.context.handle)

    def encode_slot_lookup(self, indices, slot_of, slot_stride: int, out_slot_offsets, out_all_hit,
                           t: int = 1, stream=None):
        """router_slot_lookup_k8 (moe.metal:594-617): slot byte offsets of the routed experts from the
        caller's expert -> slot table (int16, negative = not resident), and the all-hit word."""
        check(_capi.lib().mf_moe_slot_lookup(self._h, _stream(stream), _ptr(indices), t, _ptr(slot_of),
                                             slot_stride, _ptr(out_slot_offsets), _ptr(out_all_hit)),
              self.context.handle)

    def encode_routed_phase1_slots(self, slab, slot_offsets, offsets: ExpertOffsets, x, acts, t: int = 1,
                                   all_hit=None, stream=None):
        """Phase 1 over slots named directly (MoE.swift:205-253 with `slab=None` and a table of device
        addresses; MoE.swift:333-407 with a slab and byte offsets, guarded by `all_hit`)."""
        check(_capi.lib().mf_moe_phase1_slots(self._h, _stream(stream), _ptr(slab), _ptr(slot_offsets),
                                              _ptr(all_hit), C.byref(offsets), _ptr(x), t, x.stride(0) if x.dim() > 1 else self.cfg.d,
                                              _ptr(acts)), self.context.handle)

    def encode_routed_phase2_reduce_slots(self, slab, slot_offsets, offsets: ExpertOffsets, routing_weights,
                                          acts, residual, y, t: int = 1, all_hit=None, stream=None):
        """Phase 2 + rank-ordered reduce over slots named directly (MoE.swift:409-440, 333-407)."""
        check(_capi.lib().mf_moe_phase2_slots(self._h, _stream(stream), _ptr(slab), _ptr(slot_offsets),
                                              _ptr(all_hit), C.byref(offsets), _ptr(routing_weights),
                                              _ptr(acts), _ptr(residual), t, _ptr(y)), self.context.handle)

    def encode_decode_layer(self, weights: MoELayerWeights, x, y, t: int = 1, hidden=None,
                            out_indices=None, out_weights=None, stream=None):
        """The fused decode layer (router -> experts -> shared add), one call."""
        lw = weights.c()
        check(_capi.lib().mf_moe_decode_layer(self._h, _stream(stream), C.byref(lw), _ptr(x), t,
                                              _ptr(y), _ptr(hidden), _ptr(out_indices),
                                              _ptr(out_weights)), self.context.handle)

    def encode_group(self, indices, routing_weights, t: int, sorted_pairs, expert_offsets,
                     expert_counts, stream=None):
        """PrefillRouter.makeTokenExpertPairs + PrefillMoEGrouping.groupTokenExpertPairs
        (PrefillRouter.swift:91-111, PrefillMoEGrouping.swift:91-192) on device.
        sorted_pairs: int32/uint8 device tensor of t*top_k 16-byte records."""
        check(_capi.lib().mf_moe_group(self._h, _stream(stream), _ptr(indices),
                                       _ptr(routing_weights), t, _ptr(sorted_pairs),
                                       _ptr(expert_offsets), _ptr(expert_counts)),
              self.context.handle)

    def group_status(self, stream=None) -> None:
        """synchronises; raises MfError(expert out of range) if the last
        encode_group saw an index >= num_experts"""
        check(_capi.lib().mf_moe_group_status(self._h, _stream(stream)), self.context.handle)

    def prefill_workspace_bytes(self, t: int) -> int:
        return int(_capi.lib().mf_moe_prefill_workspace_bytes(self._h, t))

    def encode_prefill_layer(self, weights: MoELayerWeights, x, y, t: int, workspace=None,
                             out_indices=None, out_weights=None, stream=None):
        """Ragged prefill layer over t tokens (PrefillGroupedRoutedMoE.encodeStreamedBatched,
        PrefillGroupedRoutedMoE.swift:392-466, + reduce + shared expert).  `workspace`: uint8
        device tensor of at least prefill_workspace_bytes(t); allocated when None."""
        need = self.prefill_workspace_bytes(t)  # 0 for formats that take the decode launch
        if workspace is None:
            workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
        lw = weights.c()
        check(_capi.lib().mf_moe_prefill_layer(self._h, _stream(stream), C.byref(lw), _ptr(x), t,
                                               _ptr(y), _ptr(workspace), workspace.numel(),
                                               _ptr(out_indices), _ptr(out_weights)),
              self.context.handle)
        return workspace


    def encode_streamed_batched(self, experts: torch.Tensor, offsets: ExpertOffsets, hidden, sorted_pairs,
                                expert_counts, route_partials, t: int, workspace=None, stream=None):
        """PrefillGroupedRoutedMoE.encodeStreamedBatched (PrefillGroupedRoutedMoE.swift:392-466): the
        routed experts over a grouping the caller holds (encode_group's sorted pairs and counts).
        route_partials: float32 [t * top_k, d], row token * top_k + rank.  A grouping that fails the
        device check computes nothing and group_status() raises."""
        if experts.dim() != 2:
            raise ValueError("experts must be a 2-D uint8 pool [num_experts, blob_stride]")
        if workspace is None:
            workspace = torch.empty(max(self.prefill_workspace_bytes(t), 16), dtype=torch.uint8,
                                    device=hidden.device)
        check(_capi.lib().mf_moe_ragged_qmm(self._h, _stream(stream), _ptr(experts), experts.stride(0),
                                            C.byref(offsets), _ptr(hidden), _ptr(sorted_pairs),
                                            _ptr(expert_counts), t, _ptr(route_partials),
                                            _ptr(workspace), workspace.numel()), self.context.handle)
        return workspace

    def encode_reduce_token_major(self, route_partials, route_weights, h2, t: int, indices=None,
                                  residual=None, stream=None):
        """PrefillMoE.encodeReduceTokenMajor (PrefillMoE.swift:11-38): h2[token] = sum over ranks of
        route_weights[token, rank] * route_partials[token * top_k + rank] (+ residual), bf16."""
        check(_capi.lib().mf_moe_unpermute(self._h, _stream(stream), _ptr(route_partials),
                                           _ptr(route_weights), _ptr(indices), _ptr(residual), t,
                                           _ptr(h2)), self.context.handle)


PAIR_DTYPE = np.dtype([("token", "<u4"), ("expert", "<u4"), ("rank", "<u4"),
                       ("weight_bits", "<u4")])
GROUP_DTYPE = np.dtype([("expert", "<u4"), ("pair_start", "<u4"), ("pair_count", "<u4")])
TILE_DTYPE = np.dtype([("group_start", "<u4"), ("group_count", "<u4"), ("pair_start", "<u4"),
                       ("pair_count", "<u4")])


def PrefillTokenExpertPair(token: int, expert: int, rank: int, weight_bits: int):
    """One route record (Kernels/Prefill/MoE/PrefillRouter.swift:4-28)."""
    return (token, expert, rank, weight_bits)


@dataclass
class PrefillMoEGroupedRoutes:
    """Kernels/Prefill/MoE/PrefillMoEGrouping.swift:32-50."""
    sorted_pairs: np.ndarray
    per_expert_offsets: np.ndarray
    per_expert_counts: np.ndarray
    groups: np.ndarray
    tiles: np.ndarray
    query_count: int

    @property
    def max_pairs_per_expert(self) -> int:
        return int(self.groups["pair_count"].max()) if self.groups.size else 0

    @property
    def max_pairs_per_tile(self) -> int:
        return int(self.tiles["pair_count"].max()) if self.tiles.size else 0

    @property
    def max_live_experts_per_tile(self) -> int:
        return int(self.tiles["group_count"].max()) if self.tiles.size else 0


class PrefillMoEGrouping:
    """Kernels/Prefill/MoE/PrefillMoEGrouping.swift:90-192 (host, integer)."""

    @staticmethod
    def make_token_expert_pairs(indices: np.ndarray, weight_bits: np.ndarray, query_count: int,
                                top_k: int) -> np.ndarray:
        """PrefillRouter.makeTokenExpertPairs (PrefillRouter.swift:91-111)."""
        indices = np.asarray(indices, np.uint32).reshape(-1)
        weight_bits = np.asarray(weight_bits, np.uint32).reshape(-1)
        if indices.size != query_count * top_k or weight_bits.size != query_count * top_k:
            raise ValueError("indices / weights count mismatch")
        out = np.empty(query_count * top_k, PAIR_DTYPE)
        out["token"] = np.repeat(np.arange(query_count, dtype=np.uint32), top_k)
        out["rank"] = np.tile(np.arange(top_k, dtype=np.uint32), query_count)
        out["expert"] = indices
        out["weight_bits"] = weight_bits
        return out

    @staticmethod
    def group_token_expert_pairs(pairs, query_count: int, top_k: int, num_experts: int,
                                 tile_expert_count: int = 16,
                                 expert_sort_keys=None) -> PrefillMoEGroupedRoutes:
        if isinstance(pairs, np.ndarray) and pairs.dtype == PAIR_DTYPE:
            p = np.ascontiguousarray(pairs)
        else:
            p = np.array([tuple(x) for x in pairs], dtype=PAIR_DTYPE)
        n = p.size
        sorted_ = np.empty(n, PAIR_DTYPE)
        ne = max(num_experts, 1)
        offsets = np.empty(ne, np.uint32)
        counts = np.empty(ne, np.uint32)
        cap = max(min(ne, n), 1)
        groups = np.empty(cap, GROUP_DTYPE)
        tiles = np.empty(cap, TILE_DTYPE)
        ng, nt = C.c_size_t(0), C.c_size_t(0)
        keys = None if expert_sort_keys is None else np.ascontiguousarray(expert_sort_keys, np.uint64)
        detail = (C.c_uint32 * 2)()
        vp = lambda a: None if a is None else a.ctypes.data_as(C.c_void_p)
        rc = _capi.lib().mf_group_pairs_host(
            vp(p), n, query_count, top_k, num_experts, tile_expert_count, vp(keys),
            0 if keys is None else keys.size, vp(sorted_), vp(offsets), vp(counts), vp(groups),
            C.byref(ng), vp(tiles), C.byref(nt), C.cast(detail, C.c_void_p))
        if rc != 0:
            err = MfError(rc, f"detail={detail[0]},{detail[1]}")
            err.detail = (int(detail[0]), int(detail[1]))
            raise err
        return PrefillMoEGroupedRoutes(sorted_, offsets[:num_experts], counts[:num_experts],
                                       groups[:ng.value], tiles[:nt.value], query_count)
