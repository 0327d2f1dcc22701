"""Host-side mirror of the reference's operator interface for the quantized linear path, over
torch CUDA tensors (torch is only the owner of device memory and streams here).

Names follow the reference: `quantize_rows`, `matmul`, `prepare_quantized`, `quantized_norm`,
`quantized_gated`, `linear` (src/ops/storage.h:12, src/ops/basic.h:11,25-26,33-35,
src/ops/linear.h:11-14) and `RowScaledView` (src/core/quantization.h:33-49). Every function ends in
a call through the C ABI of libb200q.so: the per-step operations through the compiled binding `_native`
(csrc/bindings/python.cpp), and through ctypes where that one declines an argument and for everything a
program calls once.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import (BF16, F16, F32, FP8, I8, I32, Attention, Cache, Epilogue, NormFusion, Path_, RotaryPlan, RowScaled,
                   Tensor)

try:
    from . import _native
except ImportError as error:  # not built (or for another torch): importing this module still works, calling does not
    _native = _lib.MissingBinding(error)

MODES = ("int8", "fp8", "group_int8", "group_fp8")
_TORCH_TYPES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.int32: I32,
                torch.int8: I8, torch.uint8: None}
RELU, LEAKY_RELU, SILU, GELU, GELU_TANH, TANH, SIGMOID = 1, 2, 3, 4, 5, 7, 8


def groups_of(mode: str) -> tuple[int, int, int]:
    """(activation group, weight group, rotation) — reference: quantization_groups, src/core/quantization.h:19-23."""
    return (128, 128, 128) if mode.startswith("group_") else (0, 0, 0)


def format_of(mode: str) -> int:
    return FP8 if mode.endswith("fp8") else I8


def _tensor(t: torch.Tensor | None, type_code: int | None = None) -> Tensor:
    if t is None:
        return Tensor(None, 0, 0, 0, 0, -1)
    if not t.is_cuda:
        raise ValueError("operands must live on a CUDA device")
    if t.dim() == 1:
        t = t.unsqueeze(0)
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError("operands must be 2-D with a dense inner axis")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:  # a stride of 0 would be taken for dense rows
        raise ValueError("operands' rows must not overlap: expanded tensors have to be made contiguous")
    code = type_code if type_code is not None else _TORCH_TYPES[t.dtype]
    stride = t.stride(0) if t.shape[0] > 1 and t.stride(0) != t.shape[1] else 0
    if max(*t.shape, stride) > 2**31 - 1:  # ctypes would keep the low 32 bits
        raise ValueError("operands have at most 2^31 - 1 rows and columns, and as many elements between two rows")
    return Tensor(t.data_ptr(), t.shape[0], t.shape[1], stride, code, t.device.index)


@dataclass
class RowScaledView:
    """One-byte values [rows, K] + fp32 scales ([rows] or group-major [K/g, rows])."""
    values: torch.Tensor  # uint8 storage
    scales: torch.Tensor  # float32
    format: int           # I8 or FP8
    group_size: int = 0
    rotation_size: int = 0

    @staticmethod
    def empty(rows: int, cols: int, fmt: int, group: int = 0, rotation: int = 0, device="cuda") -> "RowScaledView":
        values = torch.empty(rows, cols, dtype=torch.uint8, device=device)
        shape = ((cols + group - 1) // group, rows) if group else (rows, 1)
        scales = torch.empty(shape, dtype=torch.float32, device=device)
        return RowScaledView(values, scales, fmt, group, rotation)

    def c(self) -> RowScaled:
        return RowScaled(_tensor(self.values, self.format), _tensor(self.scales, F32), self.group_size, self.rotation_size)

    def rows(self, first: int, count: int) -> "RowScaledView":
        """Leading-row view; only for per-row scales (K-group scales are row-minor)."""
        if self.group_size:
            raise ValueError("row slices of K-group scales are not contiguous")
        return RowScaledView(self.values[first:first + count], self.scales[first:first + count], self.format, 0,
                             self.rotation_size)


@dataclass
class CacheView:
    """Quantized key/value cache: one byte per value [pages, kv_heads, page_size, head_dim], one fp32 scale per token and head
    [pages, kv_heads, page_size]. Slot s is token s % page_size of page s // page_size."""
    keys: torch.Tensor          # uint8 (or int8 / float8_e4m3fn) storage
    values: torch.Tensor
    key_scales: torch.Tensor    # float32
    value_scales: torch.Tensor
    format: int                 # I8 or FP8

    @staticmethod
    def empty(pages: int, kv_heads: int, page_size: int, head_dim: int, fmt: int, device="cuda") -> "CacheView":
        """Slots hold anything until they are written; no operator reads one that its arguments do not name."""
        shape = (pages, kv_heads, page_size)
        values = (torch.empty(*shape, head_dim, dtype=torch.uint8, device=device) for _ in range(2))
        scales = (torch.empty(shape, dtype=torch.float32, device=device) for _ in range(2))
        return CacheView(*values, *scales, fmt)

    def c(self) -> Cache:
        shape, device = self.keys.shape, self.keys.device
        parts = (self.keys, self.values, self.key_scales, self.value_scales)
        if (len(shape) != 4 or self.values.shape != shape or any(t.shape != shape[:3] for t in parts[2:])
                or any(t.dtype != torch.float32 for t in parts[2:]) or any(t.element_size() != 1 for t in parts[:2])
                or any(not t.is_cuda or t.device != device or not t.is_contiguous() for t in parts)):
            raise ValueError("a cache is two contiguous one-byte tensors [pages, kv_heads, page_size, head_dim] and two float32 "
                             "tensors [pages, kv_heads, page_size] on one CUDA device")
        return Cache(*(t.data_ptr() for t in parts), *shape, self.format, device.index)


@dataclass
class Rotary:
    """Rotary positions: pair i of a head turns by turns[i] revolutions per position. The first 2 * len(turns) columns of a head take part,
    as pairs (i, i + len(turns)), or (2i, 2i + 1) when interleaved; cosine and sine are multiplied by `scale`."""
    turns: torch.Tensor  # float64 on the device
    interleaved: bool = False
    scale: float = 1.0

    SCALINGS = ("none", "linear", "base", "yarn", "wavelength")

    @staticmethod
    def plan(dims: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
             original_length: int = 0, low: float = 1.0, high: float = 0.0, device="cuda") -> "Rotary":
        """The usual turns base ** (-2 i / dims) / 2 pi, stretched by `factor` for longer contexts: "linear" all of them, "base" by a larger
        base, "yarn" and "wavelength" those that make few turns within original_length (a ramp between `low` and `high` turns)."""
        if scaling not in Rotary.SCALINGS:
            raise ValueError(f"scaling must be one of {Rotary.SCALINGS}")
        host, scale = torch.empty(max(dims // 2, 0), dtype=torch.float64), C.c_float(1.0)
        _lib.call("b200q_rotary_turns", dims, base, Rotary.SCALINGS.index(scaling), factor, original_length, low, high,
                  C.cast(host.data_ptr(), C.POINTER(C.c_double)), C.byref(scale))
        return Rotary(host.to(device), interleaved, scale.value)

    def c(self) -> RotaryPlan:
        if self.turns.dtype != torch.float64 or self.turns.dim() != 1 or not self.turns.is_cuda or not self.turns.is_contiguous():
            raise ValueError("rotary turns must be a contiguous float64 vector on a CUDA device")
        return RotaryPlan(self.turns.data_ptr(), 2 * self.turns.numel(), int(self.interleaved), self.scale, self.turns.device.index)


def attention_workspace(rows: int, sequences: int, heads: int, kv_heads: int, head_dim: int, prefix: bool = False,
                        multiprocessors: int = 148) -> int:
    """Bytes of context workspace that Context.cached_attention needs."""
    needed = C.c_size_t()
    _lib.call("b200q_attention_workspace", rows, sequences, heads, kv_heads, head_dim, int(prefix), multiprocessors, C.byref(needed))
    return needed.value


def _epilogue(bias=None, residual=None, residual_f32=None, activation=0, value_scale=1.0, output_scale=1.0,
              residual_scale=1.0, alpha=0.1, gate=None, condition=None, raw=None, rows_per_sequence=1,
              valid_rows_per_sequence=0, input_repeat=1, residual_rows=None) -> Epilogue:
    """reference: ops::Epilogue (src/ops/sequence.h:8-27); residual_rows is a device int32 tensor."""
    rows_ptr = C.c_void_p(residual_rows.data_ptr()) if residual_rows is not None else None
    return Epilogue(_tensor(bias), _tensor(residual), _tensor(residual_f32, F32), value_scale, output_scale,
                    residual_scale, alpha, activation, _tensor(gate), _tensor(condition), _tensor(raw), rows_per_sequence,
                    valid_rows_per_sequence, input_repeat, rows_ptr)


def _fusion(residual=None, projection_bias=None, raw=None, gate=None, shift=None, scale=None, rows_per_sequence=1,
            source_rows=None) -> NormFusion:
    """reference: ops::NormFusion (src/ops/sequence.h:53-57); source_rows is a device int32 tensor."""
    rows_ptr = C.c_void_p(source_rows.data_ptr()) if source_rows is not None else None
    return NormFusion(_tensor(residual), _tensor(projection_bias), _tensor(raw), _tensor(gate), _tensor(shift),
                      _tensor(scale), rows_per_sequence, rows_ptr)


if not isinstance(_native, _lib.MissingBinding):
    _native.bind(_lib.B200QError, RowScaledView.c, CacheView.c, Rotary.c)


class Context:
    """Device + stream + GEMM workspace + plan cache (reference: CudaContext, src/runtime/cuda_context.h:13-35)."""

    def __init__(self, mode: str = "int8", device: int = 0, stream: torch.cuda.Stream | None = None,
                 workspace_bytes: int = 8 << 20):
        if mode not in MODES:
            raise ValueError(f"quantization must be one of {MODES}")
        self.mode, self.device = mode, device
        self.format = format_of(mode)
        self.stream = stream
        self._workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=f"cuda:{device}")
        handle = C.c_void_p()
        stream_ptr = C.c_void_p(stream.cuda_stream) if stream is not None else None
        _lib.call("b200q_context_create", device, stream_ptr, C.c_void_p(self._workspace.data_ptr()), workspace_bytes,
                  mode.encode(), C.byref(handle))
        self._handle, self._address = handle, handle.value
        self.multiprocessors = _lib.load().b200q_multiprocessors(handle)

    def close(self):
        if getattr(self, "_handle", None):
            _lib.load().b200q_context_destroy(self._handle)
            self._handle, self._address = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- producers
    def quantize_rows(self, x: torch.Tensor, out: RowScaledView) -> RowScaledView:
        if _native.row_quantize(self._address, x, out) is NotImplemented:
            _lib.call("b200q_row_quantize", self._handle, C.byref(_tensor(x)), C.byref(out.c()))
        return out

    def quantized_norm(self, residual, update, weight, out: RowScaledView, epsilon: float, gemma=False, update_scale=None):
        """residual += update (times update_scale); out = quantized RMSNorm of it. `weight` is a parameter: it is read ahead of the
        kernels before this call, so the stream has to have been synchronized since it was written."""
        if _native.quantized_norm(self._address, residual, update, weight, out, epsilon, gemma, update_scale) is NotImplemented:
            _lib.call("b200q_quantized_norm", self._handle, C.byref(_tensor(residual)), C.byref(_tensor(update)),
                      C.byref(_tensor(weight)), C.byref(out.c()), epsilon, int(gemma), C.byref(_tensor(update_scale)))
        return out

    def quantized_gated(self, x: torch.Tensor, out: RowScaledView, kind: int = 0) -> RowScaledView:
        if _native.quantized_gated(self._address, x, out, kind) is NotImplemented:
            _lib.call("b200q_quantized_gated", self._handle, C.byref(_tensor(x)), C.byref(out.c()), kind)
        return out

    # ---- GEMM
    def prepare_quantized(self, rows: int, channels: int, reduction: int, out_dtype=torch.bfloat16,
                          groups: tuple[int, int] | None = None, weight: RowScaledView | None = None) -> tuple[int, int, int, int]:
        """Plans the shape. `weight` announces a weight of it: its producers are enqueued on this context's stream, so GEMMs may
        fetch its values and scales ahead of the kernels before them. Replaced by one of this context's calls it stays announced;
        replaced in any other way it has to be announced again (or the stream synchronized) before it is used."""
        ga, gw = groups if groups is not None else groups_of(self.mode)[:2]
        path = Path_()
        _lib.call("b200q_prepare", self._handle, rows, channels, reduction, _TORCH_TYPES[out_dtype], ga, gw, C.byref(path))
        if weight is not None:
            _lib.call("b200q_prepare_weight", self._handle, C.byref(weight.c()))
        return (path.kind, path.tokens, path.channels, path.splits)

    def select_path(self, rows, channels, reduction, groups=None):
        ga, gw = groups if groups is not None else groups_of(self.mode)[:2]
        path = Path_()
        _lib.call("b200q_select_path", self._handle, rows, channels, reduction, ga, gw, C.byref(path))
        return (path.kind, path.tokens, path.channels, path.splits)

    def seal(self):
        _lib.call("b200q_seal", self._handle)

    def matmul(self, x: RowScaledView, w: RowScaledView, out: torch.Tensor, **epilogue) -> torch.Tensor:
        """out = dequantized x @ w^T, for a shape that prepare_quantized has planned; a little faster on an announced weight."""
        if _native.linear(self._address, x, w, out, epilogue) is NotImplemented:
            ep = C.byref(_epilogue(**epilogue)) if epilogue else None
            _lib.call("b200q_linear", self._handle, C.byref(x.c()), C.byref(w.c()), C.byref(_tensor(out)), ep)
        return out

    def quant_linear(self, path, x: RowScaledView, w: RowScaledView, out: torch.Tensor, **epilogue) -> torch.Tensor:
        ep = C.byref(_epilogue(**epilogue)) if epilogue else None
        _lib.call("b200q_quant_linear", self._handle, C.byref(Path_(*path)), C.byref(x.c()), C.byref(w.c()),
                  C.byref(_tensor(out)), ep)
        return out

    def linear(self, x: torch.Tensor, w: RowScaledView, scratch: RowScaledView, out: torch.Tensor,
               quantized_output: RowScaledView | None = None, **epilogue):
        if _native.linear_forward(self._address, x, w, scratch, out, epilogue, quantized_output) is NotImplemented:
            ep = C.byref(_epilogue(**epilogue)) if epilogue else None
            qo = C.byref(quantized_output.c()) if quantized_output is not None else None
            _lib.call("b200q_linear_forward", self._handle, C.byref(_tensor(x)), C.byref(w.c()), C.byref(scratch.c()),
                      C.byref(_tensor(out)), ep, qo)
        return out

    # ---- row-wise operators around the projections
    def pointwise(self, x: torch.Tensor, y: torch.Tensor, **epilogue) -> torch.Tensor:
        if _native.pointwise(self._address, x, y, epilogue) is NotImplemented:
            _lib.call("b200q_pointwise", self._handle, C.byref(_tensor(x)), C.byref(_tensor(y)), C.byref(_epilogue(**epilogue)))
        return y

    def pointwise_quantize(self, x: torch.Tensor, out: RowScaledView, retained: torch.Tensor | None = None,
                           **epilogue) -> RowScaledView:
        if _native.pointwise_quantize(self._address, x, out, epilogue, retained) is NotImplemented:
            _lib.call("b200q_pointwise_quantize", self._handle, C.byref(_tensor(x)), C.byref(out.c()),
                      C.byref(_epilogue(**epilogue)), C.byref(_tensor(retained)))
        return out

    def layer_norm_quantize(self, x: torch.Tensor, out: RowScaledView, weight=None, bias=None, epsilon: float = 1e-5,
                            retained: torch.Tensor | None = None, **fusion) -> RowScaledView:
        if _native.layer_norm_quantize(self._address, x, out, weight, bias, epsilon, fusion, retained) is NotImplemented:
            _lib.call("b200q_layer_norm_quantize", self._handle, C.byref(_tensor(x)), C.byref(out.c()), C.byref(_tensor(weight)),
                      C.byref(_tensor(bias)), epsilon, C.byref(_fusion(**fusion)), C.byref(_tensor(retained)))
        return out

    def normalized_linear(self, x: torch.Tensor, w: RowScaledView, out: torch.Tensor, norm_weight=None, norm_bias=None,
                          epsilon: float = 1e-5, bias=None, normalized=None, fusion: dict | None = None,
                          quantized_output: RowScaledView | None = None, **epilogue) -> bool:
        """True when the fused kernel ran; False leaves the two-step path to the caller."""
        taken = C.c_int32(0)
        qo = C.byref(quantized_output.c()) if quantized_output is not None else None
        _lib.call("b200q_normalized_linear", self._handle, C.byref(_tensor(x)), C.byref(w.c()), C.byref(_tensor(bias)),
                  C.byref(_tensor(normalized)), C.byref(_tensor(out)), C.byref(_tensor(norm_weight)),
                  C.byref(_tensor(norm_bias)), epsilon, C.byref(_fusion(**(fusion or {}))), C.byref(_epilogue(**epilogue)),
                  qo, C.byref(taken))
        return bool(taken.value)

    # ---- between the QKV and the O projection
    def rotary(self, x: torch.Tensor, positions: torch.Tensor, rotary: Rotary, head_dim: int, out: torch.Tensor | None = None) -> torch.Tensor:
        """Turns every head of x [rows, heads * head_dim] by positions [rows] (int32). out may be x."""
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if _native.rotary(self._address, x, positions, rotary, head_dim, out) is NotImplemented:
            _lib.call("b200q_rotary", self._handle, C.byref(_tensor(x)), C.byref(_tensor(positions)), C.byref(rotary.c()), head_dim,
                      C.byref(_tensor(out)))
        return out

    def cache_write(self, cache: CacheView, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor | None = None,
                    rotary: Rotary | None = None, q: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                    q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, epsilon: float = 1e-6) -> None:
        """Quantizes row r of k and v [rows, kv_heads * head_dim] into slot slots[r] (int32, each at most once; negative or past the
        cache: left out). k, and q into q_out (may be q), are normalised over each head and turned first, where the arguments say so."""
        if _native.cache_write(self._address, cache, k, v, slots, positions, rotary, q, q_out, q_norm, k_norm, epsilon) is NotImplemented:
            _lib.call("b200q_cache_write", self._handle, C.byref(cache.c()), C.byref(_tensor(k)), C.byref(_tensor(v)), C.byref(_tensor(slots)),
                      C.byref(_tensor(positions)), C.byref(rotary.c()) if rotary is not None else None, C.byref(_tensor(q)),
                      C.byref(_tensor(q_out)), C.byref(_tensor(q_norm)), C.byref(_tensor(k_norm)), epsilon)

    def cache_read(self, cache: CacheView, slots: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None) -> None:
        """Row r of k and v (either may be None) = what slot slots[r] holds; zeros for a slot outside of the cache."""
        if _native.cache_read(self._address, cache, slots, k, v) is NotImplemented:
            _lib.call("b200q_cache_read", self._handle, C.byref(cache.c()), C.byref(_tensor(slots)), C.byref(_tensor(k)), C.byref(_tensor(v)))

    def cached_attention(self, q: torch.Tensor, cache: CacheView, pages: torch.Tensor, lengths: torch.Tensor, out: torch.Tensor,
                         scale: float = 0.0, query_offsets: torch.Tensor | None = None, prefix_pages: torch.Tensor | None = None,
                         prefix_length: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q [rows, heads * head_dim] over the cache. pages [sequences, n] and lengths [sequences] (int32) name each
        sequence's cached tokens, the query rows' own among them; query_offsets [sequences + 1] its rows (without it, one each). All
        rows also see the prefix_length [1] tokens on prefix_pages [m], which are read once for the batch. Rows that see nothing are
        zero, rows behind the last offset are left alone. scale 0: 1 / sqrt(head_dim)."""
        if _native.cached_attention(self._address, q, cache, pages, lengths, out, scale, query_offsets, prefix_pages,
                                    prefix_length) is NotImplemented:
            arguments = Attention(_tensor(q), _tensor(out), _tensor(pages), _tensor(lengths), _tensor(query_offsets), _tensor(prefix_pages),
                                  _tensor(prefix_length), scale)
            _lib.call("b200q_cached_attention", self._handle, C.byref(cache.c()), C.byref(arguments))
        return out

    def status(self) -> int:
        value = C.c_int32(0)
        _lib.call("b200q_status", self._handle, C.byref(value))
        return value.value


class Linear:
    """Quantized Linear layer (reference: tts::Linear, src/layers/linear.h:11-76): fuses the given 16-bit
    weight matrices by rows, quantizes them on the device at construction (the load-time step of
    Weights::quantized), and runs quantize -> GEMM -> fused epilogue per call."""

    def __init__(self, ctx: Context, parts: list[torch.Tensor], bias: torch.Tensor | None = None, max_rows: int = 64):
        self.ctx = ctx
        self._keep = (parts, bias)
        array = (Tensor * len(parts))(*[_tensor(p) for p in parts])
        handle = C.c_void_p()
        _lib.call("b200q_linear_layer_create", ctx._handle, array, len(parts), C.byref(_tensor(bias)), C.byref(handle))
        self._handle, self._address = handle, handle.value
        self.out_features = sum(p.shape[0] for p in parts)
        self.in_features = parts[0].shape[1]
        _lib.call("b200q_linear_layer_prepare", ctx._handle, self._handle, max_rows)

    def forward(self, x: torch.Tensor, out: torch.Tensor | None = None, quantized_output: RowScaledView | None = None,
                **epilogue) -> torch.Tensor:
        if out is None:
            out = torch.empty(x.shape[0], self.out_features, dtype=x.dtype, device=x.device)
        if _native.layer_forward(self.ctx._address, self._address, x, out, epilogue, quantized_output) is NotImplemented:
            ep = C.byref(_epilogue(**epilogue)) if epilogue else None
            qo = C.byref(quantized_output.c()) if quantized_output is not None else None
            _lib.call("b200q_linear_layer_forward", self.ctx._handle, self._handle, C.byref(_tensor(x)), C.byref(_tensor(out)), ep, qo)
        return out

    PLAN, PREPARE, CAPTURE, EXECUTE = 0, 1, 2, 3  # reference: ForwardContext::Mode (src/core/forward_context.h:58)

    def apply(self, mode: int, max_rows: int, x: torch.Tensor, out: torch.Tensor, **epilogue) -> torch.Tensor:
        """Phase-switched forward (reference: Linear::forward(input, output, ForwardContext &, finish))."""
        ep = C.byref(_epilogue(**epilogue)) if epilogue else None
        _lib.call("b200q_linear_layer_apply", self.ctx._handle, self._handle, mode, max_rows, C.byref(_tensor(x)),
                  C.byref(_tensor(out)), ep)
        return out

    def forward_segments(self, mode: int, max_rows: int, x: torch.Tensor, segments: list[tuple[int, int, int]],
                         out: torch.Tensor) -> torch.Tensor:
        flat = (C.c_int32 * (3 * len(segments)))(*[v for s in segments for v in s]) if segments else None
        _lib.call("b200q_linear_layer_forward_segments", self.ctx._handle, self._handle, mode, max_rows, C.byref(_tensor(x)),
                  flat, len(segments), C.byref(_tensor(out)))
        return out

    def normalized_forward(self, x: torch.Tensor, out: torch.Tensor, norm_weight=None, norm_bias=None, epsilon: float = 1e-5,
                           normalized=None, fusion: dict | None = None, quantized_output: RowScaledView | None = None,
                           **epilogue) -> torch.Tensor:
        if _native.layer_normalized_forward(self.ctx._address, self._address, x, normalized, out, norm_weight, norm_bias, epsilon,
                                            fusion, epilogue, quantized_output) is NotImplemented:
            ep = C.byref(_epilogue(**epilogue)) if epilogue else None
            qo = C.byref(quantized_output.c()) if quantized_output is not None else None
            _lib.call("b200q_linear_layer_normalized_forward", self.ctx._handle, self._handle, C.byref(_tensor(x)),
                      C.byref(_tensor(normalized)), C.byref(_tensor(out)), C.byref(_tensor(norm_weight)),
                      C.byref(_tensor(norm_bias)), epsilon, C.byref(_fusion(**(fusion or {}))), ep, qo)
        return out

    def weight(self) -> RowScaled:
        view = RowScaled()
        _lib.call("b200q_linear_layer_weight", self._handle, C.byref(view))
        return view

    def close(self):
        if getattr(self, "_handle", None):
            _lib.load().b200q_linear_layer_destroy(self._handle)
            self._handle, self._address = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
