"""Torch-facing wrappers over the C ABI.  PyTorch supplies device memory and streams only; every
computation below is a call into libsparseflow_b200.so.

Replaces, on the reference side: ``prune_24_dense_weight`` (sparseflow/nn/sparseflow_linear.py:20-35),
``torch.sparse.to_sparse_semi_structured`` (sparseflow/fused_mlp.py:22,28), the sparse matmul call
sites (sparseflow/fused_mlp.py:54,60; sparseflow/nn/sparseflow_linear.py:123) and
``fused_silu_mul`` (sparseflow/kernels/fused_silu_mul.py:33-57).
"""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass, field
from typing import Optional

import torch

from . import _lib

F16, BF16 = 0, 1
TIE_HIGH, TIE_LOW = 0, 1
ACT = {"none": 0, None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float16:
        return F16
    if t.dtype == torch.bfloat16:
        return BF16
    raise ValueError(f"expected torch.float16 or torch.bfloat16, got {t.dtype}")


def _tie(tie) -> int:
    if tie in ("high", TIE_HIGH):
        return TIE_HIGH
    if tie in ("low", TIE_LOW):
        return TIE_LOW
    raise ValueError(f"tie must be 'high' or 'low', got {tie!r}")


def _need_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """Handle of the current CUDA stream of the current device (the raw getter is ~10x cheaper than building a
    torch.cuda.Stream object; it matters for kernels of a few microseconds launched eagerly)."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


class _NoSwitch:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


_NO_SWITCH = _NoSwitch()


def _on(device: torch.device):
    """Context that makes `device` current; free when it already is."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NO_SWITCH
    return torch.cuda.device(device)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def device_status() -> int:
    """Synchronise and return the device status word (0 = ok); raises on a device-side failure."""
    w = C.c_int(0)
    rc = _lib.lib().sfb200_device_status(C.byref(w))
    if rc != 0:
        raise _lib.SfbError(f"sfb200_device_status (word 0x{w.value:x})", rc)
    return w.value


@dataclass
class Compressed24:
    """A 2:4-compressed weight: values [rows, K/2] + tiled metadata (uint8 view of the tile array)."""
    values: torch.Tensor
    meta: torch.Tensor
    rows: int
    K: int
    gate_up: bool = False   # rows interleaved 16 gate / 16 up

    @property
    def dtype(self) -> torch.dtype:
        return self.values.dtype

    def nbytes(self) -> int:
        return self.values.numel() * 2 + self.meta.numel()


def prune_compress_24(w: torch.Tensor, tie="high", want_values=True, want_meta=True,
                      want_ref_codes=False, want_pruned=False) -> dict:
    """2:4 magnitude prune + compress of w[rows, K]; returns the requested outputs."""
    _need_cuda(w, "w")
    if w.dim() != 2:
        raise ValueError(f"w must be 2D, got {w.dim()}D")
    rows, K = w.shape
    if K % 4 != 0:
        raise ValueError(f"in_features must be multiple of 4 for 2:4 (got {K})")
    if w.stride(1) != 1:
        w = w.contiguous()
    L = _lib.lib()
    dev = w.device
    out = {}
    with _on(dev):
        if want_values:
            out["values"] = torch.empty((rows, K // 2), dtype=w.dtype, device=dev)
        if want_meta:
            out["meta"] = torch.empty(L.sfb200_meta_bytes(rows, K), dtype=torch.uint8, device=dev)
        if want_ref_codes:
            out["ref_codes"] = torch.empty((rows, K // 4), dtype=torch.uint8, device=dev)
        if want_pruned:
            out["pruned"] = torch.empty((rows, K), dtype=w.dtype, device=dev)
        rc = L.sfb200_prune_compress_24(w.data_ptr(), rows, K, w.stride(0), _dt(w), _tie(tie),
                                        _ptr(out.get("values")), _ptr(out.get("meta")),
                                        _ptr(out.get("ref_codes")), _ptr(out.get("pruned")), _stream())
    _lib.check("sfb200_prune_compress_24", rc)
    return out


def compress_weight(w: torch.Tensor, tie="high") -> Compressed24:
    o = prune_compress_24(w, tie=tie)
    return Compressed24(o["values"], o["meta"], w.shape[0], w.shape[1])


def compress_gate_up(gate: torch.Tensor, up: torch.Tensor, tie="high") -> Compressed24:
    """Fused gate|up weight (2*I rows, 16-row interleave) for ``sparse_gemm_swiglu``."""
    _need_cuda(gate, "gate")
    _need_cuda(up, "up")
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("gate and up must have the same shape and dtype")
    gate = gate.contiguous()
    up = up.contiguous()
    I, K = gate.shape
    L = _lib.lib()
    with _on(gate.device):
        values = torch.empty((2 * I, K // 2), dtype=gate.dtype, device=gate.device)
        meta = torch.empty(L.sfb200_meta_bytes(2 * I, K), dtype=torch.uint8, device=gate.device)
        rc = L.sfb200_prune_compress_gate_up(gate.data_ptr(), up.data_ptr(), I, K, K, _dt(gate),
                                             _tie(tie), values.data_ptr(), meta.data_ptr(), _stream())
    _lib.check("sfb200_prune_compress_gate_up", rc)
    return Compressed24(values, meta, 2 * I, K, gate_up=True)


def validate_24(w: torch.Tensor) -> bool:
    _need_cuda(w, "w")
    if w.stride(1) != 1:
        w = w.contiguous()
    with _on(w.device):
        flag = torch.empty(1, dtype=torch.int32, device=w.device)
        rc = _lib.lib().sfb200_validate_24(w.data_ptr(), w.shape[0], w.shape[1], w.stride(0),
                                           flag.data_ptr(), _stream())
    _lib.check("sfb200_validate_24", rc)
    return bool(flag.item())


def decompress_24(cw: Compressed24) -> torch.Tensor:
    with _on(cw.values.device):
        out = torch.empty((cw.rows, cw.K), dtype=cw.dtype, device=cw.values.device)
        rc = _lib.lib().sfb200_decompress_24(cw.values.data_ptr(), cw.meta.data_ptr(), cw.rows, cw.K,
                                             out.data_ptr(), cw.K, _stream())
    _lib.check("sfb200_decompress_24", rc)
    return out


def _kernel_ready(x: torch.Tensor) -> torch.Tensor:
    """The kernels read activations through TMA: unit inner stride, row pitch a multiple of 8 elements,
    16-byte aligned base.  A view that breaks one of these (a column slice, an odd offset) is copied,
    as the reference's call sites do unconditionally (sparseflow/nn/sparseflow_linear.py:122-124)."""
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) % 8 != 0) or x.data_ptr() % 16 != 0:
        return x.contiguous()
    return x


def _check_bias(bias: torch.Tensor, x: torch.Tensor, rows: int) -> torch.Tensor:
    """The epilogue reads `rows` bias values in the GEMM's own 16-bit type."""
    if not bias.is_cuda or bias.get_device() != x.get_device():
        raise ValueError(f"bias must be a CUDA tensor on {x.device}, got {bias.device}")
    if bias.dtype != x.dtype:
        raise ValueError(f"bias dtype {bias.dtype} != activation dtype {x.dtype}")
    if bias.numel() != rows:
        raise ValueError(f"bias has {bias.numel()} elements, weight has {rows} rows")
    return bias if bias.is_contiguous() else bias.contiguous()


def sparse_gemm(x: torch.Tensor, cw: Compressed24, bias: Optional[torch.Tensor] = None,
                act: Optional[str] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[M, N] = act(x[M, K] . W^T + bias)."""
    _need_cuda(x, "x")
    if x.dim() != 2 or x.shape[1] != cw.K:
        raise ValueError(f"Expected last dim {cw.K}, got {tuple(x.shape)}")
    if x.dtype != cw.dtype:
        raise ValueError(f"x dtype {x.dtype} != weight dtype {cw.dtype}")
    x = _kernel_ready(x)
    if bias is not None:
        bias = _check_bias(bias, x, cw.rows)
    M = x.shape[0]
    dev = x.get_device()
    with _NO_SWITCH if dev == torch.cuda.current_device() else torch.cuda.device(dev):
        if out is None:
            out = x.new_empty((M, cw.rows))
        if M == 0:                      # empty batch: nothing to launch
            return out
        rc = _lib.lib().sfb200_sparse_gemm(x.data_ptr(), x.stride(0), cw.values.data_ptr(),
                                           cw.meta.data_ptr(), out.data_ptr(), out.stride(0), M, cw.rows,
                                           cw.K, _dt(x), _ptr(bias), ACT[act], _stream())
    if rc:
        _lib.check("sfb200_sparse_gemm", rc)
    return out


def sparse_gemm_swiglu(x: torch.Tensor, cw_gu: Compressed24, out: Optional[torch.Tensor] = None,
                       gate_bias: Optional[torch.Tensor] = None, up_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h[M, I] = silu(x . Wg^T + gate_bias) * (x . Wu^T + up_bias) from the fused gate|up weight."""
    _need_cuda(x, "x")
    if not cw_gu.gate_up:
        raise ValueError("weight was not built with compress_gate_up")
    if x.dim() != 2 or x.shape[1] != cw_gu.K or x.dtype != cw_gu.dtype:
        raise ValueError("shape / dtype mismatch")
    x = _kernel_ready(x)
    M, I = x.shape[0], cw_gu.rows // 2
    if gate_bias is not None:
        gate_bias = _check_bias(gate_bias, x, I)
    if up_bias is not None:
        up_bias = _check_bias(up_bias, x, I)
    dev = x.get_device()
    with _NO_SWITCH if dev == torch.cuda.current_device() else torch.cuda.device(dev):
        if out is None:
            out = x.new_empty((M, I))
        if M == 0:
            return out
        rc = _lib.lib().sfb200_sparse_gemm_swiglu_bias(x.data_ptr(), x.stride(0), cw_gu.values.data_ptr(),
                                                       cw_gu.meta.data_ptr(), _ptr(gate_bias), _ptr(up_bias),
                                                       out.data_ptr(), out.stride(0), M, I, cw_gu.K, _dt(x), _stream())
    if rc:
        _lib.check("sfb200_sparse_gemm_swiglu", rc)
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """out = silu(gate) * up for 2-D (possibly strided-row) tensors."""
    _need_cuda(gate, "gate")
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.dim() != 2:
        raise ValueError("fused_silu_mul expects two 2D tensors of equal shape and dtype")
    if gate.stride(1) != 1:
        gate = gate.contiguous()
    if up.stride(1) != 1:
        up = up.contiguous()
    with _on(gate.device):
        out = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
        if gate.numel() == 0:
            return out
        rc = _lib.lib().sfb200_silu_mul(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0),
                                        out.data_ptr(), out.stride(0), gate.shape[0], gate.shape[1],
                                        _dt(gate), _stream())
    _lib.check("sfb200_silu_mul", rc)
    return out


def force_token_tile(bn: int) -> None:
    _lib.check("sfb200_debug_force_token_tile", _lib.lib().sfb200_debug_force_token_tile(bn))


# ------------------------------------------------------------------ around the gated FFN
# A mixture of experts over 2:4 weights, the norms between two blocks, low-rank adapters.  Group sizes stay on the device:
# none of these calls waits for the GPU, and each can be captured into a CUDA graph.

_MANY = 2 ** 31 - 4097      # rows, columns and entries that the kernels count in 32 bits
MAX_NORM_COLS = 16384       # of block_norm: a row stays in a block's registers
_DT3 = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream_of(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def _on_own_device(fn):
    """The call with its first tensor's device current.  One comparison where it already is: a context manager costs a microsecond, and
    these calls are launched eagerly around kernels of a few."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kw):
        t = args[0] if args else kw[first]
        if not t.is_cuda:
            raise ValueError(f"{first} must be a CUDA tensor")
        dev = t.get_device()
        if dev == _current_device():
            return fn(*args, **kw)
        with torch.cuda.device(dev):
            return fn(*args, **kw)
    return call


def _on_device_of(x: torch.Tensor, t: Optional[torch.Tensor], name: str) -> None:
    if t is not None and (not t.is_cuda or t.get_device() != x.get_device()):
        raise ValueError(f"{name} must be a CUDA tensor on {x.device}, got {t.device}")


def _rows2d(t: torch.Tensor, name: str) -> tuple:
    """(t, row pitch in elements): 2-D with unit inner stride, rows may be strided (a view that is not so is copied)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2D, got {t.dim()}D")
    if t.numel() > _MANY and max(t.shape) > _MANY:
        raise ValueError(f"{name}: {tuple(t.shape)} is beyond 32-bit counts")
    if not t.is_contiguous() and ((t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        t = t.contiguous()
    return t, _pitch(t)


def _rows16(t: torch.Tensor, name: str) -> tuple:
    """``_rows2d`` with what 16-byte accesses need: row pitch a multiple of 8 elements, 16-byte aligned base."""
    t, pitch = _rows2d(t, name)
    if t.data_ptr() % 16 or pitch % 8:
        t = t.clone(memory_format=torch.contiguous_format)
        pitch = _pitch(t)
    return t, pitch


def _pitch(t: torch.Tensor) -> int:
    """Row pitch in elements (of one row: its length, whatever its stride says)."""
    if t.is_contiguous():
        return t.size(1)
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of the same shape (for a contiguous one without the parsing of a size: half a microsecond)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _check_out(out: torch.Tensor, like: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if tuple(out.shape) != shape or out.dtype != dtype or not out.is_cuda or out.get_device() != like.get_device():
        raise ValueError(f"out must be {shape} {dtype} on {like.device}")
    if (out.stride(-1) != 1 and shape[-1] > 1) or (out.dim() == 2 and shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError("out must have unit inner stride and rows that do not overlap")


def _extent(t: torch.Tensor) -> tuple:
    n = sum((d - 1) * s for d, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _check_apart(out: torch.Tensor, t: torch.Tensor, name: str, same: bool = False) -> None:
    """The kernels read ``t`` while they write ``out``: the two share no memory, or (``same``) are the same rows."""
    (a, b), (c, d) = _extent(out), _extent(t)
    if a < d and c < b and not (same and a == c and out.shape == t.shape and _pitch(out) == _pitch(t)):
        raise ValueError(f"out and {name} share memory")


@dataclass
class RowGroups:
    """Entries grouped by id.  ``offsets[g]`` .. ``offsets[g + 1]`` are the places of group g; ``rows[place]`` is the row the entry
    at a place belongs to (-1 behind the last group); ``slots[entry]`` is an entry's place (-1: of no group).  One that is written by hand:
    contiguous int32 tensors of these lengths."""
    offsets: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor
    groups: int
    per_row: int = 1
    made_here: bool = field(default=False, repr=False, compare=False)      # by group_rows or moe_route: not looked at again


@dataclass
class Routing:
    """A router's choice: ``weights`` [tokens, top_k] float32, ``experts`` [tokens, top_k] int32 (-1: none), and the grouping of
    the tokens by expert (``groups.slots`` has the shape of ``experts``)."""
    weights: torch.Tensor
    experts: torch.Tensor
    groups: RowGroups


def _check_groups(t: torch.Tensor, groups: RowGroups, slots: bool) -> None:
    """The kernels read ``groups + 1`` offsets, and a row and (``slots``) a slot per entry, as int32."""
    if groups.made_here:
        return _on_device_of(t, groups.offsets, "groups")
    if groups.offsets.numel() != groups.groups + 1 or (slots and groups.slots.numel() != groups.rows.numel()):
        raise ValueError(f"a grouping of {groups.groups} groups has {groups.groups + 1} offsets, and a slot per row")
    for name, v in (("offsets", groups.offsets), ("rows", groups.rows)) + ((("slots", groups.slots),) if slots else ()):
        if v.dtype != torch.int32 or not v.is_contiguous() or v.device != t.device:
            raise ValueError(f"groups.{name} must be a contiguous int32 tensor on {t.device}, got {v.dtype} on {v.device}")


def group_rows(ids: torch.Tensor, groups: int, per_row: int = 1) -> RowGroups:
    """Group entries by id, keeping their order inside a group; ids outside 0 .. groups-1 belong to no group.  ``per_row``: entries
    per row (entry i belongs to row ``i // per_row``)."""
    _need_cuda(ids, "ids")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    if not 1 <= groups <= 1024:
        raise ValueError(f"groups must be 1 .. 1024, got {groups}")
    if per_row < 1 or ids.numel() % per_row:
        raise ValueError(f"per_row {per_row} does not divide {ids.numel()} entries")
    n = ids.numel()
    if n > _MANY:
        raise ValueError(f"{n} entries are beyond 32-bit counts")
    L = _lib.calls()
    with _on(ids.device):
        if ids.dtype == torch.int64:
            ids = ids.clamp(-1, groups).to(torch.int32)
        ids = ids.contiguous()
        offsets = torch.empty(groups + 1, dtype=torch.int32, device=ids.device)
        rows = torch.empty(n, dtype=torch.int32, device=ids.device)
        slots = torch.empty(ids.shape, dtype=torch.int32, device=ids.device)
        work = torch.empty(L.sfb200_group_workspace_bytes(groups), dtype=torch.uint8, device=ids.device) if n > 4096 else None
        rc = L.sfb200_group_rows(ids.data_ptr(), n, groups, per_row, offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(), _ptr(work), _stream())
    _lib.check("sfb200_group_rows", rc)
    return RowGroups(offsets, rows, slots, groups, per_row, True)


@_on_own_device
def moe_route(logits: torch.Tensor, top_k: int, renormalize: bool = True) -> Routing:
    """Route tokens to experts: the ``top_k`` largest of ``logits[tokens, experts]`` (ties, -0 and +0 among them, to the lowest expert), their softmax
    weights (over all experts, or with ``renormalize`` over the chosen ones), and the grouping of the tokens by expert.

    A logit of -inf or NaN is never chosen; a token with fewer than ``top_k`` others gets expert -1 with weight 0 there (a row of
    padding, all -inf, goes nowhere).  +inf counts as the largest finite number."""
    dt = _DT3.get(logits.dtype)
    if dt is None:
        raise ValueError(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    logits, ld = _rows2d(logits, "logits")
    n, E = logits.shape
    if not 1 <= E <= 1024:
        raise ValueError(f"experts must be 1 .. 1024, got {E}")
    if not 1 <= top_k <= min(32, E):
        raise ValueError(f"top_k must be 1 .. {min(32, E)}, got {top_k}")
    L = _lib.calls()
    # one allocation for the four results of n * top_k words: an allocation costs as much host time as the kernel takes
    weights, chosen, slots, rows = logits.new_empty((4, n, top_k), dtype=torch.int32).unbind(0)
    weights, rows = weights.view(torch.float32), rows.flatten()
    offsets = logits.new_empty(E + 1, dtype=torch.int32)
    work = logits.new_empty(L.sfb200_group_workspace_bytes(E), dtype=torch.uint8) if n > 32 else None
    rc = L.sfb200_moe_route(logits.data_ptr(), ld, n, E, top_k, dt, 1 if renormalize else 0, weights.data_ptr(), chosen.data_ptr(),
                            offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(), _ptr(work), _stream_of(logits.get_device()))
    if rc:
        _lib.check("sfb200_moe_route", rc)
    return Routing(weights, chosen, RowGroups(offsets, rows, slots, E, top_k, True))


@dataclass
class CompressedExperts:
    """2:4-compressed weights of several experts, one after the other: values [experts, rows, K/2] + the tiled metadata of each."""
    values: torch.Tensor
    meta: torch.Tensor
    experts: int
    rows: int
    K: int
    gate_up: bool = False   # rows interleaved 16 gate / 16 up

    @property
    def dtype(self) -> torch.dtype:
        return self.values.dtype

    def nbytes(self) -> int:
        return self.values.numel() * 2 + self.meta.numel()

    def expert(self, e: int) -> Compressed24:
        m = self.meta.numel() // self.experts
        return Compressed24(self.values[e], self.meta[e * m:(e + 1) * m], self.rows, self.K, self.gate_up)


def _experts3d(w: torch.Tensor, name: str) -> torch.Tensor:
    _need_cuda(w, name)
    _dt(w)
    if w.dim() != 3:
        raise ValueError(f"{name} must be [experts, rows, K], got {w.dim()}D")
    if w.shape[2] % 64 or w.shape[1] % 8 or not 1 <= w.shape[0] <= 1024 or not w.numel():
        raise ValueError(f"{name}: 1 .. 1024 experts, rows a multiple of 8 and K of 64, got {tuple(w.shape)}")
    return w.contiguous()


def compress_experts(w: torch.Tensor, tie="high") -> CompressedExperts:
    """Prune and compress the weights ``w[experts, rows, K]`` for ``grouped_sparse_gemm`` (a weight that is 2:4 already keeps its values)."""
    w = _experts3d(w, "w")
    E, N, K = w.shape
    L = _lib.lib()
    with _on(w.device):
        each = L.sfb200_meta_bytes(N, K)
        values = torch.empty((E, N, K // 2), dtype=w.dtype, device=w.device)
        meta = torch.empty(E * each, dtype=torch.uint8, device=w.device)
        # whole metadata tiles: one weight of experts x rows; otherwise each expert's last tile is padded
        for e, rows in ((0, E * N),) if N % 128 == 0 else ((e, N) for e in range(E)):
            rc = L.sfb200_prune_compress_24(w[e].data_ptr(), rows, K, K, _dt(w), _tie(tie), values[e].data_ptr(), meta.data_ptr() + e * each, None, None,
                                            _stream())
            _lib.check("sfb200_prune_compress_24", rc)
    return CompressedExperts(values, meta, E, N, K)


def compress_gate_up_experts(gate: torch.Tensor, up: torch.Tensor, tie="high") -> CompressedExperts:
    """Fused gate|up weights of several experts (2*I rows each, 16-row interleave) for ``grouped_sparse_gemm_swiglu``."""
    gate, up = _experts3d(gate, "gate"), _experts3d(up, "up")
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise ValueError("gate and up must have the same shape, dtype and device")
    E, I, K = gate.shape
    if I % 16:
        raise ValueError(f"intermediate size must be a multiple of 16, got {I}")
    L = _lib.lib()
    with _on(gate.device):
        each = L.sfb200_meta_bytes(2 * I, K)
        values = torch.empty((E, 2 * I, K // 2), dtype=gate.dtype, device=gate.device)
        meta = torch.empty(E * each, dtype=torch.uint8, device=gate.device)
        for e, rows in ((0, E * I),) if I % 64 == 0 else ((e, I) for e in range(E)):
            rc = L.sfb200_prune_compress_gate_up(gate[e].data_ptr(), up[e].data_ptr(), rows, K, K, _dt(gate), _tie(tie), values[e].data_ptr(),
                                                 meta.data_ptr() + e * each, _stream())
            _lib.check("sfb200_prune_compress_gate_up", rc)
    return CompressedExperts(values, meta, E, 2 * I, K, gate_up=True)


def _expert_bias(b: Optional[torch.Tensor], x: torch.Tensor, experts: int, cols: int, name: str) -> Optional[torch.Tensor]:
    if b is None:
        return None
    _on_device_of(x, b, name)
    if b.dtype != x.dtype or tuple(b.shape) != (experts, cols):
        raise ValueError(f"{name} must be [{experts}, {cols}] {x.dtype}, got {tuple(b.shape)} {b.dtype}")
    return b.contiguous()


def _grouped_args(x: torch.Tensor, cw: CompressedExperts, groups: RowGroups, gather: bool):
    if x.dim() != 2 or x.shape[1] != cw.K:
        raise ValueError(f"Expected last dim {cw.K}, got {tuple(x.shape)}")
    if x.dtype != cw.dtype:
        raise ValueError(f"x dtype {x.dtype} != weight dtype {cw.dtype}")
    if groups.groups != cw.experts:
        raise ValueError(f"grouping has {groups.groups} groups, the weights {cw.experts} experts")
    _on_device_of(x, cw.values, "weights")
    _check_groups(x, groups, False)
    total = groups.rows.numel()
    if gather:
        if x.shape[0] * groups.per_row != total:
            raise ValueError(f"grouping is of {total // groups.per_row} rows, x has {x.shape[0]}")
    elif x.shape[0] != total:
        raise ValueError(f"grouping has {total} places, x has {x.shape[0]} rows (gather=True reads x through the grouping)")
    return *_rows16(x, "x"), total


def _grouped_scratch(x: torch.Tensor, total: int, cw: CompressedExperts) -> Optional[torch.Tensor]:
    n = _lib.calls().sfb200_grouped_scratch_bytes(total, cw.experts, cw.rows, cw.K)
    return torch.empty(n, dtype=torch.uint8, device=x.device) if n else None


@_on_own_device
def grouped_sparse_gemm(x: torch.Tensor, cw: CompressedExperts, groups: RowGroups, bias: Optional[torch.Tensor] = None, act: Optional[str] = None,
                        gather: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[place] = act(x[place] . W_e^T + bias[e]) for the places of every expert e.

    ``x`` holds a row per place in the order of ``groups``; with ``gather`` a row per token, read through ``groups.rows``.  Rows of the
    result behind the last group are left as they were (in a fresh result: undefined).  ``out`` shares no memory with ``x``."""
    x, ldx, total = _grouped_args(x, cw, groups, gather)
    if act not in ACT:
        raise ValueError(f"unknown activation {act!r}")
    if cw.gate_up:
        raise ValueError("gate|up weights: use grouped_sparse_gemm_swiglu")
    bias = _expert_bias(bias, x, cw.experts, cw.rows, "bias")
    if out is None:
        out = x.new_empty((total, cw.rows))
    else:
        _check_out(out, x, (total, cw.rows), x.dtype)
        _check_apart(out, x, "x")
    if total == 0:
        return out
    scratch = _grouped_scratch(x, total, cw) if gather else None
    rc = _lib.calls().sfb200_grouped_sparse_gemm(x.data_ptr(), ldx, x.shape[0], groups.rows.data_ptr() if gather else None, _ptr(scratch),
                                               cw.values.data_ptr(), cw.meta.data_ptr(), out.data_ptr(), _pitch(out), total, cw.experts, cw.rows,
                                               cw.K, _dt(x), _ptr(bias), ACT[act], groups.offsets.data_ptr(), _stream_of(x.get_device()))
    if rc:
        _lib.check("sfb200_grouped_sparse_gemm", rc)
    return out


@_on_own_device
def grouped_sparse_gemm_swiglu(x: torch.Tensor, cw_gu: CompressedExperts, groups: RowGroups, gather: bool = False,
                               gate_bias: Optional[torch.Tensor] = None, up_bias: Optional[torch.Tensor] = None,
                               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h[place] = silu(x . Wg_e^T + gate_bias[e]) * (x . Wu_e^T + up_bias[e]) from the fused gate|up weights; ``x``, ``gather`` and
    the rows behind the last group as in ``grouped_sparse_gemm``."""
    x, ldx, total = _grouped_args(x, cw_gu, groups, gather)
    if not cw_gu.gate_up:
        raise ValueError("weights were not built with compress_gate_up_experts")
    I = cw_gu.rows // 2
    gate_bias = _expert_bias(gate_bias, x, cw_gu.experts, I, "gate_bias")
    up_bias = _expert_bias(up_bias, x, cw_gu.experts, I, "up_bias")
    if out is None:
        out = x.new_empty((total, I))
    else:
        _check_out(out, x, (total, I), x.dtype)
        _check_apart(out, x, "x")
    if total == 0:
        return out
    scratch = _grouped_scratch(x, total, cw_gu) if gather else None
    rc = _lib.calls().sfb200_grouped_sparse_gemm_swiglu(x.data_ptr(), ldx, x.shape[0], groups.rows.data_ptr() if gather else None,
                                                      _ptr(scratch), cw_gu.values.data_ptr(), cw_gu.meta.data_ptr(), out.data_ptr(), _pitch(out),
                                                      total, cw_gu.experts, I, cw_gu.K, _dt(x), _ptr(gate_bias), _ptr(up_bias),
                                                      groups.offsets.data_ptr(), _stream_of(x.get_device()))
    if rc:
        _lib.check("sfb200_grouped_sparse_gemm_swiglu", rc)
    return out


@_on_own_device
def moe_combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, residual: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = residual[t] + sum_j weights[t, j] * y[slots[t, j]], in 32 bits, rounded once; a slot of -1 adds nothing.
    ``out`` may be ``residual``."""
    dt = _dt(y)
    y, ld_y = _rows2d(y, "y")
    if slots.dim() != 2 or slots.shape != weights.shape or slots.dtype != torch.int32 or weights.dtype != torch.float32:
        raise ValueError("slots must be [tokens, top_k] int32 and weights the same shape in float32")
    dev = y.get_device()
    if slots.get_device() != dev or weights.get_device() != dev:
        _on_device_of(y, slots, "slots")
        _on_device_of(y, weights, "weights")
    n, k = slots.shape
    rows, H = y.shape
    if not H or not k:
        raise ValueError(f"nothing to add up: y is {tuple(y.shape)}, slots {tuple(slots.shape)}")
    ld_res = 0
    if residual is not None:
        _on_device_of(y, residual, "residual")
        if tuple(residual.shape) != (n, H) or residual.dtype != y.dtype:
            raise ValueError(f"residual must be [{n}, {H}] {y.dtype}")
        residual, ld_res = _rows2d(residual, "residual")
    if not (slots.is_contiguous() and weights.is_contiguous()):
        slots, weights = slots.contiguous(), weights.contiguous()
    if out is None:
        out, ld_out = y.new_empty((n, H)), H
    else:
        _check_out(out, y, (n, H), y.dtype)
        _check_apart(out, y, "y")
        if residual is not None:
            _check_apart(out, residual, "residual", same=True)
        ld_out = _pitch(out)
    rc = _lib.calls().sfb200_moe_combine(y.data_ptr(), ld_y, rows, slots.data_ptr(), weights.data_ptr(), _ptr(residual), ld_res, out.data_ptr(), ld_out,
                                       n, k, H, dt, _stream_of(dev))
    if rc:
        _lib.check("sfb200_moe_combine", rc)
    return out


@_on_own_device
def block_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, *, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None,
               post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
               scale: float = 1.0, eps: float = 1e-5, post_eps: Optional[float] = None, kind: str = "rms"):
    """What stands between two blocks, in one pass: returns ``(r, h)`` with

        z = y, or norm(y) * post_weight + post_bias      (the norm after a block)
        r = x + scale * gate * z                          (the residual stream)
        h = norm(r) * weight + bias                       (the norm before the next block, of the unrounded r)

    ``kind``: "rms" or "layer".  ``x`` [rows, cols] float16, bfloat16 or float32; ``y``, the weights, the gate and ``h`` have one
    type, that of ``x`` or (``x`` float32) a 16-bit one.  ``gate``: [cols]; or [g, cols] / [g, 1], each row for rows / g consecutive
    rows.  Without ``y``: r is ``x`` itself.  ``weight=None`` (with ``y``): no second norm, h is None."""
    if kind not in ("rms", "layer"):
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    xt = _DT3.get(x.dtype)
    if xt is None:
        raise ValueError(f"x must be float16, bfloat16 or float32, got {x.dtype}")
    x, ld_x = _rows2d(x, "x")
    n, H = x.shape
    if not 1 <= H <= MAX_NORM_COLS:
        raise ValueError(f"cols must be 1 .. {MAX_NORM_COLS}, got {H}")
    dtype = y.dtype if y is not None else weight.dtype if weight is not None else x.dtype
    yt = _DT3.get(dtype)
    if yt is None or (dtype != x.dtype and x.dtype != torch.float32):
        raise ValueError(f"x {x.dtype} goes with {x.dtype}{' or a 16-bit type' if x.dtype == torch.float32 else ''}, got {dtype}")
    if y is None:
        if weight is None:
            raise ValueError("nothing to compute: neither y nor weight")
        if gate is not None or post_weight is not None or post_bias is not None:
            raise ValueError("gate and post_weight belong to y")
    if (bias is not None and weight is None) or (post_bias is not None and post_weight is None):
        raise ValueError("a bias needs its weight")

    dev = x.get_device()

    def vector(v, name):
        if v is None:
            return None
        if v.dtype is not dtype or v.dim() != 1 or v.size(0) != H or v.get_device() != dev:
            _on_device_of(x, v, name)
            raise ValueError(f"{name} must be [{H}] {dtype}, got {tuple(v.shape)} {v.dtype}")
        return v if v.is_contiguous() else v.contiguous()

    weight = vector(weight, "weight")
    if bias is not None:
        bias = vector(bias, "bias")
    if post_weight is not None:
        post_weight, post_bias = vector(post_weight, "post_weight"), vector(post_bias, "post_bias")
    ld_y = ld_gate = gate_rows = gate_cols = 0
    if y is not None:
        _on_device_of(x, y, "y")
        if y.shape != x.shape:
            raise ValueError(f"y must be {tuple(x.shape)}, got {tuple(y.shape)}")
        y, ld_y = _rows2d(y, "y")
    if gate is not None:
        _on_device_of(x, gate, "gate")
        if gate.dtype != dtype:
            raise ValueError(f"gate dtype {gate.dtype} != {dtype}")
        if gate.dim() == 1:
            gate = gate.unsqueeze(0)
        if gate.dim() != 2 or gate.shape[1] not in (1, H) or not gate.shape[0] or n % gate.shape[0]:
            raise ValueError(f"gate must be [{H}], or [g, {H}] or [g, 1] with g dividing {n} rows, got {tuple(gate.shape)}")
        gate, ld_gate = _rows2d(gate, "gate")
        gate_rows, gate_cols = gate.shape
    r = _empty_like(x) if y is not None else None
    h = (_empty_like(x if y is None else y) if y is not None or dtype is x.dtype else x.new_empty((n, H), dtype=dtype)) if weight is not None else None
    rc = _lib.calls().sfb200_block_norm(x.data_ptr(), ld_x, _ptr(y), ld_y, _ptr(weight), _ptr(bias), _ptr(post_weight), _ptr(post_bias), _ptr(gate),
                                      ld_gate, gate_rows, gate_cols, _ptr(r), H, _ptr(h), H, n, H, xt, yt, scale, eps,
                                      eps if post_eps is None else post_eps, 1 if kind == "layer" else 0, _stream_of(dev))
    if rc:
        _lib.check("sfb200_block_norm", rc)
    return (x if r is None else r), h


class LoraBank:
    """Low-rank adapters of one projection: ``a`` [adapters, rank, K], ``b`` [adapters, N, rank], ``scales`` [adapters] float32 (or one
    number).  The rank is padded with zeros to 8, 16, 32, 64 or 128 (a row of ``x`` with an infinity meets them and comes out NaN); adapters of different
    ranks go through ``from_adapters``."""
    RANKS = (8, 16, 32, 64, 128)

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales=1.0):
        _need_cuda(a, "a")
        _dt(a)
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"expected a [adapters, rank, K] and b [adapters, N, rank], got {tuple(a.shape)} and {tuple(b.shape)}")
        _on_device_of(a, b, "b")
        if b.dtype != a.dtype:
            raise ValueError(f"b dtype {b.dtype} != a dtype {a.dtype}")
        G, r, K = a.shape
        N = b.shape[1]
        if not 1 <= G <= 1024 or not 1 <= r <= 128 or not K or K % 8 or not N or N % 8:
            raise ValueError(f"1 .. 1024 adapters, rank 1 .. 128, K and N multiples of 8, got {G}, {r}, {K}, {N}")
        if isinstance(scales, torch.Tensor):
            _on_device_of(a, scales, "scales")
            if tuple(scales.shape) != (G,):
                raise ValueError(f"scales must be [{G}], got {tuple(scales.shape)}")
            self.scales = scales.detach().to(torch.float32).contiguous()
        else:
            self.scales = torch.full((G,), float(scales), dtype=torch.float32, device=a.device)
        self.rank = next(v for v in self.RANKS if v >= r)
        pad = self.rank - r
        a, b = a.detach(), b.detach()
        self.a = _kernel_ready_bank(torch.nn.functional.pad(a, (0, 0, 0, pad)) if pad else a)
        self.b = _kernel_ready_bank(torch.nn.functional.pad(b, (0, pad)) if pad else b)
        self.adapters, self.K, self.N, self.dtype = G, K, N, a.dtype

    @classmethod
    def from_adapters(cls, adapters, scales=1.0) -> "LoraBank":
        """From a list of (A [rank, K], B [N, rank]) whose ranks may differ."""
        most = max(A.shape[0] for A, _ in adapters)
        pad = torch.nn.functional.pad
        return cls(torch.stack([pad(A, (0, 0, 0, most - A.shape[0])) for A, _ in adapters]),
                   torch.stack([pad(B, (0, most - B.shape[1])) for _, B in adapters]), scales)


def _kernel_ready_bank(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


@_on_own_device
def lora_add(y: torch.Tensor, x: torch.Tensor, bank: LoraBank, groups: RowGroups, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = y[t] + scale_g * (x[t] . A_g^T) . B_g^T for the rows of adapter g (``groups = group_rows(ids, bank.adapters)``); rows of
    no adapter keep ``y``.  ``out`` may be ``y``."""
    n = x.shape[0]
    if x.dim() != 2 or x.shape[1] != bank.K or tuple(y.shape) != (n, bank.N):
        raise ValueError(f"expected x [rows, {bank.K}] and y [rows, {bank.N}], got {tuple(x.shape)} and {tuple(y.shape)}")
    if x.dtype != bank.dtype or y.dtype != bank.dtype:
        raise ValueError(f"x {x.dtype} and y {y.dtype} must have the adapters' type {bank.dtype}")
    if groups.groups != bank.adapters or groups.per_row != 1 or groups.rows.numel() != n:
        raise ValueError(f"grouping must be group_rows(ids, {bank.adapters}) of {n} rows")
    _on_device_of(y, x, "x")
    _on_device_of(y, bank.a, "adapters")
    _check_groups(y, groups, True)
    x, ld_x = _rows16(x, "x")
    if out is None:
        out = _empty_like(y)
    else:
        _check_out(out, y, (n, bank.N), y.dtype)
        _check_apart(out, x, "x")
        _check_apart(out, y, "y", same=True)
    if n == 0:
        return out
    into = out
    if out is y:
        y, ld_y = _rows16(y, "y")
        out, ld_out = y, ld_y
    else:
        y, ld_y = _rows16(y, "y")
        ld_out = _pitch(out)
        if out.data_ptr() % 16 or ld_out % 8:
            out, ld_out = y.new_empty((n, bank.N)), bank.N
    L = _lib.calls()
    work = y.new_empty(L.sfb200_lora_workspace_bytes(n, bank.rank), dtype=torch.uint8)
    rc = L.sfb200_lora_add(y.data_ptr(), ld_y, x.data_ptr(), ld_x, bank.a.data_ptr(), bank.b.data_ptr(), bank.scales.data_ptr(),
                           out.data_ptr(), ld_out, n, bank.adapters, bank.rank, bank.K, bank.N, _dt(y), groups.offsets.data_ptr(),
                           groups.rows.data_ptr(), groups.slots.data_ptr(), work.data_ptr(), _stream_of(y.get_device()))
    if rc:
        _lib.check("sfb200_lora_add", rc)
    if out is not into:
        into.copy_(out)
    return into
