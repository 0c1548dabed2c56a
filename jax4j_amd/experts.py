"""A block of experts: a host-side mirror of the engine's ``j4q_experts_*`` entry points and of what its norms are
(include/jax4j_mi355x.h). Engine-local; the reference has neither.

A decoder's layer of experts on device addresses, h the residual stream, a the output of the block before::

    experts = Experts(be, gate, up, down, experts=64)             # quantized [64 * ffn, dim], [64 * ffn, dim], [64 * dim, ffn]
    be.norm_into(h, x, rows, dim, Norm(w), block_ptr=a, residual_out_ptr=h)       # h += a; x = norm(h)
    be.quant_matvec_into(router, x, 0, logits, batch=rows)
    be.route_into(logits, ids, weights, rows, 64, 8, renormalize=True)
    experts.apply(x, ids, weights, y, rows, 8)
    be.norm_into(h, x, rows, dim, Norm(next_w), block_ptr=y, residual_out_ptr=h)  # the next block's

Pointers are device addresses (integers); calls enqueue on ``stream`` (0: the engine stream) and do not wait.
"""
from __future__ import annotations

import ctypes as C

from . import _native as N
from .backend import Mi355xBackend, _int32, _int64, _kind, _plain_addresses, check
from .tensor import DeviceBuffer, DType, IllegalArgumentException

_ACTIVATIONS = {"silu": N.ACT_SILU, "gelu": N.ACT_GELU, "relu": N.ACT_RELU}


class Norm:
    """A norm of rows (``j4q_norm``): ``kind`` "rms" or "layer"; ``weight_ptr`` (0: ones) and ``bias_ptr`` (0: zeros): fp32 [dim];
    ``weight_add`` is added to the weights."""

    def __init__(self, weight_ptr: int = 0, kind: str = "rms", *, bias_ptr: int = 0, eps: float = 1e-6, weight_add: float = 0.0):
        k = {"rms": N.NORM_RMS, "layer": N.NORM_LAYER}.get(kind)
        if k is None:
            raise IllegalArgumentException(f"unknown norm {kind!r} (rms or layer)")
        w, b = _plain_addresses(weight_ptr, bias_ptr)
        if (w | b) >> 64:
            raise IllegalArgumentException("norm: an address does not fit 64 bits")
        self.args = N.NormKind(k, eps, w or None, b or None, weight_add)
        self.ref = C.pointer(self.args)


class Experts:
    """The quantized matrices of a layer of experts; ``gate`` and ``up`` [experts * ffn, dim], ``down`` [experts * dim, ffn]. They
    cannot be released before ``destroy``. ``activation``: "silu", "gelu" (the tanh form) or "relu"."""

    def __init__(self, backend: Mi355xBackend, gate: DeviceBuffer, up: DeviceBuffer, down: DeviceBuffer, *, experts: int, activation: str = "silu"):
        self._be = backend
        self.handle = 0
        if activation not in _ACTIVATIONS:
            raise IllegalArgumentException(f"unknown activation {activation!r} (silu, gelu or relu)")
        c = N.ExpertsConfig(gate.handle, up.handle, down.handle, _int32(experts), _ACTIVATIONS[activation])
        out = C.c_uint64()
        check(backend._lib().j4q_experts_create(C.byref(c), C.byref(out)), "experts")
        self.handle = out.value

    def destroy(self) -> None:
        """Wait for the device, then give the handle's memory back; the matrices stay."""
        check(N.load().j4q_experts_destroy(self.handle), "experts destroy")
        self.handle = 0

    def info(self) -> dict:
        d = N.ExpertsDesc()
        check(N.load().j4q_experts_info(self.handle, C.byref(d)), "experts info")
        return {"experts": d.config.experts, "dim": d.dim, "ffn": d.ffn, "weight_bytes": d.weight_bytes, "bytes": d.bytes}

    def workspace(self, rows: int, top_k: int, dtype: DType = DType.F32) -> int:
        """Bytes of workspace that a call of so many rows takes; a call of fewer rows may take more, so ask for each size of call."""
        n = C.c_uint64()
        check(N.load().j4q_experts_workspace(self.handle, _int64(rows), _int32(top_k), _kind(dtype), C.byref(n)), "experts workspace")
        return n.value

    def apply(self, x_ptr: int, ids_ptr: int, weights_ptr: int, out_ptr: int, rows: int, top_k: int, dtype: DType = DType.F32, *, x_stride: int = 0,
              out_stride: int = 0, workspace_ptr: int = 0, workspace_bytes: int = 0, stream: int = 0) -> None:
        """out[r] = sum over slots of weights[r, s] * down_e (act(gate_e x[r]) * (up_e x[r])), e = ids[r, s] (none where that is no
        expert's index). x and out [rows, dim], F32 or BF16; strides in values, 0: dim. ``workspace``: the caller's, for calls that are
        captured into a graph; 0: the engine's."""
        if not type(x_ptr) is type(ids_ptr) is type(weights_ptr) is type(out_ptr) is type(workspace_ptr) is type(stream) is int:
            x_ptr, ids_ptr, weights_ptr, out_ptr, workspace_ptr, stream = _plain_addresses(x_ptr, ids_ptr, weights_ptr, out_ptr, workspace_ptr, stream)
        if top_k >> 31 or (rows | x_stride | out_stride) >> 63 or (workspace_bytes | x_ptr | ids_ptr | weights_ptr | out_ptr | workspace_ptr | stream) >> 64:
            raise IllegalArgumentException(f"experts apply: {rows} rows of {top_k} experts, a stride or an address are negative or do not fit")
        a = N.ExpertsArgs(x_ptr, ids_ptr, weights_ptr, out_ptr, rows, x_stride, out_stride, top_k, _kind(dtype), workspace_ptr, workspace_bytes)
        check(self._be._lib().j4q_experts_apply(self.handle, C.byref(a), stream), "experts apply")
