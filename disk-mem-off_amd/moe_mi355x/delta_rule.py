"""The gated delta rule over the recurrent states of a server's sequences, on the MI355X.

``mx_gated_delta_rule`` takes a ragged batch of new rows, starts every sequence from a state
slot (or from zeros) and leaves its state in a slot, chunk by chunk for prompts and token by
token for decode steps.  The reference's own recurrence (offload_runtime/executors/
qwen3_next.py:56-95) has no delta correction and carries no state; it stays with
``LinearAttnRunner`` and ``mx_gated_delta_scan``.
"""
from __future__ import annotations

import ctypes
from typing import Any

from . import _lib
from .types import DeviceBuffer

_DT = {"float32": _lib.MX_DT_F32, "float16": _lib.MX_DT_F16}


def delta_args(*, q: int, k: int, v: int, g: int, beta: int, o: int, state: int, slot_in: int,
               slot_out: int, q_start: int, n_slots: int, n_seqs: int, rows: int, max_q: int,
               n_k_heads: int, n_v_heads: int, head_dim_k: int, head_dim_v: int,
               dtype: str = "float16", qk_norm: bool = True, scale: float | None = None,
               ldq: int | None = None, ldk: int | None = None, ldv: int | None = None,
               ldo: int | None = None) -> _lib.MxGatedDelta:
    """One call's arguments (device addresses; row strides default to contiguous rows; scale
    defaults to ``head_dim_k ** -0.5``)."""
    if dtype not in _DT:
        raise ValueError(f"rows must be float32 or float16, got {dtype!r}")
    kw, vw = n_k_heads * head_dim_k, n_v_heads * head_dim_v
    if scale is None:
        scale = head_dim_k ** -0.5
    return _lib.MxGatedDelta(
        q, k, v, g, beta, o, state, slot_in, slot_out, q_start, kw if ldq is None else ldq,
        kw if ldk is None else ldk, vw if ldv is None else ldv, vw if ldo is None else ldo,
        n_slots, n_seqs, rows, max_q, n_k_heads, n_v_heads, head_dim_k, head_dim_v, _DT[dtype],
        int(bool(qk_norm)), float(scale))


def workspace_bytes(args: _lib.MxGatedDelta) -> int:
    n = ctypes.c_size_t()
    _lib.check(_lib.load().mx_gated_delta_rule_workspace_size(ctypes.byref(args),
                                                              ctypes.byref(n)),
               "mx_gated_delta_rule_workspace_size")
    return int(n.value)


class GatedDeltaRunner:
    """Workspace for gated-delta-rule calls on one stream."""

    def __init__(self, backend: Any) -> None:
        self.backend = backend
        self.lib = _lib.load()
        self._ws: DeviceBuffer | None = None

    def reserve(self, args: _lib.MxGatedDelta) -> None:
        """Workspace for this call and smaller ones (not while an earlier call still runs)."""
        need = workspace_bytes(args)
        if need and (self._ws is None or self._ws.nbytes < need):
            if self._ws is not None:
                self.backend.free_device(self._ws)
                self._ws = None
            self._ws = self.backend.alloc_device(need)

    def forward_device(self, args: _lib.MxGatedDelta, stream: Any,
                       workspace: tuple[int, int] | None = None) -> None:
        """Outputs and final states of the batch; asynchronous.  ``workspace`` (address,
        bytes) stands in for the reserved one."""
        ptr, nbytes = workspace or ((self._ws.handle, self._ws.nbytes) if self._ws else (None, 0))
        _lib.check(self.lib.mx_gated_delta_rule(ctypes.byref(args), ptr, nbytes, stream),
                   "mx_gated_delta_rule")

    def close(self) -> None:
        if self._ws is not None:
            self.backend.free_device(self._ws)
            self._ws = None
