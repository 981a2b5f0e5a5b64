"""Dispatch of the training operators to the gfx950 kernels: tensors in, raw
pointers across ``include/fa_train_abi.h``.

Every buffer -- outputs, what the backward pass reads, workspaces -- is allocated here
through torch's caching allocator on the caller's current stream, and every launch goes
to that stream, as in :mod:`frame_analytics_amd.backend`.  A kernel that refuses a call
raises :class:`~frame_analytics_amd.backend.KernelError`.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import backend
from .backend import _DTYPE_CODE, _ptr, _run, _site

DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_MOST = 1 << 30  # positions and lengths are taken as within +-2^30


def serves(t: torch.Tensor) -> bool:
    """Whether the kernels take a call on ``t``."""
    return t.dtype in DTYPES and backend._gpu_ext(t) is not None


_row_tables: dict = {}


def _row_of(positions, device: torch.device) -> torch.Tensor:
    """The table row of each slot, on the device: one per description of positions
    (a value, not a tensor), so made once.  Making it copies from the host: a graph
    capture needs an eager call before it.

    It is kept for the life of the process (17 KB at most): a captured graph holds its
    address and no reference, and launches on other streams may still read it, so memory
    given back would be read as rows of the table by a replay."""
    rows = _row_tables.get((positions, device))
    if rows is None:  # (of two threads that make it, both take the first's)
        rows = _row_tables.setdefault(
            (positions, device), torch.tensor(positions.row_of(), dtype=torch.int32, device=device))
    return rows


@functools.lru_cache(maxsize=256)
def _bytes(name: str, *shape: int) -> int:
    out = ctypes.c_int64(0)
    _run(name, *shape, ctypes.byref(out))
    return int(out.value)


def _workspace(name: str, device, *shape: int):
    n = _bytes(name, *shape)
    return (torch.empty(n, device=device, dtype=torch.uint8), n) if n else (None, 0)


def _unit(t: torch.Tensor) -> torch.Tensor:
    """``t`` (batch, heads, tokens, dim), copied unless its last dimension has stride 1 and
    256 tokens lie within the 2^31 bytes that a kernel's offsets reach."""
    near = t.shape[2] == 1 or 256 * t.element_size() * t.stride(2) < 1 << 31
    return t if near and (t.stride(-1) == 1 or t.shape[-1] == 1) else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    """An output laid out as ``t`` is where that is dense with unit last stride."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _int32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32:
        t = t.clamp(-_MOST, _MOST).to(torch.int32)
    return t.contiguous()


def _strides(*views: torch.Tensor):
    """The first three of each; 0 where there is one element, whose stride says nothing."""
    flat = [s if n > 1 else 0 for v in views for n, s in zip(v.shape[:3], v.stride()[:3])]
    return (ctypes.c_int64 * len(flat))(*flat)


# --------------------------------------------------------------------------- #
# the bias by itself
# --------------------------------------------------------------------------- #


def rel_bias(table, positions, q_len: int, k_len: int, q_start: int) -> torch.Tensor:
    table = table.contiguous()
    rows, heads = table.shape
    out = torch.empty((heads, q_len, k_len), dtype=table.dtype, device=table.device)
    row_of = _row_of(positions, table.device)
    _run("fa_gpu_rel_bias", table.data_ptr(), _DTYPE_CODE[table.dtype], rows, heads, q_len, k_len,
         row_of.data_ptr(), positions.lo, positions.slots, positions.grid_w, q_start,
         out.data_ptr(), *_site(table))
    return out


def rel_bias_backward(up, rows: int, positions, q_start: int) -> torch.Tensor:
    heads, q_len, k_len = up.shape
    out = torch.empty((rows, heads), dtype=up.dtype, device=up.device)
    row_of = _row_of(positions, up.device)
    ws, n = _workspace("fa_gpu_rel_bias_workspace", up.device, heads, q_len, k_len,
                       positions.slots)
    _run("fa_gpu_rel_bias_backward", up.data_ptr(), _strides(up), _DTYPE_CODE[up.dtype], rows,
         heads, q_len, k_len, row_of.data_ptr(), positions.lo, positions.slots, positions.grid_w,
         q_start, out.data_ptr(), _ptr(ws), n, *_site(up))
    return out


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #


def _types(q: torch.Tensor, table: torch.Tensor) -> int:
    """The dtype code of an attention; FA_TABLE_F32 where the table is wider than q."""
    return _DTYPE_CODE[q.dtype] | (0x100 if table.dtype != q.dtype else 0)


class AttentionPlan:
    """What a call's forward and backward pass hand to the library alike."""

    __slots__ = ("positions", "scale", "causal", "mask", "key_lengths", "q_start", "q_starts")

    def __init__(self, positions, scale, causal, mask, key_lengths, q_start):
        self.positions, self.scale, self.causal, self.mask = positions, scale, causal, mask
        self.key_lengths = _int32(key_lengths)
        tensor = torch.is_tensor(q_start)
        self.q_starts = _int32(q_start) if tensor else None
        self.q_start = 0 if tensor else q_start

    def tail(self, table, row_of):
        """The arguments from ``table`` to ``scale``."""
        p, m = self.positions, self.mask
        strides = None
        if m is not None:
            s = m.stride()
            strides = (ctypes.c_int64 * 4)(s[0], 0 if m.shape[1] == 1 else s[1], s[2], s[3])
        return (table.data_ptr(), table.shape[0], row_of.data_ptr(), p.lo, p.slots, p.grid_w,
                self.q_start, _ptr(self.q_starts), _ptr(self.key_lengths), _ptr(m),
                1 if m is None else m.shape[0], strides, int(self.causal), self.scale)


def rel_attention(q, k, v, table, plan: AttentionPlan, need_lse: bool):
    """``(out, what is kept of the rows' softmax, the tensors as the kernels read them)``."""
    q, k, v, table = _unit(q), _unit(k), _unit(v), table.contiguous()
    b, h, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    out = _like(q)
    lse = None
    if need_lse:  # two numbers a row, and on a line what the rounding of a 16-bit output left
        n = 2 * b * h * lq
        if q.dtype != torch.float32 and not plan.positions.grid_w:
            n = (n + 3) // 4 * 4 + (b * h * lq * d + 1) // 2
        lse = torch.empty(n, dtype=torch.float32, device=q.device)
    dev, stream = _site(q)
    ws, n = _workspace("fa_gpu_rel_attention_workspace", q.device, b, h, hk, lq, lk, d,
                       plan.positions.slots, dev)
    _run("fa_gpu_rel_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), _types(q, table),
         b, h, hk, lq, lk, d, _strides(q, k, v, out),
         *plan.tail(table, _row_of(plan.positions, q.device)), out.data_ptr(), _ptr(lse), _ptr(ws),
         n, dev, stream)
    return out, lse, (q, k, v, table)


def rel_attention_backward(g, q, k, v, out, lse, table, plan: AttentionPlan, need_table: bool):
    g = _unit(g)
    b, h, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    dq, dk, dv = _like(q), _like(k), _like(v)
    dtable = torch.empty_like(table) if need_table else None
    dev, stream = _site(q)
    ws, n = _workspace("fa_gpu_rel_attention_backward_workspace", q.device, b, h, hk, lq, lk, d,
                       plan.positions.slots, plan.positions.grid_w, int(need_table), dev)
    _run("fa_gpu_rel_attention_backward", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
         g.data_ptr(), lse.data_ptr(), _types(q, table), b, h, hk, lq, lk, d,
         _strides(q, k, v, out, g, dq, dk, dv),
         *plan.tail(table, _row_of(plan.positions, q.device)), dq.data_ptr(), dk.data_ptr(),
         dv.data_ptr(), _ptr(dtable), _ptr(ws), n, dev, stream)
    return dq, dk, dv, dtable


# --------------------------------------------------------------------------- #
# orthogonalised updates
# --------------------------------------------------------------------------- #


def orthogonalize(g, steps: int, coefficients, eps: float) -> torch.Tensor:
    g = g.contiguous()
    rows, cols = g.shape[-2:]
    batch = g.numel() // (rows * cols)
    out = torch.empty_like(g)
    code = _DTYPE_CODE[g.dtype]
    ws, n = _workspace("fa_gpu_orthogonalize_workspace", g.device, code, batch, rows, cols)
    _run("fa_gpu_orthogonalize", g.data_ptr(), code, batch, rows, cols, steps, *coefficients, eps,
         out.data_ptr(), _ptr(ws), n, *_site(g))
    return out
