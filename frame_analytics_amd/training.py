"""Operators of a training step beside the losses -- the public functions.

A network that is trained with ``1 - fa.ssim(...)`` or the other losses runs its
attention and its weight updates on the same card.  These are the ones that a
restoration transformer needs and that plain torch serves worst: attention with a
learned relative position bias (:func:`relative_attention`, differentiable, table
included), that bias by itself (:func:`relative_bias`) and the orthogonalised update
of weight matrices (:func:`orthogonalize`).  The reference has none of them.

Routing is that of the metrics: float16, bfloat16 and float32 GPU tensors run the
gfx950 kernels behind ``include/fa_train_abi.h`` (through
:mod:`frame_analytics_amd.backend_training`); CPU tensors, float64 and
``backend_hint="torch"`` run the eager PyTorch path below; ``backend_hint="native"``
raises instead of taking it.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import backend, backend_training
from .functional import _no_autocast

__all__ = ["LinePositions", "GridPositions", "relative_attention", "relative_bias",
           "orthogonalize"]

#: most differences of positions with a table row of their own (FA_REL_MAX)
_MOST_SLOTS = 4225


# --------------------------------------------------------------------------- #
# positions
# --------------------------------------------------------------------------- #


@functools.lru_cache(maxsize=256)
def _bucket_starts(n: int, max_distance: int) -> Tuple[int, ...]:
    """Where rows n // 2 + 1, n // 2 + 2, ... of a direction's n rows start."""
    half, wide = n // 2, n - n // 2
    starts, at = [], half
    for j in range(1, wide):
        least = half ** (wide - j) * max_distance ** j
        # the smallest whole number with at ** wide >= least
        at = max(at, math.floor(math.exp(math.log(least) / wide)) - 1)
        while at ** wide < least:
            at += 1
        starts.append(at)
    return tuple(starts)


@dataclass(frozen=True)
class LinePositions:
    """Tokens on a line: the table row of query ``i`` and key ``j`` goes by their
    distance, near ones each their own, farther ones in ``num_buckets`` buckets whose
    width grows with the distance, all from ``max_distance`` on the same.

    With ``bidirectional`` half of the buckets are for keys after the query; without
    it keys after the query share the row of distance 0 (causal attention does not
    see them).  Of the ``n`` rows of one direction the first ``n // 2`` hold one
    distance each; row ``n // 2 + j`` starts at distance ``(n // 2) * (max_distance /
    (n // 2)) ** (j / (n - n // 2))``, compared exactly, in whole numbers.
    """

    num_buckets: int = 32
    max_distance: int = 128
    bidirectional: bool = True

    grid_w = 0

    def __init__(self, num_buckets: int = 32, max_distance: int = 128, *,
                 bidirectional: bool = True):
        n = num_buckets // 2 if bidirectional else num_buckets
        if n < 2 or (bidirectional and num_buckets % 2):
            raise ValueError(f"num_buckets={num_buckets} is too small or odd for "
                             f"bidirectional={bidirectional}")
        if max_distance <= n // 2:
            raise ValueError(f"max_distance={max_distance} must be more than the "
                             f"{n // 2} distances with a bucket of their own")
        for name, value in (("num_buckets", int(num_buckets)), ("max_distance", int(max_distance)),
                            ("bidirectional", bool(bidirectional))):
            object.__setattr__(self, name, value)
        # about the logarithm of the last bucket's start: a search for the exact one would
        # take as long as it is far
        wide = n - n // 2
        about = (math.log(n // 2) + (wide - 1) * math.log(self.max_distance)) / wide
        starts = _bucket_starts(n, self.max_distance) if about < math.log(2 * _MOST_SLOTS) else ()
        object.__setattr__(self, "_starts", starts)
        object.__setattr__(self, "_far", starts[-1] if starts else n // 2)
        if about >= math.log(2 * _MOST_SLOTS) or self.slots > _MOST_SLOTS:
            raise ValueError(f"about {math.exp(min(about, 700)):.3g} distances each way before the "
                             f"last bucket; at most {_MOST_SLOTS} in all are supported")

    @property
    def rows(self) -> int:
        return self.num_buckets

    @property
    def lo(self) -> int:
        return -self._far if self.bidirectional else 0

    @property
    def slots(self) -> int:
        return (2 if self.bidirectional else 1) * self._far + 1

    def _row(self, delta: int) -> int:
        """Of a query ``delta`` positions after its key."""
        n = self.num_buckets // 2 if self.bidirectional else self.num_buckets
        base = n if self.bidirectional and delta < 0 else 0
        dist = abs(delta) if self.bidirectional else max(0, delta)
        if dist < n // 2:
            return base + dist
        return base + n // 2 + sum(dist >= s for s in self._starts)

    def row_of(self) -> List[int]:
        return [self._row(self.lo + t) for t in range(self.slots)]

    def check(self, q_len: int, k_len: int, q_start) -> None:
        del q_len, k_len, q_start


@dataclass(frozen=True)
class GridPositions:
    """The ``height * width`` tokens of a window, row by row: each difference of
    coordinates has a table row, ``(yi - yj + height - 1) * (2 * width - 1) + xi - xj +
    width - 1``."""

    height: int
    width: int

    def __post_init__(self):
        if self.height < 1 or self.width < 1:
            raise ValueError(f"a window needs a height and a width, got {self.height}x{self.width}")
        if self.rows > _MOST_SLOTS:
            raise ValueError(f"a {self.height}x{self.width} window has {self.rows} differences of "
                             f"coordinates; at most {_MOST_SLOTS} are supported")

    @property
    def grid_w(self) -> int:
        return self.width

    @property
    def rows(self) -> int:
        return (2 * self.height - 1) * (2 * self.width - 1)

    @property
    def lo(self) -> int:
        return -(self.rows // 2)

    @property
    def slots(self) -> int:
        return self.rows

    def row_of(self) -> List[int]:
        return list(range(self.rows))

    def check(self, q_len: int, k_len: int, q_start) -> None:
        n = self.height * self.width
        if q_len != n or k_len != n:
            raise ValueError(f"a {self.height}x{self.width} window has {n} tokens, got {q_len} "
                             f"queries and {k_len} keys")
        if torch.is_tensor(q_start) or q_start != 0:
            raise ValueError("q_start belongs to positions on a line")


Positions = Union[LinePositions, GridPositions]


def _codes(positions: Positions, n: int, device) -> torch.Tensor:
    t = torch.arange(n, device=device)
    w = positions.grid_w
    return t + (w - 1) * (t // w) if w else t


def _pair_rows(positions: Positions, q_len: int, k_len: int, q_start, device) -> torch.Tensor:
    """The table row of each pair: ``(1 or batch, q_len, k_len)``."""
    start = torch.as_tensor(q_start, device=device).reshape(-1, 1)
    cq = start + _codes(positions, q_len, device)
    delta = cq[..., None] - _codes(positions, k_len, device)
    row_of = torch.tensor(positions.row_of(), device=device)
    return row_of[(delta - positions.lo).clamp(0, positions.slots - 1)]


def _check_positions(positions, table) -> None:
    if not isinstance(positions, (LinePositions, GridPositions)):
        raise TypeError("positions must be LinePositions or GridPositions, got "
                        f"{type(positions).__name__}")
    if table.ndim != 2 or table.shape[0] != positions.rows or table.shape[1] < 1:
        raise ValueError(f"expected a table of ({positions.rows}, heads), got "
                         f"{tuple(table.shape)}")
    if not table.is_floating_point():
        raise TypeError(f"the table must be floating point, got {table.dtype}")


def _route(t: torch.Tensor, what: str, backend_hint: str) -> bool:
    """True: the kernels; False: the eager path, noted as such."""
    if backend_hint not in ("auto", "native", "torch"):
        raise ValueError(f"unknown backend_hint {backend_hint!r}")
    if backend_hint != "torch" and backend_training.serves(t):
        return True
    if backend_hint == "native":
        raise RuntimeError(f"{what}: no native kernel for {t.dtype} on {t.device}")
    backend.note_portable(what, t)
    return False


# --------------------------------------------------------------------------- #
# the bias by itself
# --------------------------------------------------------------------------- #


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, positions, q_len, k_len, q_start):
        ctx.args = (table.shape[0], positions, q_start)
        return backend_training.rel_bias(table, positions, q_len, k_len, q_start)

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        return backend_training.rel_bias_backward(up, *ctx.args), None, None, None, None


def relative_bias(table: torch.Tensor, positions: Positions, q_len: int,
                  k_len: Optional[int] = None, *, q_start: int = 0,
                  backend_hint: str = "auto") -> torch.Tensor:
    """The learned bias of every pair, ``(heads, q_len, k_len)`` in the table's type:
    ``table[row(i, j), head]``, query ``i`` standing at position ``q_start + i`` of a
    line.  ``table`` is ``(positions.rows, heads)``; its gradient is summed in float32
    in a fixed order (the same bits from run to run).

    For an attention that takes its bias as a tensor; :func:`relative_attention` adds
    it without forming it.
    """
    k_len = q_len if k_len is None else k_len
    _check_positions(positions, table)
    if q_len < 0 or k_len < 0:
        raise ValueError(f"lengths must not be negative, got {q_len} and {k_len}")
    positions.check(q_len, k_len, q_start)
    if torch.is_tensor(q_start):
        raise TypeError("relative_bias takes one q_start, an int")
    if q_len == 0 or k_len == 0:
        return table.sum() * table.new_zeros((table.shape[1], q_len, k_len))
    if _route(table, "relative_bias", backend_hint):
        return _RelativeBias.apply(table, positions, int(q_len), int(k_len), int(q_start))
    rows = _pair_rows(positions, q_len, k_len, q_start, table.device)[0]
    return table[rows].permute(2, 0, 1).contiguous()


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #


class _RelativeAttention(torch.autograd.Function):
    """Keeps q, k, v, the output and two numbers of each row's softmax; the backward pass
    forms the weights again from them."""

    @staticmethod
    def forward(ctx, q, k, v, table, plan):
        out, lse, kept = backend_training.rel_attention(q, k, v, table, plan, True)
        extra = [t for t in (plan.mask, plan.key_lengths, plan.q_starts) if t is not None]
        ctx.save_for_backward(*kept, out, lse, *extra)
        ctx.plan = plan
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, table, out, lse = ctx.saved_tensors[:6]
        dq, dk, dv, dtable = backend_training.rel_attention_backward(
            g, q, k, v, out, lse, table, ctx.plan, ctx.needs_input_grad[3])
        grads = (dq, dk, dv, dtable)
        return (*(x if want else None for x, want in zip(grads, ctx.needs_input_grad)), None)


def _tangents(*tensors: torch.Tensor) -> bool:
    """Whether any carries a forward-mode tangent, which autograd then refuses (there is no
    formula for it here): called past autograd, the kernels would drop it without a word."""
    return (forward_ad._current_level >= 0
            and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors))


class _Nothing(torch.autograd.Function):
    """No pairs: zeros, and zero gradients."""

    @staticmethod
    def forward(ctx, *inputs):
        ctx.save_for_backward(*inputs)
        return torch.zeros_like(inputs[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return tuple(torch.zeros_like(t) for t in ctx.saved_tensors)


def _portable_attention(q, k, v, table, plan):
    work = torch.float64 if q.dtype == torch.float64 else torch.float32
    group, lq, lk = q.shape[1] // k.shape[1], q.shape[2], k.shape[2]
    start = plan.q_starts if plan.q_starts is not None else plan.q_start
    dev = q.device
    with _no_autocast(q):
        keys = torch.arange(lk, device=dev)
        hidden = torch.zeros(1, 1, lq, lk, dtype=torch.bool, device=dev)
        if plan.key_lengths is not None:
            past = keys >= plan.key_lengths[:, None]  # never read, whatever it holds
            k, v = (t.masked_fill(past[:, None, :, None], 0) for t in (k, v))
            hidden = hidden | past[:, None, None, :]
        if plan.causal:
            at = (torch.as_tensor(start, device=dev).reshape(-1, 1)
                  + torch.arange(lq, device=dev))
            hidden = hidden | (keys > at[..., None])[:, None]
        if plan.mask is not None:
            hidden = hidden | ~plan.mask.repeat(q.shape[0] // plan.mask.shape[0], 1, 1, 1)
        bias = table.to(work)[_pair_rows(plan.positions, lq, lk, start, dev)].permute(0, 3, 1, 2)
        kk, vv = (t.to(work).repeat_interleave(group, dim=1) for t in (k, v))
        s = (q.to(work) @ kk.transpose(-1, -2)) * plan.scale + bias
        s = s.masked_fill(hidden, -math.inf)
        top = s.detach().amax(-1, keepdim=True)
        p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
        total = p.sum(-1, keepdim=True)
        return ((p @ vv) / total.masked_fill(total == 0, 1.0)).to(q.dtype)


def _check_attention(q, k, v, table, positions, mask, key_lengths, q_start):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.ndim != 4:
            raise ValueError(f"expected {name} of (batch, heads, tokens, dim), got shape "
                             f"{tuple(t.shape)}")
        if not t.is_floating_point():
            raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"dtype mismatch: {q.dtype}, {k.dtype}, {v.dtype}")
    b, h, lq, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}, "
                         f"v {tuple(v.shape)}")
    hk, lk = k.shape[1], k.shape[2]
    if hk < 1 or h % hk:
        raise ValueError(f"{h} query heads cannot share {hk} key heads")
    if not 1 <= d <= 128:
        raise ValueError(f"head dimensions of 1 to 128 are supported, got {d}")
    _check_positions(positions, table)
    if table.shape[1] != h:
        raise ValueError(f"the table has {table.shape[1]} heads, q has {h}")
    positions.check(lq, lk, q_start)
    rest = [("k", k), ("v", v), ("table", table)]
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be boolean (True: attend), got {mask.dtype}")
        if mask.ndim == 2:
            mask = mask[None, None]
        if (mask.ndim != 4 or mask.shape[1] not in (1, h) or tuple(mask.shape[2:]) != (lq, lk)
                or mask.shape[0] < 1 or b % mask.shape[0]):
            raise ValueError(f"expected a mask of ({lq}, {lk}) or (m, 1 or {h}, {lq}, {lk}) with m "
                             f"dividing the batch of {b}, got {tuple(mask.shape)}")
        rest.append(("mask", mask))
    for name, t in (("key_lengths", key_lengths), ("q_start", q_start)):
        if not torch.is_tensor(t):
            continue
        if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (b,):
            raise ValueError(f"{name} must be an integer tensor of ({b},), got {t.dtype} of "
                             f"{tuple(t.shape)}")
        rest.append((name, t))
    for name, t in rest:
        if t.device != q.device:
            raise ValueError(f"device mismatch: q on {q.device}, {name} on {t.device}")
    return mask


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                       positions: Positions, *, scale: Optional[float] = None,
                       causal: bool = False, mask: Optional[torch.Tensor] = None,
                       key_lengths: Optional[torch.Tensor] = None,
                       q_start: Union[int, torch.Tensor] = 0,
                       backend_hint: str = "auto") -> torch.Tensor:
    """``softmax(scale * q k^T + bias) v`` with the learned relative position bias
    ``table[row(i, j), head]``; differentiable (once) in q, k, v and the table.

    ``q`` is ``(batch, heads, tokens, dim)``, ``k`` and ``v`` ``(batch, key heads, keys,
    dim)`` with the key heads dividing the heads (each is shared by neighbouring query
    heads); any strides, the last dimension contiguous (else copied, as is a view of which
    256 tokens span 2 GiB); ``dim`` up to 128.  The result is laid out as q is (as its copy
    where it was copied).  A table of another type than q counts in float32, as
    does its gradient (a float32 parameter beside 16-bit activations loses nothing).

    ``scale`` defaults to ``dim ** -0.5``.  A pair counts where all of these allow it:
    ``causal`` (the key's position is not after the query's), ``key_lengths`` ((batch,)
    integers: the keys from there on are never read, so they may hold anything) and
    ``mask`` (boolean, True: attend; ``(tokens, keys)`` or ``(m, 1 or heads, tokens,
    keys)`` with batch entry b reading ``mask[b % m]``, as the windows of a shifted
    frame repeat).  A query for which no key counts gets zeros, and zero gradients.

    ``q_start`` is the position of the first query on the line, one for all or
    ``(batch,)`` integers: a decoding step passes one new token against its cache with
    ``q_start=key_lengths - 1``.

    The scores, the softmax and all sums are float32; its weights are rounded to q's
    type for the product with v, the weights and the scores' gradient for the gradients'
    products, and results once.  Results and gradients are the same bits from run to run.
    """
    mask = _check_attention(q, k, v, table, positions, mask, key_lengths, q_start)
    if table.dtype != q.dtype:
        table = table.to(torch.float64 if q.dtype == torch.float64 else torch.float32)
    if q.numel() == 0 or k.shape[2] == 0:
        return _Nothing.apply(q, k, v, table)
    plan = backend_training.AttentionPlan(
        positions, float(q.shape[3] ** -0.5 if scale is None else scale), bool(causal), mask,
        key_lengths, q_start)
    if _route(q, "relative_attention", backend_hint):
        if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                         or table.requires_grad)) or _tangents(q, k, v, table):
            return _RelativeAttention.apply(q, k, v, table, plan)
        return backend_training.rel_attention(q, k, v, table, plan, False)[0]
    return _portable_attention(q, k, v, table, plan)


# --------------------------------------------------------------------------- #
# orthogonalised updates
# --------------------------------------------------------------------------- #


@functools.lru_cache(maxsize=256)
def _held_in_float16(a: float, b: float, c: float, steps: int) -> bool:
    """Whether the kernels' float16 operands hold what these coefficients lead to (the
    entry point refuses the rest).

    A step takes each singular value ``s`` to ``|a s + b s^3 + c s^5|`` by itself, from
    (0, 1] on, so the largest possible one is the largest value over the range before: at
    its end or at a zero of the derivative.  X and ``A`` are held times 2048, ``b A + c
    A^2`` times 1024; a range is widened by 1/512, more than rounding adds.
    """
    most, noise = 65504 * 0.99, 1 + 1 / 512
    top, before = noise, 0.0
    for _ in range(steps):
        if not (1 / 64 <= top and 2048 * max(top, top * top) <= most):
            return False
        turns = [top * top]  # squares of singular values
        if c:
            disc = 9 * b * b - 20 * a * c
            turns.append(-b / (2 * c))
            if disc >= 0:
                turns += [(-3 * b + r) / (10 * c) for r in (math.sqrt(disc), -math.sqrt(disc))]
        elif b:
            turns.append(-a / (3 * b))
        turns = [u for u in turns if 0 < u <= top * top]
        if not 1024 * max(abs(b * u + c * u * u) for u in turns) <= most:
            return False
        after = max(math.sqrt(u) * abs(a + b * u + c * u * u) for u in turns)
        if not after < 1e30:
            return False
        if after == before:  # so will every further step's
            return True
        before, top = after, after * noise
    return True


@torch.no_grad()
def orthogonalize(update: torch.Tensor, *, steps: int = 5,
                  coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7,
                  backend_hint: str = "auto") -> torch.Tensor:
    """The update with its singular values driven towards one: ``X <- a X + (b A + c
    A^2) X`` with ``A = X X^T``, ``steps`` times from ``update / (norm + eps)`` (the
    Frobenius norm).

    ``update`` is a matrix or a stack of matrices ``(..., rows, cols)`` (flatten a
    convolution's weight to ``(out, in * kh * kw)`` first); the result has its shape
    and type and carries no gradient.  The default coefficients lift small singular
    values fast and leave them between 0.7 and 1.2; ``(1.875, -1.25, 0.375)``
    converges to one.

    The kernels hold their operands in float16: iterates of singular values within [1/64,
    5.6] (the largest of each step but the last) with ``|b s^2 + c s^4|`` below 63.
    Coefficients that leave this run the eager path, in float32 (``backend_hint="native"``
    refuses them).

    bfloat16 runs single float16 products (the result is within 1.5e-3 of exact before
    its rounding), float16 and float32 pairs of float16 (22 bits).
    """
    if update.ndim < 2:
        raise ValueError(f"expected a matrix or a stack of them, got shape {tuple(update.shape)}")
    if not update.is_floating_point():
        raise TypeError(f"update must be floating point, got {update.dtype}")
    if steps < 1:
        raise ValueError(f"steps must be at least 1, got {steps}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps}")
    a, b, c = (float(x) for x in coefficients)
    if update.numel() == 0:
        return torch.empty_like(update)
    if (backend_hint in ("auto", "native") and backend_training.serves(update)
            and not _held_in_float16(a, b, c, int(steps))):
        if backend_hint == "native":
            raise RuntimeError("orthogonalize: the kernels' float16 operands do not hold the "
                               f"iterates of the coefficients {(a, b, c)} over {steps} steps")
        backend_hint = "torch"
    if _route(update, "orthogonalize", backend_hint):
        return backend_training.orthogonalize(update, int(steps), (a, b, c), float(eps))
    with _no_autocast(update):
        x = update.to(torch.float64 if update.dtype == torch.float64 else torch.float32)
        tall = x.shape[-2] > x.shape[-1]
        if tall:
            x = x.mT
        x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
        for _ in range(steps):
            gram = x @ x.mT
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        return (x.mT if tall else x).to(update.dtype).contiguous()
