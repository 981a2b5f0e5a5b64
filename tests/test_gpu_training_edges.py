"""The training operators' kernels where their inputs are extreme: NaN, biases of the
type's limits, wide strides, many matrices, coefficients that overflow.  Tolerances as in
``test_gpu_training_ops``; what a test adds to them is derived in it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import frame_analytics_amd as fa
from oracle import training as ref
from tests.test_gpu_training_ops import DT, STEEP, UNIT, attention_case, near, normal, run_attention

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- #
# NaN
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lq,lk", [(1, 100), (1, 2500), (3, 700)])
def test_a_nan_query_answers_nan(gpu, dt, lq, lk):
    """Few queries against a cache, dealt out or not: the row of a NaN query, and it
    alone, is NaN, and so are its gradients."""
    b, h, hk, d = 2, 4, 2, 64
    pos = fa.LinePositions(32, 128, bidirectional=False)
    rows = ref.line_rows(lq, lk, lk - lq, 32, 128, False)
    tensors, g, _ = attention_case(DT[dt], b, h, hk, lq, lk, d, pos, rows, q_start=lk - lq)
    clean = run_attention(tensors, g, pos, q_start=lk - lq)
    tensors[0][1, 2, 0, 5] = float("nan")
    got = run_attention(tensors, g, pos, q_start=lk - lq)
    with torch.no_grad():
        only = fa.relative_attention(*(t.cuda() for t in tensors), pos, q_start=lk - lq)
    bad = torch.zeros(b, h, lq, dtype=torch.bool, device="cuda")
    bad[1, 2, 0] = True
    for out in (got[0], only, got[1]):
        assert torch.isnan(out[bad]).all() and not torch.isnan(out[~bad]).any()
    assert torch.equal(got[0][~bad], clean[0][~bad]) and torch.equal(only[~bad], clean[0][~bad])
    for x in got[2:4]:  # every key of its key head
        assert torch.isnan(x[1, 1]).all() and not torch.isnan(x[0]).any()
        assert not torch.isnan(x[1, 0]).any()
    assert torch.isnan(got[4][:, 2]).any() and not torch.isnan(got[4][:, [0, 1, 3]]).any()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("last", [128, 256, 640])
def test_a_nan_key_that_stands_alone_in_its_run(gpu, dt, last):
    """Keys are dealt out in runs of whole blocks: the one key past them is NaN."""
    b, h, hk, lk, d = 2, 4, 2, 1000, 32
    pos = fa.LinePositions(8, 20)
    gen = torch.Generator().manual_seed(last)
    q, k, v = (normal(gen, DT[dt], b, n, m, d).transpose(1, 2).cuda()
               for n, m in ((1, h), (lk, hk), (lk, hk)))
    table = normal(gen, DT[dt], 8, h).cuda()
    lens = torch.tensor([last + 1, last], dtype=torch.int32, device="cuda")
    k[:, 1, last] = float("nan")
    out = fa.relative_attention(q, k, v, table, pos, key_lengths=lens)
    assert torch.isnan(out[0, 2:]).all()                       # the heads of key head 1
    assert not torch.isnan(out[0, :2]).any() and not torch.isnan(out[1]).any()


def hidden_case(form, dt):
    """q, k, v, table, positions and arguments of a call with hidden pairs in each tile."""
    gen = torch.Generator().manual_seed(11)
    if form == "window":
        b, h, lq, lk, pos = 3, 2, 64, 64, fa.GridPositions(8, 8)
    elif form == "wide window":
        b, h, lq, lk, pos = 2, 2, 144, 144, fa.GridPositions(12, 12)
    else:
        b, h, pos = 2, 2, fa.LinePositions(8, 20)
        lq, lk = {"line": (80, 80), "few": (4, 600), "one run": (4, 100)}[form]
    q, k, v = (normal(gen, DT[dt], b, h, n, 32) for n in (lq, lk, lk))
    mask = torch.rand(1, 1, lq, lk, generator=gen) < 0.7
    return q, k, v, torch.zeros(pos.rows, h, dtype=DT[dt]), pos, mask


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("form", ["window", "wide window", "line", "few", "one run"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_weight_too_small_for_the_type_still_sees(gpu, dt, form, bad):
    """A value that is not finite reaches every query that sees its key, however little
    that key counts (a weight of exp(-25): zero in float16, not in float32), and none
    that does not."""
    q, k, v, table, pos, mask = hidden_case(form, dt)
    q[..., 0], k[..., 0] = 5.0, 0.0
    k[:, :, 30, 0] = -5.0
    q[..., 1:] *= 0.1
    v[:, :, 30, 7] = bad
    mask[..., 0, 30], mask[..., 1, 30] = True, False
    out = fa.relative_attention(*(t.cuda() for t in (q, k, v, table)), pos, scale=1.0,
                                mask=mask.cuda()).cpu()
    see = mask[0, 0, :, 30]
    assert not torch.isfinite(out[:, :, see, 7]).any()
    assert torch.isfinite(out[:, :, ~see]).all()
    other = torch.arange(32) != 7
    assert torch.isfinite(out[..., other]).all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("form", ["window", "wide window", "few", "one run"])
def test_what_no_query_sees_may_hold_anything(gpu, dt, form):
    """NaN and infinities at keys that the mask or the lengths hide from all, and in
    queries that see nothing, reach no result."""
    q, k, v, table, pos, mask = hidden_case(form, dt)
    gen = torch.Generator().manual_seed(12)
    table = normal(gen, DT[dt], *table.shape)
    g = normal(gen, DT[dt], *q.shape)
    b, h, lq, lk = *q.shape[:3], k.shape[2]
    mask[..., 2, :] = False
    mask[..., :, 9] = False
    lens = torch.tensor([lk, lk - 13, lk // 2][:b], dtype=torch.int32)
    see = ref.visible(b, h, lq, lk, mask=mask.numpy(), key_lengths=lens.numpy())
    rows = ref.grid_rows(pos.height, pos.width) if pos.grid_w else ref.line_rows(lq, lk, 0, 8, 20)
    want = ref.attention(*(t.double().numpy() for t in (q, k, v, table)), rows, see, 32 ** -0.5,
                         g.double().numpy())
    q[:, :, 2], g[:, :, 2] = float("nan"), float("inf")
    k[:, :, 9], v[:, :, 9] = float("inf"), float("nan")
    for i, n in enumerate(lens.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), -float("inf")
    got = run_attention((q, k, v, table), g, pos, mask=mask.cuda(), key_lengths=lens.cuda())
    for name, x, y, t in zip(("out", "dq", "dk", "dv", "dtable"), got, want, (2, 4, 4, 4, 4)):
        near(x, y, t * UNIT[dt], name)


# --------------------------------------------------------------------------- #
# biases at the type's limits
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("form", ["line", "causal", "few", "one", "window", "wide window"])
@pytest.mark.parametrize("extreme", ["lowest", "largest", "-inf"])
def test_biases_at_the_limits_of_the_type(gpu, dt, form, extreme):
    """Head 0: every entry; head 1: every other; head 2: the farthest; head 3: none.  A
    row of equal extremes has equal weights, whatever its scores (which such a bias
    rounds away); a row of -inf alone sees nothing."""
    gen = torch.Generator().manual_seed(21)
    b, h, d, kw, start = 2, 4, 32, {}, 0
    if form == "window":
        pos, lq = fa.GridPositions(8, 8), 64
        lk, rows = lq, ref.grid_rows(8, 8)
    elif form == "wide window":
        pos, lq = fa.GridPositions(9, 10), 90
        lk, rows = lq, ref.grid_rows(9, 10)
    else:
        pos = fa.LinePositions(8, 20)
        lq, lk = {"line": (150, 400), "causal": (300, 300), "few": (5, 700), "one": (1, 90)}[form]
        start = 40 if form in ("few", "one") else 0
        rows = ref.line_rows(lq, lk, start, 8, 20)
        kw = {"causal": form == "causal", "q_start": start}
    q, k, v, g = (normal(gen, DT[dt], b, h, n, d) for n in (lq, lk, lk, lq))
    table = normal(gen, DT[dt], pos.rows, h)
    info = torch.finfo(DT[dt])
    value = {"lowest": info.min, "largest": info.max, "-inf": -float("inf")}[extreme]
    table[:, 0] = value
    table[::2, 1] = value
    table[-1, 2] = value
    see = ref.visible(b, h, lq, lk, causal=form == "causal", q_start=start)
    finite = np.where(np.isinf(table.double().numpy()), 0.0, table.double().numpy())
    if extreme == "-inf":  # such a pair is hidden
        see = see & ~np.isinf(table.double().numpy())[rows].transpose(2, 0, 1)[None]
    want = ref.attention(*(t.double().numpy() for t in (q, k, v)), finite, rows, see, d ** -0.5,
                         g.double().numpy())
    got = run_attention((q, k, v, table), g, pos, **kw)
    # float16's limits round a score by 65504 2^-24, and as much the maximum beside it
    more = 4 * 65504 * 2.0 ** -24 if dt == "f16" and extreme != "-inf" else 0.0
    for name, x, y, t in zip(("out", "dq", "dk", "dv", "dtable"), got, want, (2, 4, 4, 4, 4)):
        near(x, y, t * UNIT[dt] / (1 if dt == "f32" else 2) + more, name)


def test_large_biases_keep_their_order(gpu):
    """Entries near the limits that differ: the larger takes the whole weight."""
    pos = fa.LinePositions(4, 5, bidirectional=False)
    top = torch.finfo(torch.float32).max
    v = torch.eye(12, device="cuda")[None, None]
    z = torch.zeros(1, 1, 12, 12, device="cuda")
    for values in ((-top, -0.9 * top, -0.5 * top, -0.25 * top), (top, 0.99 * top, 0.5 * top, 0.2 * top),
                   (-0.25 * top, -0.24 * top, -0.26 * top, -0.3 * top), (1e30, 1.1e30, -1e30, 1e37)):
        table = torch.tensor(values, device="cuda")[:, None]
        out = fa.relative_attention(z, z, v, table, pos, causal=True)[0, 0]
        bias = fa.relative_bias(table, pos, 12)[0].double()
        bias = bias.masked_fill(torch.ones_like(bias).triu(1).bool(), -float("inf"))
        want = torch.softmax(bias, -1)
        assert torch.equal(out.double() > 0, want > 0), values
        near(out, want.cpu().numpy(), 2e-5)


# --------------------------------------------------------------------------- #
# views, tangents
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("lq", [1, 3, 40])
def test_token_strides_of_any_width(gpu, dt, lq):
    """Tokens first: a token's stride is the whole batch's width."""
    wide = 2 ** 31 // (256 * DT[dt].itemsize) + 24
    gen = torch.Generator(device="cuda").manual_seed(1)
    pos = fa.LinePositions(8, 20)
    table = torch.randn(8, 2, generator=gen, device="cuda").to(DT[dt])

    def spread(n):
        flat = torch.empty(n * wide, dtype=DT[dt], device="cuda")
        t = flat.as_strided((1, 2, n, 16), (64, 16, wide, 1))
        t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        return t

    ts, g = [spread(n) for n in (lq, 50, 50)], spread(lq)
    plain = [t.contiguous().requires_grad_(True) for t in ts]
    want = fa.relative_attention(*plain, table, pos)
    want.backward(g.contiguous())
    ts = [t.requires_grad_(True) for t in ts]
    got = fa.relative_attention(*ts, table, pos)
    got.backward(g)
    assert torch.equal(got, want)
    assert all(torch.equal(x.grad, y.grad) for x, y in zip(ts, plain))


def test_a_tangent_is_not_dropped(gpu):
    import torch.autograd.forward_ad as fwd

    pos = fa.LinePositions(8, 20)
    q, k, v = (torch.randn(1, 2, 9, 8, device="cuda") for _ in range(3))
    table = torch.randn(8, 2, device="cuda")
    fa.relative_attention(q, k, v, table, pos)  # (a kernel ran in this test)
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        with pytest.raises((NotImplementedError, RuntimeError)):
            fa.relative_attention(dual, k, v, table, pos)
        with pytest.raises((NotImplementedError, RuntimeError)):
            fa.relative_bias(fwd.make_dual(table, torch.ones_like(table)), pos, 9)


# --------------------------------------------------------------------------- #
# updates
# --------------------------------------------------------------------------- #


def test_more_matrices_than_a_grid_holds(gpu):
    n = 65535 + 70
    gen = torch.Generator().manual_seed(3)
    g = torch.randn(n, 3, 2, generator=gen)
    got = fa.orthogonalize(g.cuda())
    for i in (0, 1, 65533, 65534, 65535, 65536, n - 1):
        near(got[i], ref.orthogonalize(g[i].double().numpy(), 5, STEEP), 3e-5, i)
    assert torch.isfinite(got).all()


#: outside what float16 operands hold: an iterate of 8 (its Gram entry), 1036, a polynomial
#: of 70, an iterate of 34
OUTSIDE = [((2.0, 0.0, 0.0), 5), ((3.0, 0.0, 1.0), 3), ((0.5, 70.0, 0.0), 1), ((1.0, 0.0, 1.0), 3)]
#: inside: iterates of 4, 1.75 (8.5 after the last step), a polynomial of 60
INSIDE = [((2.0, 0.0, 0.0), 3), ((1.0, 0.5, 0.25), 2), ((0.5, 60.0, 0.0), 1)]


def growing(dt, m, n):
    """Singular values from one down."""
    gen = torch.Generator().manual_seed(5)
    u, _, w = torch.linalg.svd(torch.randn(m, n, generator=gen), full_matrices=False)
    return ((u * torch.linspace(1.0, 0.0, m) ** 2) @ w).to(DT[dt])


@pytest.mark.portable_ok
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("coefficients,steps", OUTSIDE)
@pytest.mark.parametrize("m,n", [(1, 1), (70, 90)])
def test_coefficients_that_grow(gpu, dt, coefficients, steps, m, n):
    """Served (in float32) where float16 operands would overflow."""
    g = growing(dt, m, n)
    want = ref.orthogonalize(g.double().numpy(), steps, coefficients)
    if np.abs(want).max() > torch.finfo(DT[dt]).max / 2:
        pytest.skip("the result itself does not fit the type")
    # a step multiplies a relative error by 5 at most (s p'(s) / p(s) of these sets), three
    # steps by 125, of 2^-24 sqrt(90) each; and one rounding
    near(fa.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients), want,
         UNIT[dt] + 2e-4, (m, n))
    with pytest.raises(RuntimeError):
        fa.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients, backend_hint="native")


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("coefficients,steps", INSIDE)
@pytest.mark.parametrize("m,n", [(1, 1), (70, 90)])
def test_coefficients_that_just_fit(gpu, dt, coefficients, steps, m, n):
    g = growing(dt, m, n)
    want = ref.orthogonalize(g.double().numpy(), steps, coefficients)
    # before the rounding as the default coefficients, which multiply errors more; a single
    # value's rounding is half a unit in the last place at most
    near(fa.orthogonalize(g.cuda(), steps=steps, coefficients=coefficients, backend_hint="native"),
         want, {"bf16": 1.5e-3 + 2.0 ** -8, "f16": 2.0 ** -11 + 3e-5, "f32": 3e-5}[dt], (m, n))


# --------------------------------------------------------------------------- #
# a float32 table beside 16-bit activations
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["line", "few", "one", "window", "wide window"])
def test_a_float32_table_keeps_its_digits(gpu, dt, form):
    """Entries of some size, whose rounding to 16 bits would show in the weights; and a
    gradient that is not rounded to them."""
    gen = torch.Generator().manual_seed(31)
    b, h, d, start = 2, 2, 32, 0
    if form == "window":
        pos, lq = fa.GridPositions(8, 8), 64
        lk, rows = lq, ref.grid_rows(8, 8)
    elif form == "wide window":
        pos, lq = fa.GridPositions(9, 10), 90
        lk, rows = lq, ref.grid_rows(9, 10)
    else:
        pos = fa.LinePositions(8, 20)
        lq, lk = {"line": (150, 160), "few": (5, 700), "one": (1, 90)}[form]
        start = lk // 2 if form != "line" else 0
        rows = ref.line_rows(lq, lk, start, 8, 20)
    q, k, v, g = (normal(gen, DT[dt], b, h, n, d) for n in (lq, lk, lk, lq))
    # what they have in common cancels in a row; rounded with it to the type they are off by
    # up to 16 of its units (of one), a weight's error
    table = 20.0 + 0.7 * torch.randn(pos.rows, h, generator=gen)
    see = ref.visible(b, h, lq, lk)
    want = ref.attention(*(t.double().numpy() for t in (q, k, v, table)), rows, see, d ** -0.5,
                         g.double().numpy())
    got = run_attention((q, k, v, table), g, pos, q_start=start)
    assert got[4].dtype == torch.float32
    for name, x, y, t in zip(("out", "dq", "dk", "dv", "dtable"), got, want, (2, 4, 4, 4, 4)):
        near(x, y, t * UNIT[dt] / 2, name)
    assert not torch.equal(got[4], got[4].to(DT[dt]).float())
    with torch.no_grad():
        only = fa.relative_attention(*(t.cuda() for t in (q, k, v, table)), pos, q_start=start)
        same = fa.relative_attention(*(t.cuda() for t in (q, k, v, table.double())), pos, q_start=start)
    near(only, want[0], UNIT[dt], "out, no gradients")
    assert torch.equal(only, same)
