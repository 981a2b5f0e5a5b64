"""The training operators without a GPU: positions, the eager path against float64,
refusals, and the C ABI's declarations and argument checks."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import frame_analytics_amd as fa
from frame_analytics_amd import _build, _cabi, training
from oracle import training as ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "fa_train_abi.h"


@pytest.mark.parametrize("n,far,both", [(32, 128, True), (32, 128, False), (4, 3, True), (2, 2, False),
                                        (16, 40, True), (64, 2000, True), (9, 100, False)])
def test_line_rows(n, far, both):
    pos = fa.LinePositions(n, far, bidirectional=both)
    for delta in list(range(-far - 70, far + 70)) + [-(10 ** 9), 10 ** 9]:
        slot = min(max(delta - pos.lo, 0), pos.slots - 1)
        want = ref.line_row(-delta, n, far, both)
        assert pos.row_of()[slot] == want == pos._row(delta), delta
    rows = pos.row_of()
    seen = [r for i, r in enumerate(rows) if i == 0 or rows[i - 1] != r]
    assert len(seen) == len(set(seen))  # equal rows stand together


def test_bucket_edges_are_exact():
    # 8 * 16 ** (j / 8) is a whole number for j = 2, 4, 6: those distances start a bucket
    pos = fa.LinePositions(32, 128)
    assert [pos._row(d) for d in (15, 16, 31, 32, 63, 64)] == [9, 10, 11, 12, 13, 14]


@pytest.mark.parametrize("h,w", [(1, 1), (1, 5), (5, 1), (4, 7), (33, 33)])
def test_window_rows(h, w):
    pos = fa.GridPositions(h, w)
    rows = training._pair_rows(pos, h * w, h * w, 0, "cpu")[0].numpy()
    assert np.array_equal(rows, ref.grid_rows(h, w))
    assert pos.slots == pos.rows == rows.max() + 1


def test_positions_refuse():
    for bad in ((1, 8), (3, 8), (5, 100), (32, 8)):
        with pytest.raises(ValueError):
            fa.LinePositions(*bad)
    with pytest.raises(ValueError):
        fa.LinePositions(32, 1 << 20)
    with pytest.raises(ValueError):
        fa.GridPositions(34, 33)
    with pytest.raises(ValueError):
        fa.GridPositions(0, 3)
    assert fa.GridPositions(4, 4) == fa.GridPositions(4, 4)
    assert hash(fa.LinePositions(8, 20)) == hash(fa.LinePositions(8, 20))


@pytest.mark.parametrize("dtype,tol", [(torch.float64, 1e-12), (torch.float32, 1e-5)])
@pytest.mark.parametrize("form", ["line", "causal", "window", "mask", "lengths", "token"])
def test_eager_attention(form, dtype, tol):
    gen = torch.Generator().manual_seed(1)
    b, h, hk, lq, lk, d = 2, 4, 2, 12, 12, 6
    pos, rows, kw = fa.LinePositions(8, 20), None, {}
    if form == "causal":
        kw = {"causal": True, "q_start": 2}
    elif form == "window":
        pos, rows = fa.GridPositions(3, 4), ref.grid_rows(3, 4)
    elif form == "mask":
        mask = torch.rand(2, 1, lq, lk, generator=gen) < 0.5
        mask[0, 0, 3] = False
        kw = {"mask": mask}
    elif form == "lengths":
        kw = {"key_lengths": torch.tensor([0, 7])}
    elif form == "token":
        lq = 1
        kw = {"key_lengths": torch.tensor([5, 12]), "q_start": torch.tensor([4, 11])}
        rows = np.stack([ref.line_rows(1, lk, s, 8, 20) for s in (4, 11)])
    if rows is None:
        rows = ref.line_rows(lq, lk, kw.get("q_start", 0), 8, 20)
    mk = lambda *s: torch.randn(*s, generator=gen).to(dtype).requires_grad_(True)  # noqa: E731
    q, k, v, table = mk(b, h, lq, d), mk(b, hk, lk, d), mk(b, hk, lk, d), mk(pos.rows, h)
    up = torch.randn(b, h, lq, d, generator=gen).to(dtype)
    see = ref.visible(b, h, lq, lk, **{n: t.numpy() if torch.is_tensor(t) else t
                                       for n, t in kw.items()})
    want = ref.attention(*(t.detach().numpy() for t in (q, k, v, table)), rows, see, d ** -0.5,
                         up.numpy())
    out = fa.relative_attention(q, k, v, table, pos, **kw)
    out.backward(up)
    for x, y in zip((out, q.grad, k.grad, v.grad, table.grad), want):
        assert np.abs(x.detach().numpy() - y).max() <= tol * max(1.0, np.abs(y).max())


def test_eager_bias_and_update():
    gen = torch.Generator().manual_seed(2)
    pos = fa.LinePositions(8, 20, bidirectional=False)
    table = torch.randn(8, 3, generator=gen, dtype=torch.float64, requires_grad=True)
    out = fa.relative_bias(table, pos, 7, 11, q_start=4)
    rows = ref.line_rows(7, 11, 4, 8, 20, False)
    assert np.array_equal(out.detach().numpy(), ref.bias(table.detach().numpy(), rows))
    up = torch.randn(out.shape, generator=gen, dtype=torch.float64)
    out.backward(up)
    assert np.abs(table.grad.numpy() - ref.bias_grad(up.numpy(), rows, 8)).max() < 1e-12
    for shape in ((5, 9), (9, 5)):
        g = torch.randn(2, *shape, generator=gen, dtype=torch.float64)
        got = fa.orthogonalize(g)
        want = np.stack([ref.orthogonalize(x.numpy(), 5, (3.4445, -4.7750, 2.0315)) for x in g])
        assert np.abs(got.numpy() - want).max() < 1e-10


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(0)
    rows = ref.line_rows(5, 6, 1, 8, 20)
    see = ref.visible(1, 2, 5, 6, causal=True, q_start=1)
    ts = [rng.standard_normal(s) for s in ((1, 2, 5, 3), (1, 1, 6, 3), (1, 1, 6, 3), (8, 2))]
    up = rng.standard_normal((1, 2, 5, 3))
    grads = ref.attention(*ts, rows, see, 0.6, up)[1:]
    for i, g in enumerate(grads):
        for at in np.ndindex(g.shape):
            f = []
            for s in (1e-5, -1e-5):
                moved = [t.copy() for t in ts]
                moved[i][at] += s
                f.append((ref.attention(*moved, rows, see, 0.6) * up).sum())
            assert abs((f[0] - f[1]) / 2e-5 - g[at]) < 1e-8


def test_refusals():
    pos = fa.LinePositions(8, 20)
    q, k, t = torch.randn(2, 4, 5, 8), torch.randn(2, 2, 6, 8), torch.randn(8, 4)
    ok = dict(q=q, k=k, v=k, table=t, positions=pos)
    fa.relative_attention(**ok)
    for error, change in (
            (ValueError, {"q": q[0]}), (TypeError, {"q": q.int()}), (ValueError, {"k": k.double()}),
            (ValueError, {"v": k[:, :, :5]}), (ValueError, {"k": k[..., :7], "v": k[..., :7]}),
            (ValueError, {"q": q[:, :3], "table": t[:, :3]}), (ValueError, {"table": t[:, :3]}),
            (ValueError, {"table": t[:7]}), (TypeError, {"positions": 3}),
            (ValueError, {"positions": fa.GridPositions(1, 5), "table": torch.randn(9, 4)}),
            (TypeError, {"mask": torch.ones(5, 6)}),
            (ValueError, {"mask": torch.ones(5, 5, dtype=torch.bool)}),
            (ValueError, {"mask": torch.ones(3, 1, 5, 6, dtype=torch.bool)}),
            (ValueError, {"mask": torch.ones(2, 2, 5, 6, dtype=torch.bool)}),
            (ValueError, {"key_lengths": torch.ones(3, dtype=torch.int32)}),
            (ValueError, {"key_lengths": torch.ones(2)}),
            (ValueError, {"q_start": torch.ones(1, dtype=torch.int64)}),
            (ValueError, {"backend_hint": "cuda"}), (RuntimeError, {"backend_hint": "native"}),
            (ValueError, {"q": torch.randn(2, 4, 5, 129), "k": torch.randn(2, 2, 6, 129),
                          "v": torch.randn(2, 2, 6, 129)})):
        with pytest.raises(error):
            fa.relative_attention(**{**ok, **change})
    for args in ((t[:7], pos, 3), (t, pos, -1), (t[:, 0], pos, 3), (t.int(), pos, 3)):
        with pytest.raises((ValueError, TypeError)):
            fa.relative_bias(*args)
    with pytest.raises(TypeError):
        fa.relative_bias(t, pos, 3, q_start=torch.tensor([1]))
    for kw in ({"steps": 0}, {"eps": 0.0}, {"coefficients": (1.0, 2.0)}):
        with pytest.raises(ValueError):
            fa.orthogonalize(torch.randn(3, 4), **kw)
    with pytest.raises(ValueError):
        fa.orthogonalize(torch.randn(3))
    with pytest.raises(TypeError):
        fa.orthogonalize(torch.ones(3, 3, dtype=torch.int64))


# --------------------------------------------------------------------------- #
# the C ABI
# --------------------------------------------------------------------------- #


def _declared():
    txt = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"FA_API\s+int\s+(fa_\w+)\s*\(([^)]*)\)\s*;", txt, flags=re.S)}


@pytest.fixture(scope="module")
def lib():
    if not _build.library_path().exists():
        _build.build()
    return _cabi.bind(ctypes.CDLL(str(_build.library_path())), _cabi.TRAIN_SIGNATURES)


def test_header_binder_and_library_agree(lib):
    decl = _declared()
    assert set(decl) == set(_cabi.TRAIN_SIGNATURES)
    for name, n in decl.items():
        assert len(_cabi.TRAIN_SIGNATURES[name][0]) == n, name
        assert hasattr(lib, name), name
    assert not set(decl) & set(_cabi.SIGNATURES)


def test_callers_match_ctypes(lib):
    callers = _cabi.load_callers(_cabi.load_gpu()[0], _cabi.TRAIN_SIGNATURES)
    assert set(callers) == {n for n in _cabi.TRAIN_SIGNATURES if not n.endswith("workspace")}
    for name, fast in callers.items():
        args = [None if k is ctypes.c_void_p else 0.5 if k is ctypes.c_double else 0
                for k in _cabi.TRAIN_SIGNATURES[name][0]]
        want = getattr(lib, name)(*args)
        assert want != 0 and fast(*args) == want, name


def test_arguments_are_checked_before_any_gpu_work(lib):
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    n64 = ctypes.c_int64(0)
    out = ctypes.byref(n64)
    st = (ctypes.c_int64 * 24)()
    bias = lib.fa_gpu_rel_bias
    assert bias(None, 3, 8, 2, 5, 5, p, -4, 9, 0, 0, p, 0, None) == 5
    assert bias(p, 3, 8, 2, 5, 5, None, -4, 9, 0, 0, p, 0, None) == 5
    assert bias(p, 3, 8, 0, 5, 5, p, -4, 9, 0, 0, p, 0, None) == 2
    assert bias(p, 3, 8, 2, 5, 5, p, -4, 4226, 0, 0, p, 0, None) == 2
    assert bias(p, 3, 49, 2, 16, 16, p, -24, 49, 5, 0, p, 0, None) == 2   # 16 is no 5 x ?
    assert bias(p, 3, 49, 2, 16, 16, p, -24, 48, 4, 0, p, 0, None) == 2   # not the whole window
    assert bias(p, 3, 49, 2, 16, 16, p, -24, 49, 4, 1, p, 0, None) == 2   # a window has no start
    ws = lib.fa_gpu_rel_bias_workspace
    assert ws(2, 100, 5, 9, out) == 0 and n64.value >= 2 * 9 * 4
    small = n64.value - 1
    assert ws(2, 100, 5, 9, None) == 5 and ws(2, 0, 5, 9, out) == 2
    back = lib.fa_gpu_rel_bias_backward
    assert back(p, st, 3, 8, 2, 100, 5, p, -4, 9, 0, 0, p, p, small, 0, None) == 5
    att = lib.fa_gpu_rel_attention

    def attention(dtype=3, b=1, h=2, hk=1, lq=4, lk=4, d=8, strides=st, n=9, grid=0, mask=None,
                  mask_b=1, ms=None, table=p):
        return att(p, p, p, dtype, b, h, hk, lq, lk, d, strides, table, 8, p, -4, n, grid, 0, None,
                   None, mask, mask_b, ms, 0, 1.0, p, None, None, 0, 0, None)

    assert attention(strides=None) == 5 and attention(table=None) == 5
    for kw in ({"b": 0}, {"h": 3, "hk": 2}, {"lq": 0}, {"lk": 0}, {"d": 129}, {"d": 0}, {"n": 0},
               {"grid": 4}, {"mask": p, "mask_b": 2, "ms": st}):
        assert attention(**kw) == 2, kw
    assert attention(mask=p) == 5  # a mask without strides
    aws = lib.fa_gpu_rel_attention_workspace
    assert aws(1, 2, 1, 4, 4, 8, 9, 0, None) == 5
    assert aws(1, 2, 1, 4, 4, 8, 0, 0, out) == 2
    bws = lib.fa_gpu_rel_attention_backward_workspace
    assert bws(1, 2, 1, 4, 4, 8, 9, 0, 1, 0, out) == 0 and n64.value >= 2 * 4 * 4 + 2 * 9 * 4
    need = n64.value
    bwd = lib.fa_gpu_rel_attention_backward
    assert bwd(p, p, p, p, p, p, 3, 1, 2, 1, 4, 4, 8, st, p, 8, p, -4, 9, 0, 0, None, None, None, 1,
               None, 0, 1.0, p, p, p, p, p, need - 1, 0, None) == 5
    ows = lib.fa_gpu_orthogonalize_workspace
    assert ows(2, 1, 100, 50, out) == 0 and n64.value > 0
    assert ows(0, 1, 100, 50, out) == 1 and ows(3, 0, 100, 50, out) == 2
    ort = lib.fa_gpu_orthogonalize
    assert ort(p, 3, 1, 8, 8, 0, 1.0, 1.0, 1.0, 1e-7, p, p, 1 << 40, 0, None) == 5  # no step
    assert ort(p, 3, 1, 8, 8, 1, 1.0, 1.0, 1.0, 0.0, p, p, 1 << 40, 0, None) == 5   # no eps
    assert ort(p, 3, 1, 8, 8, 1, 1.0, 1.0, 1.0, 1e-7, p, p, 16, 0, None) == 5       # workspace
    assert ort(p, 0, 1, 8, 8, 1, 1.0, 1.0, 1.0, 1e-7, p, p, 1 << 40, 0, None) == 1  # uint8


def test_example_trains():
    import importlib.util

    path = Path(__file__).resolve().parents[1] / "examples" / "train_restorer.py"
    spec = importlib.util.spec_from_file_location("train_restorer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses = module.main(["--steps", "5", "--size", "32", "--batch", "2", "--device", "cpu"])
    assert losses[-1] < losses[0]
