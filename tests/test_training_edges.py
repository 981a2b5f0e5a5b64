"""The training operators at the edges of their range, without a GPU."""

from __future__ import annotations

import ctypes
import fnmatch
from pathlib import Path

import numpy as np
import pytest
import torch

import frame_analytics_amd as fa
from frame_analytics_amd import _build, _cabi, backend_training, training
from oracle import training as ref


def test_row_tables_are_never_given_back():
    """A captured graph reads a table by its address: later descriptions, however many,
    leave it where it is."""
    cpu = torch.device("cpu")
    first = [fa.GridPositions(3, 5), fa.LinePositions(32, 128)]
    tables = [backend_training._row_of(p, cpu) for p in first]
    for w in range(1, 300):
        backend_training._row_of(fa.GridPositions(1, w), cpu)
        backend_training._row_of(fa.LinePositions(8, 20 + w), cpu)
    again = [fa.GridPositions(3, 5), fa.LinePositions(32, 128, bidirectional=True)]
    for p, t in zip(again, tables):
        assert backend_training._row_of(p, cpu) is t
        assert t.tolist() == p.row_of() and t.dtype == torch.int32
    other = fa.LinePositions(32, 128, bidirectional=False)
    assert backend_training._row_of(other, cpu).tolist() == other.row_of()


def test_a_failed_build_leaves_no_file(monkeypatch, tmp_path):
    """Neither half a library nor its temporary, whose name .gitignore holds too."""
    wrote = []

    def fails(cmd, verbose):
        out = Path(cmd[list(cmd).index("-o") + 1])
        out.write_bytes(b"half")
        wrote.append(out)
        raise RuntimeError("command failed")

    monkeypatch.setattr(_build, "LIBDIR", tmp_path)
    monkeypatch.setattr(_build, "_run", fails)
    for build in (_build.build_cpu, _build.build_call):
        with pytest.raises(RuntimeError):
            build()
    ignored = [line for line in (_build.REPO / ".gitignore").read_text().splitlines()
               if line and not line.startswith("#")]
    assert wrote and not list(tmp_path.iterdir())
    for out in wrote:
        assert any(fnmatch.fnmatchcase(out.name, pattern) for pattern in ignored), out.name


def test_what_float16_holds_of_an_update():
    """The largest singular value that coefficients lead to, against a fine grid of them."""
    held = training._held_in_float16
    for coefficients, steps in (((3.4445, -4.7750, 2.0315), 5), ((1.875, -1.25, 0.375), 6),
                                ((3.4445, -4.7750, 2.0315), 10 ** 6), ((2.0, 0.0, 0.0), 3),
                                ((1.0, 0.5, 0.25), 2), ((0.5, 60.0, 0.0), 1), ((1.5, -0.5, 0.0), 9)):
        assert held(*coefficients, steps), coefficients
    nan, inf = float("nan"), float("inf")
    for coefficients, steps in (((2.0, 0.0, 0.0), 5), ((3.0, 0.0, 1.0), 3), ((0.5, 70.0, 0.0), 1),
                                ((1.0, 0.0, 1.0), 3), ((0.1, 0.0, 0.0), 5), ((nan, 0.0, 0.0), 1),
                                ((1.0, inf, 0.0), 1), ((1.0, 0.0, nan), 2), ((1e300, 1e300, 1e300), 4)):
        assert not held(*coefficients, steps), coefficients
    rng = np.random.default_rng(0)
    verdicts = []
    for _ in range(300):
        a, b, c = rng.normal(size=3) * (3.0, 5.0, 3.0)
        s, fits, margin = np.linspace(0.0, 1.0, 20001), True, 1.0
        for _ in range(3):
            top = np.abs(s).max()
            worst = max(2048 * top, 2048 * top ** 2, 1024 * np.abs(b * s ** 2 + c * s ** 4).max())
            fits &= worst <= 65504 and top >= 1 / 64
            margin = min(margin, abs(np.log(worst / 65504)), abs(np.log(top * 64)))
            s = a * s + b * s ** 3 + c * s ** 5
            if not fits:
                break
        if margin > 0.2:  # farther from the limit than the widening
            verdicts.append(fits)
            assert held(a, b, c, 3) == fits, (a, b, c)
    assert 20 < sum(verdicts) < len(verdicts) - 20


def test_the_entry_point_refuses_what_float16_does_not_hold():
    if not _build.library_path().exists():
        _build.build()
    lib = _cabi.bind(ctypes.CDLL(str(_build.library_path())), _cabi.TRAIN_SIGNATURES)
    p = ctypes.addressof(ctypes.create_string_buffer(4096))
    nan = float("nan")
    for a, b, c, steps in ((2.0, 0.0, 0.0, 5), (3.0, 0.0, 1.0, 3), (0.5, 70.0, 0.0, 1),
                           (1.0, 0.0, 1.0, 3), (0.1, 0.0, 0.0, 5), (nan, 0.0, 0.0, 1), (1.0, nan, 0.0, 1)):
        assert lib.fa_gpu_orthogonalize(p, 3, 1, 8, 8, steps, a, b, c, 1e-7, p, p, 1 << 40, 0, None) == 5


@pytest.mark.timeout(60)
@pytest.mark.parametrize("args", [(32, 10 ** 18), (32, 10 ** 30), (16, 10 ** 400), (10 ** 7, 10 ** 8)])
@pytest.mark.parametrize("both", [True, False])
def test_distances_too_far_are_refused_at_once(args, both):
    """Not after a search that counts up to them."""
    with pytest.raises(ValueError, match="supported"):
        fa.LinePositions(*args, bidirectional=both)


def test_a_float32_table_keeps_its_digits():
    """Beside 16-bit activations, on the eager path; its gradient too."""
    gen = torch.Generator().manual_seed(3)
    pos, d = fa.LinePositions(8, 20), 8
    q, k, v = (torch.randn(1, 2, 12, d, generator=gen).bfloat16() for _ in range(3))
    table = (20 + torch.randn(8, 2, generator=gen)).requires_grad_(True)
    up = torch.randn(1, 2, 12, d, generator=gen).bfloat16()
    out = fa.relative_attention(q, k, v, table, pos)
    out.backward(up)
    want = ref.attention(*(t.detach().double().numpy() for t in (q, k, v, table)),
                         ref.line_rows(12, 12, 0, 8, 20), ref.visible(1, 2, 12, 12), d ** -0.5,
                         up.double().numpy())
    assert table.grad.dtype == torch.float32
    for x, y, tol in ((out, want[0], 2.0 ** -8), (table.grad, want[4], 1e-5)):
        assert np.linalg.norm(x.detach().double().numpy() - y) <= tol * np.linalg.norm(y)


def test_stacks_of_small_matrices_are_not_padded_to_wide_tiles():
    """Whatever their number, matrices of up to 64 rows take tiles of 64: each operand
    (three of X, two of the square ones, hi and lo) is 64 x 64 of float16, beside the norm's
    sums."""
    if not _build.library_path().exists():
        _build.build()
    lib = _cabi.bind(ctypes.CDLL(str(_build.library_path())), _cabi.TRAIN_SIGNATURES)
    out = ctypes.c_int64(0)
    for batch, rows, cols in ((1, 16, 27), (4096, 16, 27), (600, 64, 64), (65535, 3, 2)):
        assert lib.fa_gpu_orthogonalize_workspace(3, batch, rows, cols, ctypes.byref(out)) == 0
        assert out.value <= batch * (5 * 2 * 64 * 64 * 2 + 512 * 8 + 4) + 8 * 256
