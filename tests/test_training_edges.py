"""The training operators at the edges of their range, without a GPU."""

from __future__ import annotations

import fnmatch
from pathlib import Path

import pytest
import torch

import frame_analytics_amd as fa
from frame_analytics_amd import _build, backend_training


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
