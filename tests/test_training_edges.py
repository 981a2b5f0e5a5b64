"""The training operators at the edges of their range, without a GPU."""

from __future__ import annotations

import torch

import frame_analytics_amd as fa
from frame_analytics_amd import backend_training


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
