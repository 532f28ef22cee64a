"""The line of JSON that bench.py ends with (CPU only)."""
from __future__ import annotations

import json

import bench


def test_result_line_is_one_line_without_spaces_between_values():
    r = {"metric": "dequant GB/s, all of it", "value": 6617.05, "vs_baseline": None, "flags": [True, False],
         "config": {"workload": "a, b", "legs": [{"ms": 1.5, "name": "x"}] * 3}}
    line = bench.result_line(r)
    assert json.loads(line) == r and "\n" not in line
    assert line.count(", ") == 2  # those of the texts


def test_a_timeline_lists_its_longest_gaps_only():
    """A leg with many gaps between its loads does not lengthen the line without bound."""
    loads, at = [], 0.0
    for n in range(20):  # block n is copied for 5 ms, n + 2 ms after the one before
        loads.append((f"blocks.{n}", 0, at, at + 5.0))
        at += 5.0 + n + 2.0
    gaps = bench.load_gap_causes({"loads": loads})
    assert [g["gap_ms"] for g in gaps] == [20.0, 19.0, 18.0]
