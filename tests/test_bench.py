"""bench.py's lines where the reference CPU runtime is not built."""

from __future__ import annotations

import json
import sys
from types import SimpleNamespace


def test_reference_arm_without_the_reference(monkeypatch, capsys):
    """One line that says why, and no error."""
    import bench
    import oracle

    monkeypatch.setattr(oracle, "REF_LIB", bench.REPO / "oracle" / "_ref" / "missing.so")
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--steps", "1", "--warmup", "3"])
    bench.main()
    lines = capsys.readouterr().out.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and "missing.so" in line["unavailable"] and "\n" not in line["unavailable"]
    bench.run_reference_arm(SimpleNamespace(int8=False), SimpleNamespace(rank=1))  # another rank says nothing
    assert capsys.readouterr().out == ""
