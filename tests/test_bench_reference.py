"""The reference arm of bench.py measures the reference or nothing."""
import json
import sys

import bench
from oracle import oracle_py


def test_without_a_reference_build_the_arm_is_unavailable(monkeypatch, capsys):
    def never(*_, **__):
        raise AssertionError("something else was measured in the reference's place")

    monkeypatch.setattr(oracle_py, "ref_available", lambda: False)
    monkeypatch.setattr(bench, "prepare_model", never)
    monkeypatch.setattr(oracle_py, "PortModel", never)
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--steps", "2", "--warmup", "3"])
    bench.main()
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
