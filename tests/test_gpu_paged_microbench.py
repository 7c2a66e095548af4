"""The bytes that the microbenchmark of the paged operators counts are those that the measured cases count."""
import importlib.util
import json
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")


@pytest.mark.parametrize("rows,lo,hi,br,n", [(5, 40, 900, 16, 9), (64, 15, 1600, 32, 20), (1, 700, 700, 64, 40)])
def test_bytes_are_those_of_the_measured_cases(capsys, monkeypatch, rows, lo, hi, br, n):
    from goinfer_b200 import microbench
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("measured_cases", at)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    monkeypatch.setattr(sys, "argv", f"microbench paged --rows {rows} --ctx-lo {lo} --ctx-hi {hi} --heads 8 --kv-heads 2 --head-dim 64 --block-rows {br} "
                                     f"--select {n} --iters 2".split())
    microbench.main()
    got = {x["kernel"].split()[1]: x["bytes"] for x in map(json.loads, capsys.readouterr().out.splitlines())}
    layout = (8, 2, 64)
    assert got["append"] == cases.work(cases._append("", rows, lo, hi, 1, layout, br))["bytes"]
    assert got["select"] == cases.work(cases._select("", rows, lo + 1, hi + 1, layout, br, n))["bytes"]
    assert got["attend"] == cases.work(cases._attend("", rows, lo + 1, hi + 1, layout, br, n))["bytes"]
    assert got["plan"] == 4 * 8 * rows
