"""bench.py where ctorch's CPU backend has not been built: the reference arm says so in its line, and the other
arms leave the CPU baseline out."""
import json
import os
import sys

import pytest

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))


@pytest.fixture
def unbuilt(monkeypatch):
    import bench
    from oracle import oracle

    monkeypatch.setattr(oracle, "REF_SO", "/nonexistent/libctorch_ref.so")
    for v in ("RANK", "LOCAL_RANK", "WORLD_SIZE"):
        monkeypatch.delenv(v, raising=False)
    return bench


def test_reference_arm_prints_why_it_is_unavailable(unbuilt, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--gpus", "1", "--steps", "2", "--warmup", "3"])
    assert unbuilt.main() == 0
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and "not built" in line["unavailable"]


def test_reference_arm_prints_one_line_for_all_ranks(unbuilt, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--gpus", "2"])
    monkeypatch.setenv("RANK", "1")
    monkeypatch.setenv("WORLD_SIZE", "2")
    assert unbuilt.main() == 0
    assert capsys.readouterr().out == ""


@pytest.mark.parametrize("argv,arm", [([], "run_b200"), (["--suite"], "run_suite")])
def test_other_arms_leave_the_cpu_baseline_out(unbuilt, monkeypatch, capsys, argv, arm):
    seen = []
    monkeypatch.setattr(unbuilt, arm, lambda args: seen.append(args.no_cpu_baseline) or 0)
    monkeypatch.setattr(sys, "argv", ["bench.py", *argv])
    assert unbuilt.main() == 0
    assert seen == [True]
    out = capsys.readouterr()
    assert out.out == "" and "not built" in out.err
