"""The example that runs the 8-bit operators together trains and rolls out."""
import importlib.util
import os
import re
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_example_runs(monkeypatch, capsys):
    path = os.path.join(ROOT, "examples", "eight_bit_rollout.py")
    spec = importlib.util.spec_from_file_location("eight_bit_rollout", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    monkeypatch.setattr(sys, "argv", [path, "--particles", "3000", "--steps", "4", "--epochs", "12"])
    example.main()
    out = capsys.readouterr().out
    losses = [float(v) for v in re.findall(r"loss (?:on another cloud )?([0-9.]+)", out)]
    held = [int(v) for v in re.findall(r"holds (\d+) MiB", out)]
    assert len(losses) == 4 and len(held) == 2 and held[1] < held[0]
    assert abs(losses[1] - losses[0]) < 0.1 * losses[0] and abs(losses[3] - losses[2]) < 0.1 * losses[2]
