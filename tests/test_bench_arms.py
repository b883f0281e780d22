"""bench.py's host arms where the reference is not installed: the reference arm says so and loads
nothing of this package, the port is an arm of its own."""

from __future__ import annotations

import json
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


def _run(impl: str) -> tuple[dict, bool]:
    code = (
        "import runpy, sys\n"
        f"sys.argv = ['bench.py', '--impl', '{impl}', '--steps', '1', '--warmup', '3']\n"
        "runpy.run_path('bench.py', run_name='__main__')\n"
        "maps = open('/proc/self/maps').read()\n"
        "print('PRODUCT', 'libaios_b200' in maps or any(m.split('.')[0] == 'aios_b200' for m in sys.modules))\n"
    )
    proc = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-2000:]
    lines = proc.stdout.strip().splitlines()
    return json.loads(next(x for x in lines if x.startswith("{"))), lines[-1] == "PRODUCT True"


@pytest.mark.skipif((REPO / "baseline" / "_ref" / "aios" / "ime.py").exists(), reason="the reference is installed")
def test_reference_arm_without_the_reference() -> None:
    line, product = _run("reference")
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference" and "baseline/_ref" in line["unavailable"]
    assert "\n" not in line["unavailable"] and not product


def test_the_port_is_called_so() -> None:
    line, _ = _run("port")
    assert line["impl"] == "port" and line["cpu_baseline"]["kind"] == "port" and line["value"] > 0
