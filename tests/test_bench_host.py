"""bench.py's host legs where the reference's own CPU kernel is not built."""
from __future__ import annotations

import json
import subprocess
import sys
import time

from conftest import REPO


def test_the_reference_arm_says_that_it_is_unavailable():
    """One line and exit code 0, at once, instead of timing another implementation."""
    code = ("import sys; sys.path[:0] = ['.', 'oracle']\n"
            "import slr_oracle; slr_oracle.ref_avx2_module = lambda: None\n"
            "import bench; sys.argv = ['bench.py', '--impl', 'reference', '--steps', '2', '--warmup', '1']\n"
            "bench.main()\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout)
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference" and "not built" in line["unavailable"]


def test_the_cpu_baseline_keeps_its_budget(monkeypatch):
    """Without the kernel the plain C port is timed, on as many tokens as the budget allows."""
    monkeypatch.syspath_prepend(str(REPO))
    import bench
    import slr_oracle
    from s_salaad_b200 import workloads

    monkeypatch.setattr(slr_oracle, "ref_avx2_module", lambda: None)
    crow, col = workloads.bernoulli_structure(64, 64, 0.4, seed=1)
    spec = workloads.LayerSpec("l", 2048, 2048, 256, 32, 32, crow, col, seed=2, bias_std=0.01)
    t0 = time.perf_counter()
    times, tokens, kind, cores, _ = bench.cpu_reference_run([spec], 4096, 0, 1, 1.0)
    assert time.perf_counter() - t0 < 30
    assert kind == "port" and cores == 1 and len(times) >= 3 and 1 <= tokens < 4096
    # a sample that fits is timed whole
    assert bench.cpu_reference_run([spec], 2, 0, 1, 2.0)[1] == 2
