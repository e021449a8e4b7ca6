"""Regression test of "defect (a)" (a host SIGSEGV inside a later hipGraphLaunch after mid-life hipGraphExecDestroy calls, seen with
graphs launched on a normal-priority stream): the library must survive every stream-creation / -destruction history of its process.
It launches its step graphs on a stream of another priority class, on which the crash was never seen.
The reference has no such state (one tf.Session per process, sga.py:178-182)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_step_graphs_survive_adversarial_stream_histories():
    """tests/tools/graph_stream_stress.py in a subprocess (a crash must not take pytest down): 64 histories of six ballast streams,
    freed-memory poisoning on (MALLOC_PERTURB_: a use of freed memory shows instead of finding what was there before), a fresh
    handle each, the three fork-point candidates instantiated and launched, two of them destroyed in mid-life, bit-equal
    results."""
    env = dict(os.environ, MALLOC_PERTURB_="165")
    env.pop("SGA_LAUNCH_STREAM", None)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "tools", "graph_stream_stress.py")], env=env, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, (r.returncode, r.stdout[-600:], r.stderr[-1500:])
    assert "survived 64 stream histories" in r.stdout, r.stdout[-600:]
