"""Building of the native parts with several processes or threads at it (no GPU needed)."""
import os
import subprocess
import sys
import threading
import time

import pytest

from prism_b200 import build as b

WHOLE = b"x" * 1000


def _slow_compiler(calls):
    """A compiler that writes its output in two halves."""
    def run(cmd, check):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "wb") as f:
            f.write(WHOLE[:500])
            f.flush()
            time.sleep(0.2)
            f.write(WHOLE[500:])
    return run


def test_a_file_appears_whole_and_is_built_once(tmp_path, monkeypatch):
    target, calls, seen = str(tmp_path / "ext.so"), [], set()
    monkeypatch.setattr(b, "torch_ops_lib", lambda: target)
    monkeypatch.setattr(b.subprocess, "run", _slow_compiler(calls))
    threads = [threading.Thread(target=b.build_torch_ops) for _ in range(4)]
    for t in threads:
        t.start()
    while any(t.is_alive() for t in threads):
        if os.path.exists(target):
            seen.add(os.path.getsize(target))
        time.sleep(0.005)
    assert seen <= {len(WHOLE)} and open(target, "rb").read() == WHOLE
    assert len(calls) == 1
    assert os.listdir(tmp_path) == ["ext.so"]


def test_a_failed_build_leaves_nothing(tmp_path, monkeypatch):
    target = str(tmp_path / "ext.so")

    def fail(cmd, check):
        open(cmd[cmd.index("-o") + 1], "wb").write(WHOLE[:10])
        raise subprocess.CalledProcessError(1, cmd)
    monkeypatch.setattr(b, "torch_ops_lib", lambda: target)
    monkeypatch.setattr(b.subprocess, "run", fail)
    with pytest.raises(subprocess.CalledProcessError):
        b.build_torch_ops()
    assert os.listdir(tmp_path) == []


def test_processes_build_once(tmp_path):
    """Four processes find the file absent at the same time."""
    code = f"""
import sys, time
sys.path.insert(0, {os.path.dirname(os.path.dirname(os.path.abspath(__file__)))!r})
from prism_b200 import build as b
b.torch_ops_lib = lambda: {str(tmp_path / 'ext.so')!r}
def run(cmd, check):
    open({str(tmp_path / 'calls')!r}, "a").write("x")
    time.sleep(0.3)
    open(cmd[cmd.index("-o") + 1], "wb").write({WHOLE!r})
b.subprocess.run = run
b.build_torch_ops()
"""
    ranks = [subprocess.Popen([sys.executable, "-c", code]) for _ in range(4)]
    assert [r.wait(timeout=120) for r in ranks] == [0] * 4
    assert (tmp_path / "calls").read_text() == "x"
