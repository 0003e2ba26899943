"""What only Python's cycle collector frees is freed where a test module ends. A test that compares torch.cuda.memory_allocated() over a
window must not depend on when the collector runs: tensors that an earlier module left in a cycle (in the frames that an exception
kept by a test holds, say) would be freed within the window."""
import os
import subprocess
import sys

LEAVES = """
import gc, weakref
class Held: pass
left = None
def test_leaves_a_cycle():
    global left
    gc.disable()
    held = Held()
    held.itself = held
    left = weakref.ref(held)
    del held
    assert left() is not None
"""
FINDS = """
import test_a_leaves
def test_finds_none():
    assert test_a_leaves.left is not None and test_a_leaves.left() is None
"""


def test_a_module_leaves_nothing_to_the_collector(tmp_path):
    (tmp_path / "test_a_leaves.py").write_text(LEAVES)
    (tmp_path / "test_b_finds.py").write_text(FINDS)
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join(p for p in (here, os.environ.get("PYTHONPATH")) if p)
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "conftest", "-p", "no:cacheprovider", "--rootdir", str(tmp_path),
                          str(tmp_path)], cwd=str(tmp_path), env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "2 passed" in run.stdout, run.stdout + run.stderr
