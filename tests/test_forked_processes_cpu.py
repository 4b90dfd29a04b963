"""What one test module leaves behind must not be destroyed in a process that a later one forks: device tensors and captured graphs among
it would call a HIP runtime that the fork does not have."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))

LEAVES = '''
import gc, os
class Held:
    def __init__(self):
        self.me = self                      # only a collection finds it
    def __del__(self):
        open("destroyed_by", "a").write(f"{os.getpid()}\\n")
def test_leaves_something_behind():
    gc.disable()
    Held()
'''
FORKS = '''
import gc, multiprocessing as mp, os
def test_forks():
    child = mp.get_context("fork").Process(target=gc.collect)
    child.start()
    child.join()
    assert child.exitcode == 0
    assert open("destroyed_by").read().split() == [str(os.getpid())]
'''


def test_a_module_leaves_nothing_for_a_fork_to_destroy(tmp_path):
    (tmp_path / "conftest.py").write_text(open(os.path.join(HERE, "conftest.py")).read())
    (tmp_path / "test_a.py").write_text(LEAVES)
    (tmp_path / "test_b.py").write_text(FORKS)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "test_a.py", "test_b.py"], cwd=tmp_path, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "2 passed" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
